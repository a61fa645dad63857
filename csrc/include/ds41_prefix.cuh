// What the kernels of attention over a shared prefix share (prefix_attn.cu, prefix_group.cu, prefix_latent.cu).
//
// A row's keys are divided into parts: ranges of pages that several requests' page tables begin with, read once for all of them, and
// ranges of its own.  Softmax over a divided set of keys needs of every part only its maximum m, its sum l = sum exp(s - m) and its
// unnormalised result o = sum exp(s - m) v: with M = max m_i the whole is sum exp(m_i - M) o_i / sum exp(m_i - M) l_i.
//
// The plan is made on the host from the page tables (ops/prefix.py).  A unit is a range of keys, the rows that see them and a key/value
// head; the parts of row r are the cells cell[r] .. cell[r] + parts[r] - 1 of [cell][head].  A tail is a range behind the shared
// pages: its rows belong to one request, and it ends at the last of their positions, which the host does not know.
#pragma once
#include "ds41_stack.cuh"

namespace ds41 {

struct PrefixUnit {
  int slot, first, rows, key0, key1, part, tail, head;
};
constexpr int kUnitInts = 8;

__device__ __forceinline__ PrefixUnit prefix_unit(const ds41_prefix_plan& p, int i) {
  const int4 a = *reinterpret_cast<const int4*>(p.units + 1ll * i * kUnitInts);
  const int4 b = *reinterpret_cast<const int4*>(p.units + 1ll * i * kUnitInts + 4);
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}
__device__ __forceinline__ int prefix_row(const ds41_prefix_plan& p, const PrefixUnit& u, int i) {
  return u.tail ? u.first + i : p.order[u.first + i];
}
// Whole warps: the keys [first, end) that a unit's rows see.  `first` is a page's; a chunk's border may lie inside, and between the
// windows of rows in different chunks there may be places that nobody sees.  Those and the ones behind `end`, which shared pages have
// as well since rows may stand inside them, may hold anything.  In two steps, so that the positions of several units can be under
// way together.
struct PrefixRows {
  int low, high;                       // of this lane's rows that see any of the unit's keys; of all lanes' behind prefix_span()
  int wide_low, wide_high;             // the longest window of one of them, inside the unit
};
__device__ __forceinline__ PrefixRows prefix_rows(const ds41_prefix_plan& p, const PrefixUnit& u, const int* row_pos, const int* row_slot,
                                                  int chunk) {
  PrefixRows v = {u.key1, 0, u.key0, u.key0};
  for (int i = threadIdx.x & 31; i < u.rows; i += 32) {
    const int r = prefix_row(p, u, i), pos = row_pos[r];
    const int low = chunk > 0 ? pos - pos % chunk : 0, from = max(low, u.key0), high = min(pos + 1, u.key1);
    if (row_slot[r] < 0 || from >= high) continue;
    v.low = min(v.low, low);
    v.high = max(v.high, high);
    if (high - from > v.wide_high - v.wide_low) {
      v.wide_low = from;
      v.wide_high = high;
    }
  }
  return v;
}
__device__ __forceinline__ void prefix_span(const PrefixUnit& u, PrefixRows& v, int chunk, int page_tokens, int& first, int& end) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    v.low = min(v.low, __shfl_xor_sync(0xffffffffu, v.low, o));
    v.high = max(v.high, __shfl_xor_sync(0xffffffffu, v.high, o));
  }
  first = chunk > 0 ? max(u.key0, v.low - v.low % page_tokens) : u.key0;
  end = max(first, min(u.key1, v.high));
}
// Whole warps: the longest window of all lanes' rows.
__device__ __forceinline__ void prefix_widest(const PrefixRows& v, int& low, int& high) {
  low = v.wide_low;
  high = v.wide_high;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const int l = __shfl_xor_sync(0xffffffffu, low, o), h = __shfl_xor_sync(0xffffffffu, high, o);
    if (h - l > high - low) {
      low = l;
      high = h;
    }
  }
}
// Whole warps: which of the 64 places from `key` on are seen by one of this lane's rows of a unit.
__device__ __forceinline__ unsigned long long prefix_seen(const ds41_prefix_plan& p, const PrefixUnit& u, const int* row_pos,
                                                          const int* row_slot, int chunk, int key) {
  unsigned long long seen = 0;
  for (int i = threadIdx.x & 31; i < u.rows; i += 32) {
    const int r = prefix_row(p, u, i), pos = row_pos[r];
    const int from = max(pos - pos % chunk - key, 0), to = min(min(pos + 1, u.key1) - key, 64);
    if (row_slot[r] >= 0 && from < to) seen |= (~0ull >> (64 - (to - from))) << from;
  }
  return seen;
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}

// Four products of 16 columns of K each in one go, by the one thread that calls this; `accumulate` is the first one's.  Between two
// products written one by one the compiler moves every operand to the uniform registers again: 128 x 64 x 16 took 83 cycles each
// with A in tensor memory and 52 with A in shared memory, 34 and 50 so (32 is the tensor core's time, 48 that of two operands from
// shared memory).  ASTEP / BSTEP: from one product's operands to the next one's, in columns of tensor memory or units of 16 bytes.
template <int BSTEP>
__device__ __forceinline__ void umma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b32 x;\n\t.reg .b64 y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "add.s32 x, %1, 8;\n\tadd.s64 y, %2, %5;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
      "add.s32 x, %1, 16;\n\tadd.s64 y, %2, %6;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
      "add.s32 x, %1, 24;\n\tadd.s64 y, %2, %7;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(BSTEP), "n"(2 * BSTEP), "n"(3 * BSTEP)
      : "memory");
}
template <int ASTEP, int BSTEP>
__device__ __forceinline__ void umma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "add.s64 x, %1, %5;\n\tadd.s64 y, %2, %8;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t"
      "add.s64 x, %1, %6;\n\tadd.s64 y, %2, %9;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t"
      "add.s64 x, %1, %7;\n\tadd.s64 y, %2, %10;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(ASTEP), "n"(2 * ASTEP), "n"(3 * ASTEP), "n"(BSTEP), "n"(2 * BSTEP),
        "n"(3 * BSTEP)
      : "memory");
}

// Thirty-two bytes, 32-byte aligned.
__device__ __forceinline__ void load32(const void* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}
// Eight neighbouring values, 32-byte aligned: a whole sector of L2 per thread, as neighbouring threads store to rows far apart.
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// A warp's 32 rows of 32 columns, a thread to a row as tensor memory hands them out, into rows of global memory: the eight threads of a
// group exchange their rows' pieces of 16 bytes (8 x 8 of them, in three steps), so that a store covers whole lines of 128 bytes.
// Thread-wise every store is 32 requests: 128 rows of 256 columns took 7500 cycles, 4600 so, of 32 live rows the other way 2000 and
// 3900.  `at`: this thread's row, < 0: none.
__device__ __forceinline__ void store_rows(float* base, long long at, uint32_t (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 1; m < 8; m *= 2) {
    const bool up = (lane & m) != 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((j & m) == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t &low = v[4 * j + e], &high = v[4 * (j | m) + e];
          const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? low : high, m);
          if (up) low = got;
          else high = got;
        }
      }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const long long row = __shfl_sync(0xffffffffu, at, (lane & 24) + j);
    if (row >= 0) *reinterpret_cast<uint4*>(base + row + 4 * (lane & 7)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
}

inline bool prefix_plan_ok(const ds41_prefix_plan* p) {
  return p != nullptr && p->units != nullptr && p->n_units != nullptr && p->turns != nullptr && p->order != nullptr && p->cell != nullptr &&
         p->owner != nullptr && p->parts != nullptr && p->part_o != nullptr && p->part_ml != nullptr && p->max_units > 0 && p->rows_per_unit > 0 &&
         p->grid > 0 && !(reinterpret_cast<uintptr_t>(p->units) & 15) && !(reinterpret_cast<uintptr_t>(p->part_o) & 31) &&
         !(reinterpret_cast<uintptr_t>(p->part_ml) & 7);
}

}  // namespace ds41
