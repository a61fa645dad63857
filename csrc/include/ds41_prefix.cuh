// What the kernels of attention over a shared prefix share (prefix_attn.cu, prefix_group.cu, prefix_latent.cu, and the forms of
// group_attn.cu / latent_attn.cu that finish it).
//
// Row r's keys are divided at own[r], a multiple of the page size: the positions below it lie in pages that several requests' page
// tables begin with, and are read once for all of them; the row reads the others by itself.  Softmax over a divided set of keys
// needs of every part only its maximum m, its sum l = sum exp(s - m) and its unnormalised result o = sum exp(s - m) v: with
// M = max m_i the whole is sum exp(m_i - M) o_i / sum exp(m_i - M) l_i.
//
// The plan is made on the host from the page tables (ops/prefix.py).  An item is a range of keys of one prefix and some of the
// rows that share it; the parts of row r are the cells cell[r] .. cell[r] + parts[r] - 1 of [cell][head].
#pragma once
#include <type_traits>

#include "ds41_stack.cuh"

namespace ds41 {

struct PrefixItem {
  int slot, first, rows, key0, key1, split;      // rows order[first] .. of the pass; keys [key0, key1) of the slot's page table
};
constexpr int kItemInts = 8;

__device__ __forceinline__ PrefixItem prefix_item(const ds41_prefix_plan& p, int i) {
  const int4 a = *reinterpret_cast<const int4*>(p.items + 1ll * i * kItemInts);
  const int2 b = *reinterpret_cast<const int2*>(p.items + 1ll * i * kItemInts + 4);
  return {a.x, a.y, a.z, a.w, b.x, b.y};
}

// a launch without a prefix
struct NoPrefix {};
template <typename X>
constexpr bool kHasPrefix = !std::is_same<X, NoPrefix>::value;

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

// Eight neighbouring values, 32-byte aligned: a whole sector of L2 per thread, as neighbouring threads store to rows far apart.
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

inline bool prefix_plan_ok(const ds41_prefix_plan* p) {
  return p != nullptr && p->items != nullptr && p->n_items != nullptr && p->order != nullptr && p->own != nullptr &&
         p->cell != nullptr && p->parts != nullptr && p->part_o != nullptr && p->part_ml != nullptr && p->max_items > 0 &&
         p->rows_per_item > 0 && p->grid > 0 && !(reinterpret_cast<uintptr_t>(p->items) & 15) &&
         !(reinterpret_cast<uintptr_t>(p->part_o) & 31) && !(reinterpret_cast<uintptr_t>(p->part_ml) & 7);
}

}  // namespace ds41
