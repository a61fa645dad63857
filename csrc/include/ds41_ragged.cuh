// What the kernels of ragged passes share (ragged.cu, ragged_attend.cu).
//
// The new tokens of a request are divided into blocks of `unit_tokens`; a unit is a block, a key/value head (or half of its values'
// columns) and a range of key tiles (a piece).  Softmax over a divided set of keys needs of every piece only its maximum m, its sum
// l = sum exp(s - m) and its unnormalised result o = sum exp(s - m) v: with M = max m_i the whole is sum exp(m_i - M) o_i /
// sum exp(m_i - M) l_i.  The CTA that finishes the last piece of a block and head joins them, in their order.
//
// The result of a token that has no place in the cache, as its page is not leased, is zeros: the heads' kernel has no query of it, and what
// lies in its place may be of another pass.
#pragma once
#include "ds41_stack.cuh"

namespace ds41 {

constexpr int kRaggedInts = 12;

struct RaggedUnit {
  int slot, row0, tokens, pos0, head, tile0, tiles, piece, pieces, cell, counter, step;
  int v0;                    // its first column of a value
};
__device__ __forceinline__ RaggedUnit ragged_unit(const ds41_ragged_pass& p, int i) {
  const int4* u = reinterpret_cast<const int4*>(p.units + 1ll * i * kRaggedInts);
  const int4 a = u[0], b = u[1], c = u[2];
  const int half = b.x & (p.v_parts - 1);
  return {a.x, a.y, a.z, a.w, b.x >> (p.v_parts - 1), b.y, b.z, b.w, c.x, c.y, c.z, c.w, half * (p.vdim >> 1)};
}

// First position that a row at `pos` sees behind the first tokens.
__host__ __device__ __forceinline__ int ragged_low(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }

// The keys that rows at p0 .. p1 see, as one row of places: the first `lead` of them are positions 0 .. lead - 1, place v behind them is
// position v + shift.  Places come in runs, within which positions follow one another and lie in one page.  A range of first
// tokens that reaches the window is a part of it.
struct RaggedWalk {
  int lead, shift, places;
};
struct Runs {                // of a power of two
  int mask;
  __device__ __forceinline__ int down(int x) const { return x & ~mask; }
  __device__ __forceinline__ int up(int x) const { return (x + mask) & ~mask; }
};
struct AnyRuns {
  int align;
  __device__ __forceinline__ int down(int x) const { return x - x % align; }
  __device__ __forceinline__ int up(int x) const { return (x + align - 1) / align * align; }
};
template <typename R>
__device__ __forceinline__ RaggedWalk ragged_walk(int p0, int p1, int window, int first, R runs) {
  int base = runs.down(ragged_low(p0, window));
  const int f = first < p1 + 1 ? first : p1 + 1;
  int lead = f > 0 ? runs.up(f) : 0;
  if (lead >= base) {
    if (lead > 0) base = 0;
    lead = 0;
  }
  return {lead, base - lead, lead + p1 + 1 - base};
}

// Counts a finished piece; true in the whole group if it was the last one.  Every thread of the group (barrier `id`, `threads` of them) has
// stored its part.
__device__ __forceinline__ bool ragged_last(unsigned int* counter, int pieces, bool first_thread, int id, int threads, volatile int* flag) {
  __threadfence();
  named_barrier(id, threads);
  if (first_thread) {
    const bool last = atomicAdd(counter, 1u) + 1 == static_cast<unsigned>(pieces);
    if (last) *counter = 0;
    *flag = last;
  }
  named_barrier(id, threads);
  const bool last = *flag != 0;
  if (last) __threadfence();
  named_barrier(id, threads);
  return last;
}

__device__ __forceinline__ float4 ragged_part(const float* p) { return __ldcg(reinterpret_cast<const float4*>(p)); }

constexpr float kLog2E = 1.4426950408889634f;

// Joins rows [r, n) of a block's pieces, the rows of warp `warp` of `warps`: 8, 16 or 32 lanes to a (token, head) row, along the pieces for
// their maxima and sums, and along the columns for their results, eight pieces' at a time; the next row's maxima are under way meanwhile.
// One row and one load after another, nine pieces of 63 rows of 48 columns took 28 us; 5 so.
template <typename T>
__device__ __forceinline__ void ragged_join(const ds41_ragged_pass& p, const ds41_ragged_attend_args& a, const RaggedUnit& u, int r0,
                                            int n, int warp, int warps) {
  const int vp = p.vdim / p.v_parts, span = vp <= 32 ? 8 : vp <= 64 ? 16 : 32;
  const int lane = threadIdx.x & (span - 1), from_lane = threadIdx.x & 31 & ~(span - 1);
  const int group = p.heads / p.kv_heads, step = warps * (32 / span);
  auto ml_at = [&](int r, int i) {
    return r < n && i < u.pieces ? __ldcg(reinterpret_cast<const float2*>(p.part_ml) + (1ll * u.cell + 1ll * i * u.step + r))
                                 : make_float2(-INFINITY, 0.f);
  };
  r0 += warp * (32 / span);                              // the warp's first row
  int r = r0 + from_lane / span;
  float2 next = ml_at(r, lane);
  float next_gate = 0.f, next_sink = -INFINITY;
  int next_place = -1;
  auto head_of = [&](int r) {                            // rows from n on have nothing, and are not stored
    const int row = u.row0 + min(r, n - 1) / group, h = u.head * group + r % group;
    next_place = p.row_place[row];
    if (a.gate.data != nullptr) next_gate = proj_at(a.gate, row, h);
    if (a.sink != nullptr) next_sink = a.sink[h];
  };
  head_of(r);
  for (; r0 < n; r0 += step, r += step) {
    const float2 ml = next;                              // of the first pieces
    const float gate = next_gate, sink = next_sink * kLog2E;
    const bool placed = next_place >= 0;
    next = ml_at(r + step, lane);
    head_of(r + step);
    const int row = u.row0 + min(r, n - 1) / group, h = u.head * group + r % group;
    float top = ml.x;
    for (int i = lane + span; i < u.pieces; i += span) top = fmaxf(top, ml_at(r, i).x);
    for (int o = span / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float whole = fmaxf(top, sink), base = whole == -INFINITY ? 0.f : whole;
    auto weight = [&](float2 x) { return x.x == -INFINITY ? 0.f : exp2f(x.x - base); };
    float den = weight(ml) * ml.y;
    for (int i = lane + span; i < u.pieces; i += span) {
      const float2 x = ml_at(r, i);
      den += weight(x) * x.y;
    }
    for (int o = span / 2; o; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    den += a.sink != nullptr ? exp2f(sink - base) : 0.f;
    float f = 1.f / den;                                 // a NaN in a maximum or the sink is in the sum
    if (a.gate.data != nullptr) f *= sigmoid_f32(gate);
    T* out = static_cast<T*>(a.out) + row * a.out_row + 1ll * h * p.vdim + u.v0;
    for (int c0 = 0; c0 < vp; c0 += 4 * span) {
      const int c = c0 + 4 * lane;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i0 = 0; i0 < u.pieces; i0 += span) {
        const float2 x = i0 == 0 ? ml : ml_at(r, i0 + lane);
        const unsigned there = __ballot_sync(0xffffffffu, x.x != -INFINITY) >> from_lane;      // others saw nothing and left nothing
        const float w = weight(x);
        const float* from = p.part_o + (1ll * u.cell + 1ll * i0 * u.step + r) * vp + c;
#pragma unroll 1
        for (int j = 0; j < min(span, u.pieces - i0); j += 8) {
          float4 v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            v[k] = c < vp && there >> (j + k) & 1 ? ragged_part(from + 1ll * (j + k) * u.step * vp) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float wk = __shfl_sync(0xffffffffu, w, from_lane + j + k);
            o.x += wk * v[k].x;
            o.y += wk * v[k].y;
            o.z += wk * v[k].z;
            o.w += wk * v[k].w;
          }
        }
      }
      if (c < vp && r < n) store4(out + c, placed ? make_float4(o.x * f, o.y * f, o.z * f, o.w * f) : make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
}

cudaError_t launch_ragged_tiled(const ds41_ragged_attend_args& a, const ds41_ragged_pass& p, cudaStream_t stream);

}  // namespace ds41
