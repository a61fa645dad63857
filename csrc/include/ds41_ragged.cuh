// What the kernels of ragged passes share (ragged.cu, ragged_attend.cu).
//
// The new tokens of a request are divided into blocks of `unit_tokens`; a unit is a block, a key/value head and a range of key tiles
// (a piece).  Softmax over a divided set of keys needs of every piece only its maximum m, its sum l = sum exp(s - m) and its
// unnormalised result o = sum exp(s - m) v: with M = max m_i the whole is sum exp(m_i - M) o_i / sum exp(m_i - M) l_i.  The CTA that
// finishes the last piece of a block and head joins them, in their order.
#pragma once
#include "ds41_stack.cuh"

namespace ds41 {

constexpr int kRaggedInts = 12;

struct RaggedUnit {
  int slot, row0, tokens, pos0, head, tile0, tiles, piece, pieces, cell, counter, step;
};
__device__ __forceinline__ RaggedUnit ragged_unit(const ds41_ragged_pass& p, int i) {
  const int4* u = reinterpret_cast<const int4*>(p.units + 1ll * i * kRaggedInts);
  const int4 a = u[0], b = u[1], c = u[2];
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
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

// Joins rows [r, n) of a block's pieces: a warp per (token, head) row, its lanes along the columns.
template <typename T>
__device__ __forceinline__ void ragged_join(const ds41_ragged_pass& p, const ds41_ragged_attend_args& a, const RaggedUnit& u, int r,
                                            int n, int warps) {
  const int lane = threadIdx.x & 31, group = p.heads / p.kv_heads;
  for (; r < n; r += warps) {
    const int row = u.row0 + r / group, h = u.head * group + r % group;
    float top = -INFINITY;
    for (int i = lane; i < u.pieces; i += 32) top = fmaxf(top, __ldcg(p.part_ml + 2 * (1ll * u.cell + 1ll * i * u.step + r)));
    top = warp_max(top);
    const float sink = a.sink != nullptr ? a.sink[h] * kLog2E : -INFINITY;
    const float whole = fmaxf(top, sink), base = whole == -INFINITY ? 0.f : whole;
    float den = 0.f;
    for (int i = lane; i < u.pieces; i += 32) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + (1ll * u.cell + 1ll * i * u.step + r));
      den += ml.x == -INFINITY ? 0.f : exp2f(ml.x - base) * ml.y;
    }
    den = warp_sum(den) + (a.sink != nullptr ? exp2f(sink - base) : 0.f);
    float f = 1.f / den;                                 // a NaN in a maximum or the sink is in the sum
    if (a.gate.data != nullptr) f *= sigmoid_f32(proj_at(a.gate, row, h));
    T* out = static_cast<T*>(a.out) + row * a.out_row + 1ll * h * p.vdim;
    for (int c = 4 * lane; c < p.vdim; c += 128) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < u.pieces; ++i) {
        const long long cell = 1ll * u.cell + 1ll * i * u.step + r;
        const float m = __ldcg(p.part_ml + 2 * cell);
        if (m == -INFINITY) continue;
        const float w = exp2f(m - base);
        const float4 v = ragged_part(p.part_o + cell * p.vdim + c);
        o.x += w * v.x;
        o.y += w * v.y;
        o.z += w * v.z;
        o.w += w * v.w;
      }
      store4(out + c, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
    }
  }
}

cudaError_t launch_ragged_tiled(const ds41_ragged_attend_args& a, const ds41_ragged_pass& p, cudaStream_t stream);

}  // namespace ds41
