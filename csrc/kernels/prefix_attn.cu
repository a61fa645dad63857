// Attention of rows that share prefixes: its parts for every type and size, and their join.
//
// A block takes sixteen queries (head and row) of a unit and walks its keys 32 at a time through shared memory, so that a cached
// value that was read once serves sixteen queries: scores by warps of 8 queries x 8 keys, or two pairs to a thread where a key has at most
// 64 values (32 bits, the first and the second: 6 rows of 16 heads over 500 keys of 576 values 23.9 and 29.8 us, of 48 values 28.5 and
// 25.3; 8 rows of 16 heads over 1000 keys of 128 values 21.8 and 22.3, of 32 values 22.5 and 19.3), a softmax state per query
// (running maximum and sum), results in registers.  A warp fetches four of the keys, whose places it looks up a tile ahead; values that
// are a part of their key (a latent) are fetched once.  It serves 32-bit rows and the sizes that the tensor-core forms
// (prefix_group.cu, prefix_latent.cu) leave out, and is bound by its 32-bit products and their operands from shared memory.
#include "ds41_group.cuh"
#include "ds41_prefix.cuh"
#include "ds41_tma.h"

namespace ds41 {

int launch_prefix_group(const ds41_group_attend_args& a, const ds41_prefix_plan& plan, cudaStream_t st);
int launch_prefix_latent(const ds41_latent_attend_args& a, const ds41_prefix_plan& plan, int n_pages, cudaStream_t st);

constexpr int kSimpleQueries = 16;
constexpr int kSimpleKeys = 32;
constexpr int kSimpleLd = kSimpleQueries + 4;      // of the weights: a key's lie side by side, four of them in one load

struct SimpleArgs {
  const void *q, *q2, *pool;         // a query is [d1 values of q | d2 of q2]
  const int *page_table, *row_pos, *row_slot;
  long long ld_q, ld_q2;
  int q_head, q2_head;               // values between a row's heads
  int d1, d2, vp, row_len;
  int k_lane, v_at, v_lane;          // key / value head g of a cache row: keys at g * k_lane, values at v_at + g * v_lane
  int inside;                        // the values are the first values of the key
  int per_lane, heads, chunk, max_pages, page_tokens, n_pages;
  float scale;
};

inline int simple_smem(const SimpleArgs& p) {
  const int dp = p.d1 + p.d2;
  return 4 * (kSimpleQueries * (dp + 4) + kSimpleKeys * (dp + 4) + (p.inside ? 0 : kSimpleKeys * p.vp) + kSimpleKeys * kSimpleLd) +
         16 * kSimpleQueries;
}

__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                     __uint_as_float(v.y & 0xffff0000u));
}

// QPT: queries whose columns a thread accumulates.  WIDE: rows of more than 64 values.
template <typename T, int QPT, bool WIDE>
__global__ void __launch_bounds__(256, QPT <= 4 ? 2 : 1) prefix_simple_kernel(const SimpleArgs p, const ds41_prefix_plan plan) {
  extern __shared__ __align__(16) float ps_smem[];
  const int dp = p.d1 + p.d2, ds = dp + 4, nc = p.vp / 4;
  float* qs = ps_smem;                                        // [16][ds]
  float* ks = qs + kSimpleQueries * ds;                       // [32][ds]
  float* vs = p.inside ? ks : ks + kSimpleKeys * ds;          // [32][vs_ld]
  const int vs_ld = p.inside ? ds : p.vp;
  float* sc = p.inside ? ks + kSimpleKeys * ds : vs + kSimpleKeys * p.vp;      // [32][20] scores, then weights
  float* ms = sc + kSimpleKeys * kSimpleLd;                   // [16] maxima
  float* ls = ms + kSimpleQueries;                            // [16] sums
  float* keep = ls + kSimpleQueries;                          // [16] factor on what was summed before
  int* lim = reinterpret_cast<int*>(keep + kSimpleQueries);   // [16] end of what a query sees
  __shared__ int low[kSimpleQueries], row_of[kSimpleQueries];
  __shared__ bool leased[kSimpleKeys];                        // a key without a page is not there
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int subs = (plan.rows_per_unit * p.per_lane + kSimpleQueries - 1) / kSimpleQueries;
  // every unit's first sixteen queries, then the second sixteen of those that have them: a block's next ones are not always the ones
  // that only full units have
  const int places = *plan.n_units;
  for (int unit = blockIdx.x; unit < places * subs; unit += gridDim.x) {
    const PrefixUnit it = prefix_unit(plan, unit % places);
    const int g = it.head, i0 = unit / places * kSimpleQueries, count = it.rows * p.per_lane;
    if (i0 >= count) continue;
    __syncthreads();                     // the last unit's shared memory is no longer read
    if (tid < kSimpleQueries) {
      int r = -1, lo = 0, hi = 0;
      if (i0 + tid < count) {
        r = prefix_row(plan, it, (i0 + tid) / p.per_lane);
        const int pos = p.row_pos[r];
        if (p.row_slot[r] >= 0) {
          lo = p.chunk > 0 ? pos - pos % p.chunk : 0;
          hi = min(pos + 1, it.key1);
        }
      }
      row_of[tid] = r;
      low[tid] = lo;
      lim[tid] = hi;
      ms[tid] = -INFINITY;
      ls[tid] = 0.f;
    }
    __syncthreads();
    for (int u = warp; u < kSimpleQueries; u += 8) {
      const int r = row_of[u], h = g * p.per_lane + (i0 + u) % p.per_lane;
      const T* q = static_cast<const T*>(p.q) + r * p.ld_q + 1ll * h * p.q_head;
      const T* q2 = static_cast<const T*>(p.q2) + r * p.ld_q2 + 1ll * h * p.q2_head - p.d1;
#pragma unroll 4
      for (int d = 4 * lane; d < dp; d += 128)
        *reinterpret_cast<float4*>(qs + u * ds + d) = r >= 0 ? four((d < p.d1 ? q : q2) + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    int from = INT_MAX, to = 0;
#pragma unroll
    for (int u = 0; u < kSimpleQueries; ++u) {
      if (low[u] < lim[u]) from = min(from, low[u]);
      to = max(to, lim[u]);
    }
    from = max(it.key0, from);
    float4 acc[QPT];
#pragma unroll
    for (int u = 0; u < QPT; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int col = tid % nc, u0 = tid / nc * QPT;
    auto row_at = [&](int key) {           // pool row of a key, -1: none
      const int pg = key / p.page_tokens;
      const int id = key >= from && key < to && pg < p.max_pages ? p.page_table[1ll * it.slot * p.max_pages + pg] : -1;
      return static_cast<unsigned>(id) < static_cast<unsigned>(p.n_pages) ? id * p.page_tokens + (key - pg * p.page_tokens) : -1;
    };
    int next = lane < 4 && from < to ? row_at(from + warp + 8 * lane) : -1;
    const T* pool_k = static_cast<const T*>(p.pool) + g * p.k_lane;
    const T* pool_v = static_cast<const T*>(p.pool) + p.v_at + g * p.v_lane;
    for (int t0 = from; t0 < to; t0 += kSimpleKeys) {
      __syncthreads();
      long long at[4];
      bool there[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = __shfl_sync(0xffffffffu, next, k);
        there[k] = row >= 0;
        at[k] = 1ll * row * p.row_len;
      }
      auto fetch = [&](const T* src, float* dst, int ld, int width) {
#pragma unroll 2
        for (int d = 4 * lane; d < width; d += 128) {
          float4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = there[k] ? four(src + at[k] + d) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < 4; ++k) *reinterpret_cast<float4*>(dst + (warp + 8 * k) * ld + d) = v[k];
        }
      };
      if (lane < 4) leased[warp + 8 * lane] = next >= 0;
      fetch(pool_k, ks, ds, dp);
      if (!p.inside) fetch(pool_v, vs, vs_ld, p.vp);
      next = lane < 4 ? row_at(t0 + kSimpleKeys + warp + 8 * lane) : -1;
      __syncthreads();
      if constexpr (!WIDE) {             // a thread's two keys of a query: narrow rows leave most lanes of the other form without columns
        const int u = tid >> 4, j = tid & 15;
        float a = 0.f, b = 0.f;
#pragma unroll 4
        for (int d = 0; d < dp; d += 4) {
          const float4 x = four(qs + u * ds + d), y = four(ks + j * ds + d), z = four(ks + (j + 16) * ds + d);
          a += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
          b += x.x * z.x + x.y * z.y + x.z * z.z + x.w * z.w;
        }
        const int key = t0 + j;
        sc[j * kSimpleLd + u] = leased[j] && key >= low[u] && key < lim[u] ? a * p.scale : -INFINITY;
        sc[(j + 16) * kSimpleLd + u] = leased[j + 16] && key + 16 >= low[u] && key + 16 < lim[u] ? b * p.scale : -INFINITY;
      } else {
        // a warp's 8 queries x 8 keys, the columns by lane: 16 loads for 256 products, then the lanes' sums are added and shared out
        const float *x = qs + (warp & 1) * 8 * ds, *y = ks + (warp >> 1) * 8 * ds;
        float s[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i] = 0.f;
#pragma unroll 1
        for (int d = 4 * lane; d < dp; d += 128) {
          float4 q[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) q[u] = four(x + u * ds + d);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 k = four(y + j * ds + d);
#pragma unroll
            for (int u = 0; u < 8; ++u) s[8 * u + j] += q[u].x * k.x + q[u].y * k.y + q[u].z * k.z + q[u].w * k.w;
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1)
#pragma unroll
          for (int i = 0; i < 2 * o; ++i) {
            const bool up = lane & o;
            const float mine = up ? s[i + 2 * o] : s[i], other = up ? s[i] : s[i + 2 * o];
            s[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
          }
        // this lane's: query lane / 4, keys 2 (lane % 4) and the next
        const int u = (warp & 1) * 8 + (lane >> 2), j = (warp >> 1) * 8 + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          sc[(j + i) * kSimpleLd + u] =
              leased[j + i] && t0 + j + i >= low[u] && t0 + j + i < lim[u] ? s[i] * p.scale : -INFINITY;
      }
      __syncthreads();
      for (int u = 2 * warp; u < 2 * warp + 2; ++u) {
        const float s = sc[lane * kSimpleLd + u], top = fmaxf(ms[u], warp_max(s));
        const float e = s == -INFINITY ? 0.f : expf(s - top);
        const float f = ms[u] == -INFINITY ? 0.f : expf(ms[u] - top), sum = warp_sum(e);
        __syncwarp();
        sc[lane * kSimpleLd + u] = e;
        if (lane == 0) {
          ls[u] = ls[u] * f + sum;
          ms[u] = top;
          keep[u] = f;
        }
      }
      __syncthreads();
      if (u0 < kSimpleQueries) {
#pragma unroll
        for (int u = 0; u < QPT; ++u) {
          const float f = keep[u0 + u];
          acc[u].x *= f;
          acc[u].y *= f;
          acc[u].z *= f;
          acc[u].w *= f;
        }
#pragma unroll 4
        for (int j = 0; j < kSimpleKeys; ++j) {
          const float4 v = four(vs + j * vs_ld + 4 * col);
          alignas(16) float w[QPT];
          if constexpr (QPT >= 4) {
#pragma unroll
            for (int u = 0; u < QPT; u += 4) *reinterpret_cast<float4*>(w + u) = four(sc + j * kSimpleLd + u0 + u);
          } else {
#pragma unroll
            for (int u = 0; u < QPT; ++u) w[u] = sc[j * kSimpleLd + u0 + u];
          }
#pragma unroll
          for (int u = 0; u < QPT; ++u)
            if (w[u] != 0.f) {           // what a query does not see may be anything
              acc[u].x += w[u] * v.x;
              acc[u].y += w[u] * v.y;
              acc[u].z += w[u] * v.z;
              acc[u].w += w[u] * v.w;
            }
        }
      }
    }
    __syncthreads();
    if (u0 < kSimpleQueries)
#pragma unroll
      for (int u = 0; u < QPT; ++u) {
        const int r = row_of[u0 + u];
        if (r < 0) continue;
        const int h = g * p.per_lane + (i0 + u0 + u) % p.per_lane;
        const long long cell = (1ll * plan.cell[r] + it.part) * p.heads + h;
        *reinterpret_cast<float4*>(plan.part_o + cell * p.vp + 4 * col) = acc[u];
        if (col == 0) *reinterpret_cast<float2*>(plan.part_ml + 2 * cell) = make_float2(ms[u0 + u] * 1.4426950408889634f, ls[u0 + u]);
      }
  }
}

template <typename T, int QPT, bool WIDE>
static int launch_simple(const SimpleArgs& p, const ds41_prefix_plan& plan, cudaStream_t st) {
  const int smem = simple_smem(p);
  if (smem > 220 * 1024) return cudaErrorInvalidValue;
  const cudaError_t e = cudaFuncSetAttribute(prefix_simple_kernel<T, QPT, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const long long most = 1ll * plan.max_units * ((plan.rows_per_unit * p.per_lane + kSimpleQueries - 1) / kSimpleQueries);
  const int blocks = static_cast<int>(most < 4 * sm_count() ? most : 4 * sm_count());
  return launch_pdl(prefix_simple_kernel<T, QPT, WIDE>, dim3(blocks), dim3(256), smem, st, p, plan);
}

template <typename T, bool WIDE>
static int dispatch_simple(const SimpleArgs& p, const ds41_prefix_plan& plan, cudaStream_t st) {
  const int nc = p.vp / 4;
  if (16 * nc <= 256) return launch_simple<T, 1, WIDE>(p, plan, st);
  if (8 * nc <= 256) return launch_simple<T, 2, WIDE>(p, plan, st);
  if (4 * nc <= 256) return launch_simple<T, 4, WIDE>(p, plan, st);
  if (2 * nc <= 256) return launch_simple<T, 8, WIDE>(p, plan, st);
  if (nc <= 256) return launch_simple<T, 16, WIDE>(p, plan, st);
  return cudaErrorInvalidValue;
}

static int run_simple(const SimpleArgs& p, const ds41_prefix_plan& plan, int f32, cudaStream_t st) {
  // rows of four values at a time
  if ((p.ld_q & 3) || (p.ld_q2 & 3) || (p.q_head & 3) || (p.q2_head & 3) || (p.row_len & 3) || (p.d1 & 3) || (p.d2 & 3) || (p.vp & 3) ||
      ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.q2) | reinterpret_cast<uintptr_t>(p.pool)) & (f32 ? 15 : 7)))
    return cudaErrorInvalidValue;
  if (p.d1 + p.d2 > 64) return f32 ? dispatch_simple<float, true>(p, plan, st) : dispatch_simple<__nv_bfloat16, true>(p, plan, st);
  return f32 ? dispatch_simple<float, false>(p, plan, st) : dispatch_simple<__nv_bfloat16, false>(p, plan, st);
}

// A warp joins 128 columns of a (row, head): the lanes find the parts' weights, then every lane sums four columns over the parts, PARTS
// of them under way together.  Rows without a slot become zero; rows of another slot than the plan's become NaN and are reported.
// The launch also keeps the convolution's last inputs where the attention has one (ds41_group.cuh).
// A chain of loads from L2: small launches want many of them under way (101 registers), large ones many warps (56).  Whole calls with 8 / 4
// parts: 37 rows of 6 heads in 13 parts 15.7 / 18.3 us, 32 rows of 32 heads 22.8 / 24.5 (1024 warps); 32 rows x 32 heads x 512 columns
// (4096 warps) 33.0 / 31.6 us, 128 rows (16384) 214 / 207.
template <typename T, int PARTS>
__global__ void __launch_bounds__(128, PARTS == 8 ? 1 : 9)
prefix_join_kernel(const ds41_prefix_plan plan, const float* sink, const ds41_proj gate, int rows, int heads, int vp, T* out, int ld_out,
                   const ds41_group_attend_args keep) {
  const int lane = threadIdx.x & 31, strips = (vp + 127) / 128;
  const unsigned w = 4 * blockIdx.x + (threadIdx.x >> 5);
  const unsigned pair = w / strips;
  const int r = pair / heads, h = pair % heads, c = (w - pair * strips) * 128 + 4 * lane;
  pdl_launch_dependents();
  // the plan was copied to the device, not computed there: it may be read before the wait
  const int n = r < rows ? plan.parts[r] : 0, owner = r < rows ? plan.owner[r] : 0;
  const long long cell = r < rows ? 1ll * plan.cell[r] * heads + h : 0;
  pdl_wait();
  if (r >= rows) return;
  const int slot = keep.row_slot[r];
  // a row of another slot than the one that the plan holds its keys for: no result is right
  const bool stray = slot >= 0 && slot + 1 != owner;
  if (stray && w % (heads * strips) == 0 && lane == 0 && keep.status != nullptr &&
      atomicCAS(keep.status, kStatusOk, kStatusBadArgument) == kStatusOk) {
    keep.status[1] = 540;
    keep.status[2] = r;
    keep.status[3] = slot;
  }
  // parts of a row without a slot are empty, so that its sum stays zero; that of a stray one becomes NaN
  const float sk = stray ? NAN : sink != nullptr && slot >= 0 ? sink[h] * 1.4426950408889634f : -INFINITY;
  if (keep.taps > 1 && slot >= 0)
    keep_inputs(keep, r, slot, keep.row_pos[r], w % (heads * strips), heads * strips, lane, 32);
  const float2* ml = reinterpret_cast<const float2*>(plan.part_ml) + cell;
  const float* part = plan.part_o + cell * vp + c;
  const long long step = 1ll * heads * vp;
  float2 mine = lane < n ? ml[1ll * lane * heads] : make_float2(-INFINITY, 0.f);
  float all = fmaxf(sk, mine.x);
  for (int s = lane + 32; s < n; s += 32) all = fmaxf(all, ml[1ll * s * heads].x);
  all = warp_max(all);
  float den = lane > 0 || sk == -INFINITY ? 0.f : exp2f(sk - all);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < n; s0 += 32) {
    if (s0 > 0) mine = s0 + lane < n ? ml[1ll * (s0 + lane) * heads] : make_float2(-INFINITY, 0.f);
    const float e = mine.x > -INFINITY ? exp2f(mine.x - all) : 0.f;
    den += e * mine.y;
    for (int k0 = 0; k0 < 32 && s0 + k0 < n; k0 += PARTS) {
      float4 o[PARTS];
      float f[PARTS];
#pragma unroll
      for (int k = 0; k < PARTS; ++k) {
        f[k] = __shfl_sync(0xffffffffu, e, k0 + k);
        // a part without a weight may hold anything: nothing may have been written
        if (f[k] > 0.f && c < vp) o[k] = *reinterpret_cast<const float4*>(part + (s0 + k0 + k) * step);
      }
#pragma unroll
      for (int k = 0; k < PARTS; ++k)
        if (f[k] > 0.f && c < vp) {
          a.x += f[k] * o[k].x;
          a.y += f[k] * o[k].y;
          a.z += f[k] * o[k].z;
          a.w += f[k] * o[k].w;
        }
    }
  }
  den = warp_sum(den);
  // nothing seen: zeros, whatever the gate is; a NaN among the scores left its part a sum of NaN, whatever the maximum was
  const float f = den > 0.f ? (gate.data != nullptr ? sigmoid_f32(proj_at(gate, r, h)) : 1.f) * (1.0f / den) : den;
  if (c < vp) store4(out + 1ll * r * ld_out + h * vp + c, make_float4(a.x * f, a.y * f, a.z * f, a.w * f));
}

template <typename T>
static int launch_join(const ds41_prefix_plan& plan, const float* sink, const ds41_proj& gate, int rows, int heads, int vp, void* out,
                       int ld_out, const ds41_group_attend_args& keep, cudaStream_t st) {
  const long long warps = 1ll * rows * heads * ((vp + 127) / 128);
  if (warps >= 1ll << 31) return cudaErrorInvalidValue;
  return launch_pdl(warps < 20 * sm_count() ? prefix_join_kernel<T, 8> : prefix_join_kernel<T, 4>,
                    dim3(static_cast<unsigned>((warps + 3) / 4)), dim3(128), 0, st, plan, sink, gate, rows, heads, vp, static_cast<T*>(out),
                    ld_out, keep);
}

}  // namespace ds41

using namespace ds41;

extern "C" int ds41_prefix_group(const ds41_group_attend_args* a, const ds41_prefix_plan* plan, void* stream) {
  if (!prefix_plan_ok(plan) || !group_attend_ok(a) || a->n_pages <= 0 ||
      1ll * a->n_pages * a->page_tokens >= 1ll << 31 || (a->ld_out & 3) || (reinterpret_cast<uintptr_t>(a->out) & (a->f32 ? 15 : 7)))
    return cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int e = launch_prefix_group(*a, *plan, st);
  if (e == cudaErrorNotSupported) {
    SimpleArgs p{};
    p.q = a->q; p.q2 = a->q; p.pool = a->pool;
    p.page_table = a->page_table; p.row_pos = a->row_pos; p.row_slot = a->row_slot;
    p.ld_q = a->ld_q; p.q_head = a->dim_pad; p.d1 = a->dim_pad; p.vp = a->vdim_pad;
    p.row_len = a->kv_heads * (a->dim_pad + a->vdim_pad);
    p.k_lane = a->dim_pad; p.v_at = a->kv_heads * a->dim_pad; p.v_lane = a->vdim_pad;
    p.per_lane = a->heads / a->kv_heads; p.heads = a->heads;
    p.chunk = a->chunk; p.max_pages = a->max_pages; p.page_tokens = a->page_tokens; p.n_pages = a->n_pages;
    p.scale = a->scale;
    e = run_simple(p, *plan, a->f32, st);
  }
  if (e != cudaSuccess) return e;
  return a->f32 ? launch_join<float>(*plan, nullptr, a->gate, a->rows, a->heads, a->vdim_pad, a->out, a->ld_out, *a, st)
                : launch_join<__nv_bfloat16>(*plan, nullptr, a->gate, a->rows, a->heads, a->vdim_pad, a->out, a->ld_out, *a, st);
}

extern "C" int ds41_prefix_latent(const ds41_latent_attend_args* a, const ds41_prefix_plan* plan, int n_pages, const float* sink, void* out,
                                  int ld_out, void* stream) {
  if (!prefix_plan_ok(plan) || a == nullptr || a->rows <= 0 || a->heads <= 0 || a->heads > 65535 || a->kv_pad <= 0 || (a->kv_pad & 3) ||
      a->row_len < a->kv_pad || (a->row_len & 3) || n_pages <= 0 || a->max_pages <= 0 || a->page_tokens <= 0 ||
      1ll * n_pages * a->page_tokens >= 1ll << 31 || a->q_abs == nullptr ||
      (a->row_len > a->kv_pad && a->q_rot == nullptr) || a->pool == nullptr || a->page_table == nullptr || a->row_pos == nullptr ||
      a->row_slot == nullptr || out == nullptr || ld_out < a->heads * a->kv_pad || (ld_out & 3) ||
      (reinterpret_cast<uintptr_t>(out) & (a->f32 ? 15 : 7)))
    return cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int e = launch_prefix_latent(*a, *plan, n_pages, st);
  if (e == cudaErrorNotSupported) {
    SimpleArgs p{};
    p.q = a->q_abs; p.q2 = a->q_rot; p.pool = a->pool;
    p.page_table = a->page_table; p.row_pos = a->row_pos; p.row_slot = a->row_slot;
    p.ld_q = a->ld_q_abs; p.q_head = a->kv_pad; p.ld_q2 = a->ld_q_rot; p.q2_head = a->q_rot_stride;
    p.d1 = a->kv_pad; p.d2 = a->row_len - a->kv_pad; p.vp = a->kv_pad; p.row_len = a->row_len;
    p.per_lane = a->heads; p.heads = a->heads; p.inside = 1;
    p.max_pages = a->max_pages; p.page_tokens = a->page_tokens; p.n_pages = n_pages;
    p.scale = a->scale;
    e = run_simple(p, *plan, a->f32, st);
  }
  if (e != cudaSuccess) return e;
  const ds41_proj none{};
  ds41_group_attend_args keep{};
  keep.taps = 1;
  keep.row_slot = a->row_slot;
  keep.status = a->status;
  return a->f32 ? launch_join<float>(*plan, sink, none, a->rows, a->heads, a->kv_pad, out, ld_out, keep, st)
                : launch_join<__nv_bfloat16>(*plan, sink, none, a->rows, a->heads, a->kv_pad, out, ld_out, keep, st);
}
