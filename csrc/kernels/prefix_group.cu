// Grouped-query attention over the common keys of rows that share a prefix, on tcgen05.
//
// The queries of one key/value head are packed: (row, head) pairs of an item's rows are the 128 rows of a tensor-core tile, so that a
// tile of keys and values is read once for all of them and the products have the shape of a prompt's.  A CTA has two tiles:
//   more than 128 queries : two tiles of queries that walk the same keys;
//   up to 128             : the same queries twice, over the even and the odd tiles of keys, joined through tensor memory at the end.
// Either way one tile's softmax runs while the tensor core works on the other's products.
//   warps 0-3, 4-7 : queries into shared memory, softmax of tile 0 / 1 (one thread per query), partial results
//   warp 8         : TMA producer: key and value tiles of 128 positions, page by page, into rings of stages
//   warp 9         : tcgen05.mma issue: S = Q K^T into TMEM, O += P V with P in TMEM where it replaces its S
// The running maximum is raised when it grew by more than 2^8 only; what leaves is (m, l, unnormalised O) in 32 bits.  P is rounded
// to bf16 as the operand of the second product; l sums the unrounded weights.
#include <cuda.h>

#include "ds41_group.cuh"
#include "ds41_prefix.cuh"
#include "ds41_tma.h"

namespace ds41 {

constexpr int kPgThreads = 320;
constexpr int kPgTile = 128;                   // queries per tile, keys per tile
constexpr int kPgChunk = kPgTile * 128;        // bytes of 128 rows x 64 bf16 columns

struct PrefixGroupParams {
  const __nv_bfloat16* q;
  const int *page_table, *row_pos, *row_slot;
  long long ld_q;
  int heads, kv_heads, n, dp, vp, kd, vc, k_stages, v_stages;
  int chunk, max_pages, page_tokens, box, hidden_row;      // a row beyond the pool: reads as zeros
  float scale_log2;
  int* status;
};

__global__ void __launch_bounds__(kPgThreads, 1)
prefix_group_kernel(const __grid_constant__ CUtensorMap pool, const PrefixGroupParams p, const ds41_prefix_plan plan) {
  extern __shared__ uint8_t pg_raw[];
  uint8_t* smem = pg_raw + ((1024u - (smem_u32(pg_raw) & 1023u)) & 1023u);
  const int q_bytes = p.kd * kPgChunk, k_bytes = q_bytes, v_bytes = p.vc * kPgChunk;
  uint8_t* s_q = smem;                                   // two tiles
  uint8_t* s_k = s_q + 2 * q_bytes;
  uint8_t* s_v = s_k + p.k_stages * k_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_v + p.v_stages * v_bytes);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;        // [2]
  uint64_t* k_empty = bars + 3;
  uint64_t* v_full = bars + 5;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 9;        // [2] per tile: S complete (and every earlier MMA of the issuing thread)
  uint64_t* p_full = bars + 11;       // [2] per tile: P written, O rescaled
  uint64_t* o_full = bars + 13;       // [2] per tile: the unit's last product
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
  int* s_row = reinterpret_cast<int*>(bars + 16);        // [256] pass row of a packed query, -1: none
  float2* s_ml = reinterpret_cast<float2*>(s_row + 2 * kPgTile);      // [2][128]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    mbar_init(q_full, 2 * kPgTile);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kPgTile);
      mbar_init(&o_full[i], 1);
    }
    mbar_init_fence();
    tma_prefetch_desc(&pool);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const int units = *plan.n_items * p.kv_heads;
  // keys [first, first + 128 tiles) that an item's rows walk: a chunk's border may lie inside (whole warps)
  auto span = [&](const PrefixItem& it, int& first) {
    first = it.key0;
    if (p.chunk > 0) {
      int low = it.key1;
      for (int i = lane; i < it.rows; i += 32) low = min(low, chunk_start(p.row_pos[plan.order[it.first + i]], p.chunk));
#pragma unroll
      for (int o = 16; o; o >>= 1) low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
      first = max(first, low - low % p.page_tokens);
    }
    return first < it.key1 ? (it.key1 - first + kPgTile - 1) / kPgTile : 0;
  };

  if (warp == 8) {
    const int boxes = kPgTile / p.box;
    int kt = 0;                                          // key tiles so far: key and value rings
    bool ok = true;
    for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x) {
      const PrefixItem it = prefix_item(plan, unit / p.kv_heads);
      const int g = unit % p.kv_heads;
      int first;
      const int n = span(it, first);
      const int* table = p.page_table + 1ll * it.slot * p.max_pages;
      int row = 0, u = 0, u_row = 0;                     // lane i: pool row of box i of the walk, 32 boxes at a time
      for (int j = 0; j < n && ok; ++j, ++kt) {
        int at[16];                                      // this tile's boxes (at most 128 / 8)
        auto locate = [&](int i) {
          if ((u & 31) == 0) {
            const int key = first + (u + lane) * p.box, pg = key / p.page_tokens;
            const int id = key < it.key1 && pg < p.max_pages ? table[pg] : -1;
            row = id >= 0 ? id * p.page_tokens + (key - pg * p.page_tokens) : p.hidden_row;
          }
          u_row = __shfl_sync(0xffffffffu, row, u & 31);
          ++u;
          return u_row;
        };
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < boxes) at[i] = locate(i);
        const int ks = kt % p.k_stages, vs = kt % p.v_stages;
        ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[ks], ((kt / p.k_stages) & 1) ^ 1, p.status, 460)) != 0;
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(&k_full[ks], k_bytes);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i < boxes)
              for (int c = 0; c < p.kd; ++c)
                tma_load_3d(s_k + ks * k_bytes + c * kPgChunk + i * p.box * 128, &pool, &k_full[ks], g * p.dp + 64 * c, at[i], 0);
        }
        __syncwarp();
        ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[vs], ((kt / p.v_stages) & 1) ^ 1, p.status, 461)) != 0;
        if (!ok) {
          ++kt;
          break;
        }
        if (lane == 0) {
          mbar_expect_tx(&v_full[vs], v_bytes);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i < boxes)
              for (int c = 0; c < p.vc; ++c)
                tma_load_3d(s_v + vs * v_bytes + c * kPgChunk + i * p.box * 128, &pool, &v_full[vs],
                            p.kv_heads * p.dp + g * p.vp + 64 * c, at[i], 0);
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) {
      // something else gave up: let the copies under way land before the shared memory goes away
      for (int b = max(0, kt - 2); b < kt; ++b) {
        for (int i = 0; i < (1 << 20) && !mbar_test_wait(&k_full[b % p.k_stages], (b / p.k_stages) & 1); ++i) {
        }
        for (int i = 0; i < (1 << 20) && !mbar_test_wait(&v_full[b % p.v_stages], (b / p.v_stages) & 1); ++i) {
        }
      }
    }
  } else if (warp == 9) {
    const bool leader = elect_one();
    const uint32_t idesc_s = umma_idesc(kPgTile, kPgTile, 1u, 1u);
    const uint32_t idesc_pv = umma_idesc_bmn(kPgTile, p.vp, 1u, 1u);
    const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q)), k_desc = umma_desc_sw128(smem_u32(s_k));
    const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(s_v), kPgChunk, 1024);
    const int kd16 = p.dp / 16;
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      const bool ok = mbar_wait(bar, parity, p.status, where);
      return __all_sync(0xffffffffu, ok) != 0;
    };
    auto issue_s = [&](int t, int q_tile, int stage) {
      const uint64_t qd = q_desc + static_cast<uint64_t>(q_tile * q_bytes / 16);
      const uint64_t kd = k_desc + static_cast<uint64_t>(stage * k_bytes / 16);
      for (int k = 0; k < kd16; ++k) {
        const uint64_t off = static_cast<uint64_t>((k >> 2) * (kPgChunk / 16) + (k & 3) * 2);
        umma_bf16_if(leader, tmem + t * 128, qd + off, kd + off, idesc_s, k > 0 ? 1u : 0u);
      }
      tc_commit_if(leader, &s_full[t]);
    };
    auto issue_pv = [&](int t, int stage, bool first) {
      const uint64_t vd = v_desc + static_cast<uint64_t>(stage * v_bytes / 16);
#pragma unroll
      for (int k = 0; k < kPgTile / 16; ++k)
        umma_bf16_ts_if(leader, tmem + 256 + t * 128, tmem + t * 128 + 8 * k, vd + 128 * k, idesc_pv, first && k == 0 ? 0u : 1u);
    };
    bool ok = true;
    int kt = 0, done[2] = {0, 0}, live = 0;              // key tiles; products of each tile; units with work so far
    for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x) {
      const PrefixItem it = prefix_item(plan, unit / p.kv_heads);
      int first;
      const int n = span(it, first);
      if (n == 0) continue;
      ok = wait(q_full, live & 1, 470);
      ++live;
      if (!ok) break;
      tc_fence_after();
      auto key_ready = [&](int j) { return wait(&k_full[(kt + j) % p.k_stages], ((kt + j) / p.k_stages) & 1, 471); };
      auto value_ready = [&](int j) { return wait(&v_full[(kt + j) % p.v_stages], ((kt + j) / p.v_stages) & 1, 472); };
      if (it.rows * p.n > kPgTile) {
        ok = key_ready(0);
        if (!ok) break;
        tc_fence_after();
        issue_s(0, 0, kt % p.k_stages);
        issue_s(1, 1, kt % p.k_stages);
        tc_commit_if(leader, &k_empty[kt % p.k_stages]);
        for (int j = 0; j < n && ok; ++j) {
          const int vs = (kt + j) % p.v_stages, ks = (kt + j + 1) % p.k_stages;
          ok = value_ready(j);
          if (ok && j + 1 < n) ok = key_ready(j + 1);
          if (!ok) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok) ok = wait(&p_full[t], done[t] & 1, 473 + t);
            if (!ok) break;
            ++done[t];
            tc_fence_after();
            issue_pv(t, vs, j == 0);
            if (j == n - 1) tc_commit_if(leader, &o_full[t]);
            if (t == 1) tc_commit_if(leader, &v_empty[vs]);
            if (j + 1 < n) issue_s(t, t, ks);
          }
          if (ok && j + 1 < n) tc_commit_if(leader, &k_empty[ks]);
        }
      } else {
        for (int j = 0; j < 2 && j < n && ok; ++j) {
          ok = key_ready(j);
          if (!ok) break;
          tc_fence_after();
          issue_s(j, 0, (kt + j) % p.k_stages);
          tc_commit_if(leader, &k_empty[(kt + j) % p.k_stages]);
        }
        for (int j = 0; j < n && ok; ++j) {
          const int t = j & 1, vs = (kt + j) % p.v_stages;
          ok = value_ready(j) && wait(&p_full[t], done[t] & 1, 473 + t);
          if (!ok) break;
          ++done[t];
          tc_fence_after();
          issue_pv(t, vs, j < 2);
          if (j + 2 >= n) tc_commit_if(leader, &o_full[t]);
          tc_commit_if(leader, &v_empty[vs]);
          if (j + 2 < n) {
            ok = key_ready(j + 2);
            if (!ok) break;
            tc_fence_after();
            issue_s(t, 0, (kt + j + 2) % p.k_stages);
            tc_commit_if(leader, &k_empty[(kt + j + 2) % p.k_stages]);
          }
        }
      }
      kt += n;
    }
  } else {
    const int t = warp >> 2, quad = warp & 3, tid = threadIdx.x, mine = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_t = tmem + lanes + t * 128, o_t = tmem + lanes + 256 + t * 128;
    int tiles = 0, outs[2] = {0, 0};                     // tiles of S seen by this half; finished results of both
    bool ok = true;
    // the loop runs to its end whatever happened: its barriers are for all eight warps
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
      const PrefixItem it = prefix_item(plan, unit / p.kv_heads);
      const int g = unit % p.kv_heads, count = it.rows * p.n;
      const bool both = count <= kPgTile;                // the same queries in both tiles
      int first;
      const int n = span(it, first);
      const int mine_q = both ? mine : t * kPgTile + mine;
      int r = -1, lo = 0, hi = 0;
      if (mine_q < count) {
        r = plan.order[it.first + mine_q / p.n];
        const int pos = p.row_pos[r];
        if (p.row_slot[r] >= 0) {
          lo = chunk_start(pos, p.chunk);
          hi = min(min(plan.own[r], pos + 1), it.key1);
        }
      }
      s_row[t * kPgTile + mine] = r;                     // equal in both halves where the queries are
      named_barrier(1, 2 * kPgTile);
      if (n > 0) {
        const int pieces = p.dp / 8, q_tiles = both ? 1 : 2;
        for (int i = tid; i < q_tiles * kPgTile * pieces; i += 2 * kPgTile) {
          const int x = i / pieces, c = i % pieces, row = s_row[x], y = x & (kPgTile - 1);
          uint4 v = make_uint4(0, 0, 0, 0);
          if (row >= 0) v = *reinterpret_cast<const uint4*>(p.q + row * p.ld_q + 1ll * (g * p.n + x % p.n) * p.dp + 8 * c);
          *reinterpret_cast<uint4*>(s_q + (x >> 7) * q_bytes + (c >> 3) * kPgChunk + y * 128 + (((c & 7) ^ (y & 7)) << 4)) = v;
        }
        fence_async_smem();
        mbar_arrive(q_full);
      }
      // limits of the warp's queries: tiles between them need no look at single keys
      int low = hi > lo ? lo : 0, high = hi > lo ? hi : 0x7fffffff;
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        low = max(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = min(high, __shfl_xor_sync(0xffffffffu, high, o));
      }
      float m = -INFINITY, l = 0.f;
      const int step = both ? 2 : 1, from = both ? t : 0;
      for (int j = from; j < n && ok; j += step) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], tiles & 1, p.status, 480 + t)) != 0;
        if (!ok) break;
        ++tiles;
        tc_fence_after();
        const int key0 = first + j * kPgTile;
        const bool edge = key0 < low || key0 + kPgTile > high;
        const int shown = hi - key0, hidden = lo - key0;             // columns [hidden, shown) of this tile are visible
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld_32x32(s_t + 32 * c, v);
          tmem_wait_ld();
          if (edge) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * c + i < shown && 32 * c + i >= hidden) top = fmaxf(top, __uint_as_float(v[i]) * p.scale_log2);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(v[i]) * p.scale_log2);
          }
        }
        const bool grow = top > m + 8.f || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? top : m;
          const float alpha = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
          if (grow) l *= alpha;
          m = m_new;
          if (j > from) {
            const float keep = grow ? alpha : 1.f;
            for (int c = 0; c < p.vp; c += 16) {
              uint32_t o[16];
              tmem_ld_32x16(o_t + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st_32x16(o_t + c, o);
            }
          }
        }
        const float neg = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32], w[16];
          tmem_ld_32x32(s_t + 32 * c, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float a = ex2_approx(fmaf(__uint_as_float(v[2 * i]), p.scale_log2, neg));
            float b = ex2_approx(fmaf(__uint_as_float(v[2 * i + 1]), p.scale_log2, neg));
            if (edge) {
              const int x = 32 * c + 2 * i;
              a = x < shown && x >= hidden ? a : 0.f;
              b = x + 1 < shown && x + 1 >= hidden ? b : 0.f;
            }
            l += a + b;
            const __nv_bfloat162 q = __floats2bfloat162_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&q);
          }
          tmem_st_32x16(s_t + 16 * c, w);                // columns whose S this thread has read
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (hi <= lo) {                                    // a query that sees nothing here: tiles without an edge did not look
        m = -INFINITY;
        l = 0.f;
      }
      if (both) s_ml[t * kPgTile + mine] = make_float2(m, l);
      // which results exist: tile x has one where it had a tile of keys
      const bool has[2] = {n > 0, both ? n > 1 : n > 0};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (!has[x]) continue;
        if (ok && (both || x == t)) ok = __all_sync(0xffffffffu, mbar_wait(&o_full[x], outs[x] & 1, p.status, 490 + x)) != 0;
        ++outs[x];
      }
      tc_fence_after();
      named_barrier(1, 2 * kPgTile);                     // s_ml is there
      const bool write = ok && r >= 0;
      const long long cell = write ? (1ll * plan.cell[r] + it.split) * p.heads + g * p.n + mine_q % p.n : 0;
      float f0 = 1.f, f1 = 0.f;                          // factors on the two tiles' results
      if (both) {
        const float2 a = s_ml[mine], b = s_ml[kPgTile + mine];
        m = fmaxf(a.x, b.x);
        f0 = a.x == -INFINITY ? 0.f : ex2_approx(a.x - m);
        f1 = b.x == -INFINITY ? 0.f : ex2_approx(b.x - m);
        l = a.y * f0 + b.y * f1;
      }
      if (write && !(both && t == 1)) *reinterpret_cast<float2*>(plan.part_ml + 2 * cell) = make_float2(m, l);
      if (ok && n > 0) {                                 // whole warps: tensor memory is read by all lanes
        float* dst = plan.part_o + cell * p.vp;
        const int half = p.vp / 32 * 16, c0 = both && t == 1 ? half : 0, c1 = both && t == 0 ? half : p.vp;
        for (int c = c0; c < c1; c += 16) {
          uint32_t a[16], b[16];
          tmem_ld_32x16((both ? tmem + lanes + 256 : o_t) + c, a);
          if (has[1] && both) tmem_ld_32x16(tmem + lanes + 384 + c, b);
          tmem_wait_ld();
          if (write) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              float o[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                o[e] = f0 * __uint_as_float(a[i + e]);
                if (has[1] && both) o[e] += f1 * __uint_as_float(b[i + e]);
              }
              *reinterpret_cast<float4*>(dst + c + i) = make_float4(o[0], o[1], o[2], o[3]);
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      named_barrier(1, 2 * kPgTile);                     // tensor memory and s_ml may be written again
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Stages and shared memory of a launch; false: the sizes do not fit.
static bool plan_prefix_group(const ds41_group_attend_args& a, const ds41_prefix_plan& plan, PrefixGroupParams& p, int& smem) {
  p.n = a.heads / a.kv_heads;
  if (a.f32 || a.n_pages <= 0 || a.vdim_pad > 128 || (a.ld_q & 7) || plan.rows_per_item * p.n > 2 * kPgTile ||
      ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.pool)) & 15) ||
      1ll * a.n_pages * a.page_tokens >= (1ll << 31) - 1)
    return false;
  if (a.page_tokens % kPgTile == 0) p.box = kPgTile;
  else if (kPgTile % a.page_tokens == 0 && a.page_tokens >= 8) p.box = a.page_tokens;
  else return false;
  p.kd = (a.dim_pad + 63) / 64;
  p.vc = (a.vdim_pad + 63) / 64;
  const int qk = p.kd * kPgChunk, v = p.vc * kPgChunk;
  constexpr int kExtra = 1024 + 128 + 4 * 2 * kPgTile + 8 * 2 * kPgTile, kLimit = 227 * 1024 - kExtra;
  p.k_stages = p.v_stages = 1;
  if (3 * qk + v > kLimit) return false;
  if (4 * qk + v <= kLimit) p.k_stages = 2;
  if ((2 + p.k_stages) * qk + 2 * v <= kLimit) p.v_stages = 2;
  smem = (2 + p.k_stages) * qk + p.v_stages * v + kExtra;
  return true;
}

// cudaErrorNotSupported: these sizes are for the simple form
int launch_prefix_group(const ds41_group_attend_args& a, const ds41_prefix_plan& plan, cudaStream_t st) {
  PrefixGroupParams p{};
  int smem = 0;
  if (!plan_prefix_group(a, plan, p, smem)) return cudaErrorNotSupported;
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.page_table = a.page_table; p.row_pos = a.row_pos; p.row_slot = a.row_slot;
  p.ld_q = a.ld_q; p.heads = a.heads; p.kv_heads = a.kv_heads; p.dp = a.dim_pad; p.vp = a.vdim_pad;
  p.chunk = a.chunk; p.max_pages = a.max_pages; p.page_tokens = a.page_tokens; p.hidden_row = a.n_pages * a.page_tokens;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = a.status;
  CUtensorMap pool;
  const int row_len = a.kv_heads * (a.dim_pad + a.vdim_pad);
  cudaError_t e = make_tensor_map_3d(&pool, a.pool, TmaDtype::kBF16, row_len, p.hidden_row, 1, 2ull * row_len, 0, 64, p.box, true);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(prefix_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(prefix_group_kernel, dim3(plan.grid), dim3(kPgThreads), smem, st, pool, p, plan);
}

}  // namespace ds41
