// Parts of grouped-query attention for rows that share prefixes, on tcgen05.
//
// The queries of one key/value head are packed: (row, head) pairs of a unit's rows are the 128 rows of a tensor-core tile, so that a
// tile of keys and values is read once for all of them and the products have the shape of a prompt's.  A CTA walks units, its copies
// running ahead into the next one, and has two tiles:
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

  const int units = *plan.n_units;
  // the key tiles of a unit (whole warps)
  auto span = [&](const PrefixUnit& it, int& first, int& end) {
    prefix_span(plan, it, p.row_pos, p.row_slot, p.chunk, p.page_tokens, first, end);
    return (end - first + kPgTile - 1) / kPgTile;
  };

  if (warp == 8) {
    const int boxes = kPgTile / p.box;
    int kt = 0, k_stage = 0, v_stage = 0;                // key tiles so far, places in the rings
    uint32_t k_free = 1, v_free = 1;
    bool ok = true;
    for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x) {
      const PrefixUnit it = prefix_unit(plan, unit);
      if (it.rows == 0) continue;
      const int g = it.head;
      int first, end;
      const int n = span(it, first, end);
      const int* table = p.page_table + 1ll * it.slot * p.max_pages;
      int row = 0, u = 0;                                // lane i: pool row of box i of the walk, 32 boxes at a time
      for (int j = 0; j < n; ++j, ++kt, u += boxes) {
        if ((u & 31) == 0) {                             // boxes divides 32
          const int key = first + (u + lane) * p.box, pg = key / p.page_tokens;
          const int id = key < end && pg < p.max_pages ? table[pg] : -1;
          row = id >= 0 ? id * p.page_tokens + (key - pg * p.page_tokens) : p.hidden_row;
        }
        // one tile of keys or values: `chunks` chunks of 64 columns from column x on
        auto fetch = [&](uint8_t* dst, uint64_t* bar, int x, int chunks) {
          if (lane == 0) mbar_expect_tx(bar, chunks * kPgChunk);
#pragma unroll 1
          for (int i = 0; i < boxes; ++i) {
            const int at = __shfl_sync(0xffffffffu, row, (u + i) & 31);
            if (lane == 0)
#pragma unroll 1
              for (int c = 0; c < chunks; ++c) tma_load_3d(dst + c * kPgChunk + i * p.box * 128, &pool, bar, x + 64 * c, at, 0);
            __syncwarp();
          }
        };
        ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[k_stage], k_free, p.status, 460)) != 0;
        if (!ok) break;
        fetch(s_k + k_stage * k_bytes, &k_full[k_stage], g * p.dp, p.kd);
        if (++k_stage == p.k_stages) {
          k_stage = 0;
          k_free ^= 1;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[v_stage], v_free, p.status, 461)) != 0;
        if (!ok) {
          ++kt;
          break;
        }
        fetch(s_v + v_stage * v_bytes, &v_full[v_stage], p.kv_heads * p.dp + g * p.vp, p.vc);
        if (++v_stage == p.v_stages) {
          v_stage = 0;
          v_free ^= 1;
        }
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
    const int whole = p.dp / 64, rest = p.dp / 16 - 4 * whole;
    bool ok = true;
    int kt = 0, done[2] = {0, 0}, live = 0;              // key tiles; products of each tile; units with work so far
    for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x) {
      const PrefixUnit it = prefix_unit(plan, unit);
      if (it.rows == 0) continue;
      int first, end;
      const int n = span(it, first, end);
      if (n == 0) continue;
      if (leader) {                                      // one thread: votes and the like between two products cost as much as the products
        ok = mbar_wait(q_full, live & 1, p.status, 470);
        ++live;
        tc_fence_after();
        const bool both = it.rows * p.n <= kPgTile;
        const int step = both ? 2 : 1;
        // per tile: its next scores and next values, as numbers of key tiles; scores overwrite the P that the values before them read
        int sj[2] = {0, both ? 1 : 0}, pj[2] = {0, both ? 1 : 0};
        uint32_t idle = 0;
        long long since = 0;
        while (ok && (pj[0] < n || pj[1] < n)) {
          bool moved = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (pj[t] < sj[t] && pj[t] < n) {
              const int at = kt + pj[t], stage = p.v_stages == 2 ? at & 1 : 0, phase = p.v_stages == 2 ? (at >> 1) & 1 : at & 1;
              if (mbar_test_wait(&p_full[t], done[t] & 1) && mbar_test_wait(&v_full[stage], phase)) {
                tc_fence_after();
                const uint64_t vd = v_desc + static_cast<uint64_t>(stage * v_bytes / 16);
                const uint32_t o = tmem + 256 + t * 128, a = tmem + t * 128;
                umma4_ts<128>(o, a, vd, idesc_pv, pj[t] >= step);
                umma4_ts<128>(o, a + 32, vd + 512, idesc_pv, 1u);
                ++done[t];
                if (both || pj[t ^ 1] > pj[t]) tc_commit_if(true, &v_empty[stage]);      // the tile's last reader
                pj[t] += step;
                if (pj[t] >= n) tc_commit_if(true, &o_full[t]);
                moved = true;
              }
            }
            if (sj[t] < n && sj[t] == pj[t]) {
              const int at = kt + sj[t], stage = p.k_stages == 2 ? at & 1 : 0, phase = p.k_stages == 2 ? (at >> 1) & 1 : at & 1;
              if (mbar_test_wait(&k_full[stage], phase)) {
                tc_fence_after();
                uint64_t a = q_desc + static_cast<uint64_t>(both ? 0 : t * q_bytes / 16), b = k_desc + static_cast<uint64_t>(stage * k_bytes / 16);
#pragma unroll 1
                for (int c = 0; c < whole; ++c, a += kPgChunk / 16, b += kPgChunk / 16) umma4_ss<2, 2>(tmem + t * 128, a, b, idesc_s, c);
#pragma unroll 1
                for (int k = 0; k < rest; ++k) umma_bf16(tmem + t * 128, a + 2 * k, b + 2 * k, idesc_s, whole > 0 || k > 0);
                tc_commit_if(true, &s_full[t]);
                if (both || sj[t ^ 1] > sj[t]) tc_commit_if(true, &k_empty[stage]);
                sj[t] += step;
                moved = true;
              }
            }
          }
          if (moved) {
            idle = 0;
            since = 0;
          } else if ((++idle & 0x3ff) == 0) {            // as long as any other wait: see mbar_wait
            if (since == 0) since = clock64();
            if (clock64() - since > DS41_WAIT_LIMIT_CYCLES ||
                (p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != kStatusOk)) {
              if (p.status != nullptr && atomicCAS(p.status, kStatusOk, kStatusMbarTimeout) == kStatusOk) {
                p.status[1] = 471;
                p.status[2] = static_cast<int>(blockIdx.x);
                p.status[3] = pj[0];
              }
              ok = false;
            }
          }
        }
        kt += n;
      }
      ok = __ballot_sync(0xffffffffu, leader && ok) != 0;
    }
  } else {
    const int t = warp >> 2, quad = warp & 3, mine = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_t = tmem + lanes + t * 128, o_t = tmem + lanes + 256 + t * 128;
    int kt = 0, tiles = 0, outs[2] = {0, 0};             // key tiles so far; tiles of S seen by this half; finished results of both
    bool ok = true;
    // the loop runs to its end whatever happened: its barriers are for all eight warps
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
      const PrefixUnit it = prefix_unit(plan, unit);
      if (it.rows == 0) continue;
      const int g = it.head, count = it.rows * p.n;
      const bool both = count <= kPgTile;                // the same queries in both tiles
      int first, end;
      const int n = span(it, first, end);
      const int mine_q = both ? mine : t * kPgTile + mine;
      int r = -1, lo = 0, hi = 0;
      if (mine_q < count) {
        r = prefix_row(plan, it, mine_q / p.n);
        const int pos = p.row_pos[r];
        if (p.row_slot[r] >= 0) {
          lo = chunk_start(pos, p.chunk);
          hi = min(pos + 1, it.key1);
        }
      }
      s_row[t * kPgTile + mine] = r;                     // equal in both halves where the queries are
      named_barrier(1, 2 * kPgTile);
      if (n > 0) {
        // a row's 16-byte pieces by neighbouring lanes, four rows of a lane under way together
        const int pieces = p.dp / 8, per = 32 / pieces, sub = lane / pieces, c = lane % pieces, rows = (both ? 1 : 2) * kPgTile;
        for (int x0 = warp * per + sub; x0 < rows; x0 += 32 * per) {
          uint4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int x = x0 + 8 * per * k, row = sub < per && x < rows ? s_row[x] : -1;
            v[k] = make_uint4(0, 0, 0, 0);
            if (row >= 0) v[k] = *reinterpret_cast<const uint4*>(p.q + row * p.ld_q + 1ll * (g * p.n + x % p.n) * p.dp + 8 * c);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int x = x0 + 8 * per * k, y = x & (kPgTile - 1);
            if (sub < per && x < rows)
              *reinterpret_cast<uint4*>(s_q + (x >> 7) * q_bytes + (c >> 3) * kPgChunk + y * 128 + (((c & 7) ^ (y & 7)) << 4)) = v[k];
          }
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
        // Two halves of 64 columns, each read twice: the loops' bodies have to stay in the instruction cache, which this code shares
        // with the other roles' (unrolled over the tile, 42 % of all cycles were waits for instructions)
        float top = -INFINITY;
        uint32_t v[64];
        auto load = [&](int c) {
          tmem_ld_32x32(s_t + c, reinterpret_cast<uint32_t(&)[32]>(v[0]));
          tmem_ld_32x32(s_t + c + 32, reinterpret_cast<uint32_t(&)[32]>(v[32]));
          tmem_wait_ld();
          if (edge) {
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = c + i < shown && c + i >= hidden ? v[i] : 0xff800000u;
          }
        };
#pragma unroll 1
        for (int c = 0; c < kPgTile; c += 64) {
          load(c);
          float tops[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 64; i += 2) tops[(i >> 1) & 3] = fmaxf(tops[(i >> 1) & 3], fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
          top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        }
        top *= p.scale_log2;
        const bool grow = top > m + 8.f || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? top : m;
          const float alpha = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
          if (grow) l *= alpha;
          m = m_new;
          if (j > from) {
            const float keep = grow ? alpha : 1.f;
#pragma unroll 1
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
        const float2 by = make_float2(p.scale_log2, p.scale_log2), off = make_float2(neg, neg);
        float2 sums[2] = {};
#pragma unroll 1
        for (int c = 0; c < kPgTile; c += 64) {
          load(c);
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float2 e = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), by, off);
            e = make_float2(ex2_approx(e.x), ex2_approx(e.y));
            sums[i & 1] = add2(sums[i & 1], e);
            const __nv_bfloat162 q = __floats2bfloat162_rn(e.x, e.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&q);
          }
          tmem_st_32x32(s_t + c / 2, w);                 // columns whose S this thread has read
        }
        sums[0] = add2(sums[0], sums[1]);
        l += sums[0].x + sums[0].y;
        if (it.tail && key0 + kPgTile > end) {
          // Places behind the last position belong to nobody, and a weight of zero does not take a NaN or an infinity away: their values
          // become zeros, a thread to a place.
          const int at = kt + j, stage = p.v_stages == 2 ? at & 1 : 0, phase = p.v_stages == 2 ? (at >> 1) & 1 : at & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&v_full[stage], phase, p.status, 484 + t)) != 0;
          if (!ok) break;
          if (key0 + mine >= end)
            for (int i = 0; i < 8 * p.vc; ++i)
              *reinterpret_cast<uint4*>(s_v + stage * v_bytes + (i >> 3) * kPgChunk + mine * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      kt += n;
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
      const long long cell = write ? (1ll * plan.cell[r] + it.part) * p.heads + g * p.n + mine_q % p.n : 0;
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
            for (int i = 0; i < 16; i += 8) {
              float o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                o[e] = f0 * __uint_as_float(a[i + e]);
                if (has[1] && both) o[e] += f1 * __uint_as_float(b[i + e]);
              }
              store8(dst + c + i, o);
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
  if (a.f32 || a.n_pages <= 0 || a.vdim_pad > 128 || (a.ld_q & 7) || plan.rows_per_unit * p.n > 2 * kPgTile ||
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
