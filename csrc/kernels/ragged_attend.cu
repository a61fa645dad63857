// Attention of a ragged pass on tcgen05: bf16, up to 256 values of a key and 128 of a value, pages of 16 to 128 tokens or whole 128s.
//
// The queries of one key/value head are packed: the (token, head) pairs of a block's tokens are the rows of a tensor-core tile, so that a
// tile of keys and values is read once for all of them.  A CTA has two tiles of 128 rows.  A block of many tokens fills both, which then
// walk the same keys; a block of a few rows (decode) has them twice, and its two copies take the key tiles in turn.  Either way one
// tile's softmax runs while the tensor core works on the other's products.
//   warps 0-3, 4-7 : softmax of tile 0 / 1 (one thread per row), results
//   warp 8, 11     : TMA producers: queries and keys / values, page by page, a lane per copy
//   warp 9         : tcgen05.mma issue: S = Q K^T into TMEM, O += P V with P read from TMEM where it replaces its S
//   warp 10        : zeros in place of values that no row of the unit sees: their weights are zeros, but they may hold anything
// The running maximum is raised when it grew by more than 2^8 only, so the accumulated output is rarely rescaled.  P is rounded to bf16
// as the operand of the second product; the sums take the unrounded weights.
//
// A CTA walks the units blockIdx.x, 2 * grid - 1 - blockIdx.x, ... of a list with the longest first; all roles but the softmax run ahead.
#include <cuda.h>

#include <atomic>

#include "ds41_prefix.cuh"
#include "ds41_ragged.cuh"
#include "ds41_tma.h"

namespace ds41 {

constexpr int kRtThreads = 384;
constexpr int kRtTile = 128;                   // rows of a tile, keys of a tile
constexpr int kRtChunk = kRtTile * 128;        // bytes of 128 rows x 64 bf16 columns
constexpr int kRtStages = 4, kRtSlotRows = 64;

struct TiledParams {
  ds41_ragged_attend_args a;
  ds41_ragged_pass p;
  int group, per_tile;       // query heads of a key/value head, tokens of a tile
  int kd, vc;                // 64-column chunks of a key and a value
  int k_stages, v_stages;
  int box, slot_rows;        // rows of a copy; most rows of a block whose tiles take the keys in turn
  int hidden_row;            // beyond the pool: reads as zeros
  float scale_log2;
};

struct TiledShared {
  uint64_t q_full, q_free;                     // queries are there; the unit's last scores are done
  uint64_t k_full[kRtStages], k_empty[kRtStages], v_full[kRtStages], v_empty[kRtStages];
  uint64_t v_clean[kRtStages];                 // places that nobody sees are zeros
  uint64_t s_full[2], p_full[2], o_full[2];    // per tile: S complete (and every earlier product); P written, O rescaled; O complete
  uint64_t half_full, half_read[2];            // the second tile's half of a unit whose keys were taken in turn
  float2 half_ml[kRtSlotRows];
  uint32_t tmem;
  int flag[2];
};

// What every role knows of a unit.
struct TiledUnit {
  RaggedUnit u;
  RaggedWalk walk;
  bool turns;                // its tiles take the key tiles in turn
  int tok0;                  // tokens of tile 0 (in turns: of both)
  int n[2];                  // key tiles of either tile
};

__device__ __forceinline__ TiledUnit tiled_unit(const TiledParams& t, int i) {
  TiledUnit x;
  x.u = ragged_unit(t.p, i);
  const RaggedUnit& u = x.u;
  x.turns = u.tokens * t.group <= t.slot_rows;
  x.tok0 = x.turns ? u.tokens : (u.tokens + 1) / 2;
  x.walk = ragged_walk(u.pos0, u.pos0 + u.tokens - 1, t.p.window, t.p.first, t.box);
  if (x.turns) {
    x.n[0] = (u.tiles + 1) / 2;
    x.n[1] = u.tiles / 2;
  } else {
    const int seen = u.pos0 + x.tok0 - x.walk.shift;                     // places up to tile 0's last row
    x.n[0] = min(max((seen + kRtTile - 1) / kRtTile - u.tile0, 0), u.tiles);
    x.n[1] = u.tokens > x.tok0 ? u.tiles : 0;
  }
  return x;
}

// The unit of a CTA's turn: the list goes back and forth.
__device__ __forceinline__ int unit_at(int turn) {
  return turn * static_cast<int>(gridDim.x) +
         (turn & 1 ? static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The lowest n bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// All lanes, or one thread by itself.
#define WARP_WAIT(bar, parity, where) (__all_sync(0xffffffffu, mbar_wait(bar, parity, t.p.status, where)) != 0)

__global__ void __launch_bounds__(kRtThreads, 1)
ragged_tiled_kernel(const __grid_constant__ CUtensorMap queries, const __grid_constant__ CUtensorMap pool,
                    const __grid_constant__ TiledParams t) {
  extern __shared__ uint8_t rt_raw[];
  uint8_t* smem = rt_raw + ((1024u - (smem_u32(rt_raw) & 1023u)) & 1023u);
  const int q_bytes = t.kd * kRtChunk, k_bytes = q_bytes, v_bytes = t.vc * kRtChunk;
  uint8_t* s_q = smem;                                   // two tiles
  uint8_t* s_k = s_q + 2 * q_bytes;
  uint8_t* s_v = s_k + t.k_stages * k_bytes;
  TiledShared& sh = *reinterpret_cast<TiledShared*>(s_v + t.v_stages * v_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int dp = t.p.dim, vp = t.p.vdim;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_free, 1);
    for (int i = 0; i < kRtStages; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_clean[i], 1);
      mbar_init(&sh.v_empty[i], 2);                      // the products, the cleaner
    }
    mbar_init(&sh.half_full, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.half_read[i], 4);
    }
    mbar_init_fence();
    tma_prefetch_desc(&queries);
    tma_prefetch_desc(&pool);
  }
  if (warp == 9) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  pdl_wait();
  const int units = t.p.header[0];

  if (warp == 8 || warp == 11) {
    const bool values = warp == 11;
    const int chunks = values ? t.vc : t.kd, stages = values ? t.v_stages : t.k_stages, bytes = values ? v_bytes : k_bytes;
    uint8_t* ring = values ? s_v : s_k;
    uint64_t *full = values ? sh.v_full : sh.k_full, *empty = values ? sh.v_empty : sh.k_empty;
    const int box = lane / chunks, chunk = lane - box * chunks;          // this lane's copy of a tile
    const bool copies = box < kRtTile / t.box;
    uint8_t* const dst = ring + chunk * kRtChunk + box * t.box * 128;
    int count = 0, stage = 0, done = 0, halves = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int turn = 0; unit_at(turn) < units && ok; ++turn) {
      const TiledUnit x = tiled_unit(t, unit_at(turn));
      if (x.u.tiles == 0) continue;
      auto locate = [&](int s) {
        const int place = (x.u.tile0 + s) * kRtTile + box * t.box, pos = place < x.walk.lead ? place : place + x.walk.shift;
        const int pg = pos / t.p.page_tokens;
        const int id = copies && place < x.walk.places && pg < t.a.max_pages
                           ? __ldg(t.a.page_table + 1ll * x.u.slot * t.a.max_pages + pg) : -1;
        return static_cast<unsigned>(id) < static_cast<unsigned>(t.a.n_pages) ? id * t.p.page_tokens + (pos - pg * t.p.page_tokens)
                                                                              : t.hidden_row;
      };
      int row = locate(0);
      if (!values) {
        ok = WARP_WAIT(&sh.q_free, (done & 1) ^ 1, 600);
        // the second tile's place holds halves of units that went in turns
        for (int h = max(0, halves - 2); h < halves && ok && !x.turns; ++h) ok = WARP_WAIT(&sh.half_read[h & 1], (h >> 1) & 1, 601);
        if (!ok) break;
        const bool second = !x.turns && x.u.tokens > x.tok0;
        if (lane == 0) mbar_expect_tx(&sh.q_full, (second ? 2 : 1) * t.kd * t.per_tile * t.group * 128);
        __syncwarp();
        if (lane < (second ? 2 : 1) * t.kd) {
          const int k = lane / t.kd, c = lane - k * t.kd;
          tma_load_3d(s_q + k * q_bytes + c * kRtChunk, &queries, &sh.q_full, 64 * c, x.u.head * t.group, x.u.row0 + k * x.tok0);
        }
        ++done;
        if (x.turns && x.u.tiles > 1) ++halves;
      }
      const int col = (values ? t.p.kv_heads * dp + x.u.head * vp : x.u.head * dp) + 64 * chunk;
      for (int s = 0; s < x.u.tiles; ++s) {
        const int at = row;
        if (s + 1 < x.u.tiles) row = locate(s + 1);
        ok = WARP_WAIT(&empty[stage], phase, values ? 603 : 602);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&full[stage], bytes);
        __syncwarp();
        if (copies) tma_load_3d(dst + stage * bytes, &pool, &full[stage], col, at, 0);
        ++count;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && lane == 0) {                              // something gave up: the copies under way land before the memory goes away
      auto drain = [](uint64_t* bar, uint32_t parity) {
        for (int i = 0; i < (1 << 18) && !mbar_test_wait(bar, parity); ++i) {
        }
      };
      if (!values && done > 0) drain(&sh.q_full, (done - 1) & 1);
      for (int b = max(0, count - stages); b < count; ++b) drain(&full[b % stages], (b / stages) & 1);
    }
  } else if (warp == 9) {
    if (elect_one()) {
      const uint32_t idesc_s = umma_idesc(kRtTile, kRtTile, 1u, 1u), idesc_pv = umma_idesc_bmn(kRtTile, vp, 1u, 1u);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q)), k_desc = umma_desc_sw128(smem_u32(s_k));
      const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(s_v), kRtChunk, 1024);
      const int whole = dp / 64, rest = dp / 16 - 4 * whole;
      int begun = 0, count = 0, products[2] = {0, 0};     // units, key tiles, products of either tile
      bool ok = true;
      for (int turn = 0; unit_at(turn) < units && ok; ++turn) {
        const TiledUnit x = tiled_unit(t, unit_at(turn));
        const int n = x.u.tiles, ahead = x.turns ? 2 : 1;
        if (n == 0) continue;
        const int low = ragged_low(x.u.pos0, t.p.window) - x.walk.shift;
        auto takes = [&](int i, int s) { return x.turns ? s < n && (s & 1) == i : s < x.n[i]; };
        auto scores = [&](int i, int s) {                // the tile's keys have landed
          uint64_t a = q_desc + (x.turns ? 0u : static_cast<uint64_t>(i * q_bytes / 16));
          uint64_t b = k_desc + static_cast<uint64_t>((count + s) % t.k_stages * (k_bytes / 16));
#pragma unroll 1
          for (int c = 0; c < whole; ++c, a += kRtChunk / 16, b += kRtChunk / 16) umma4_ss<2, 2>(tmem + i * 128, a, b, idesc_s, c);
#pragma unroll 1
          for (int k = 0; k < rest; ++k) umma_bf16(tmem + i * 128, a + 2 * k, b + 2 * k, idesc_s, whole > 0 || k > 0);
          tc_commit(&sh.s_full[i]);
        };
        auto keys = [&](int s) {
          const int at = count + s;
          if (!mbar_wait(&sh.k_full[at % t.k_stages], (at / t.k_stages) & 1, t.p.status, 610)) return false;
          tc_fence_after();
          return true;
        };
        auto keys_read = [&](int s) {
          tc_commit(&sh.k_empty[(count + s) % t.k_stages]);
          if (s == n - 1) tc_commit(&sh.q_free);
        };
        ok = mbar_wait(&sh.q_full, begun & 1, t.p.status, 611);
        ++begun;
        for (int s = 0; s < ahead && s < n && ok; ++s) {
          ok = keys(s);
          if (!ok) break;
          for (int i = 0; i < 2; ++i)
            if (takes(i, s)) scores(i, s);
          keys_read(s);
        }
        for (int s = 0; s < n && ok; ++s) {
          const int at = count + s, vs = at % t.v_stages, place0 = (x.u.tile0 + s) * kRtTile;
          const bool unseen = place0 + kRtTile > x.walk.places || (max(place0, t.p.first) < min(place0 + kRtTile, low));
          ok = mbar_wait(unseen ? &sh.v_clean[vs] : &sh.v_full[vs], (at / t.v_stages) & 1, t.p.status, 612);
          if (ok && s + ahead < n) ok = keys(s + ahead);
          if (!ok) break;
          for (int i = 0; i < 2 && ok; ++i) {
            if (takes(i, s)) {
              ok = mbar_wait(&sh.p_full[i], products[i] & 1, t.p.status, 614 + i);
              if (!ok) break;
              tc_fence_after();
              const uint64_t v = v_desc + static_cast<uint64_t>(vs * (v_bytes / 16));
              const bool first = s == (x.turns ? i : 0);
              umma4_ts<128>(tmem + 256 + i * 128, tmem + i * 128, v, idesc_pv, !first);
              umma4_ts<128>(tmem + 256 + i * 128, tmem + i * 128 + 32, v + 512, idesc_pv, 1);
              ++products[i];
              if (!takes(i, s + ahead)) tc_commit(&sh.o_full[i]);
            }
            if (x.turns ? takes(i, s) : i == 1) tc_commit(&sh.v_empty[vs]);
            if (takes(i, s + ahead)) scores(i, s + ahead);
          }
          if (ok && s + ahead < n) keys_read(s + ahead);
        }
        count += n;
      }
    }
    __syncwarp();
  } else if (warp == 10) {
    int count = 0;
    bool ok = true;
    for (int turn = 0; unit_at(turn) < units && ok; ++turn) {
      const TiledUnit x = tiled_unit(t, unit_at(turn));
      const int low = ragged_low(x.u.pos0, t.p.window) - x.walk.shift;
      for (int s = 0; s < x.u.tiles; ++s, ++count) {
        const int vs = count % t.v_stages, place0 = (x.u.tile0 + s) * kRtTile;
        ok = WARP_WAIT(&sh.v_full[vs], (count / t.v_stages) & 1, 620);
        if (!ok) break;
        // places [a, b) and [c, 128) of the tile are seen by nobody
        const int a = max(0, t.p.first - place0), b = min(kRtTile, low - place0), c = min(kRtTile, x.walk.places - place0);
        if (a < b || c < kRtTile) {
          for (int k = 0; k < t.vc; ++k) {
            uint8_t* v = s_v + vs * v_bytes + k * kRtChunk + 16 * (lane & 7);
            for (int r = a + (lane >> 3); r < b; r += 4) *reinterpret_cast<uint4*>(v + r * 128) = make_uint4(0, 0, 0, 0);
            for (int r = c + (lane >> 3); r < kRtTile; r += 4) *reinterpret_cast<uint4*>(v + r * 128) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sh.v_clean[vs]);
          mbar_arrive(&sh.v_empty[vs]);
        }
      }
    }
  } else {
    // Where a wait gave up, `ok` stays false and later ones are left out, but every barrier that warps share is reached.
    const int i = warp >> 2, quad = warp & 3, mine = quad * 32 + lane, tid = mine;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_t = tmem + lanes + i * 128, o_t = tmem + lanes + 256 + i * 128;
    const int mine_tok = mine / t.group, mine_head = mine - mine_tok * t.group;
    int tiles = 0, outputs = 0, halves = 0;
    bool ok = true;
    for (int turn = 0; unit_at(turn) < units; ++turn) {
      const TiledUnit x = tiled_unit(t, unit_at(turn));
      const RaggedUnit& u = x.u;
      if (u.tiles == 0) {
        for (int r = threadIdx.x; r < u.tokens * t.group; r += 256) {
          uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(t.a.out) + (u.row0 + r / t.group) * t.a.out_row +
                                                1ll * (u.head * t.group + r % t.group) * vp);
          for (int c = 0; c < vp / 8; ++c) out[c] = make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      const int first_tok = i && !x.turns ? x.tok0 : 0, toks = x.turns ? u.tokens : (i ? u.tokens - x.tok0 : x.tok0);
      const bool live = mine_tok < toks && mine < t.per_tile * t.group;
      const int pos = u.pos0 + first_tok + min(mine_tok, toks - 1);
      // visible places of this thread's row: [0, a) and [b, e); of all of its warp's: up to a_all, from b_all to e_all
      const int shift = x.walk.shift;
      const int e = pos + 1 - shift, b = ragged_low(pos, t.p.window) - shift, a = min(t.p.first, e);
      const int b_all = __shfl_sync(0xffffffffu, b, 31), e_all = __shfl_sync(0xffffffffu, e, 0), a_all = min(t.p.first, e_all);
      const bool idle = !__any_sync(0xffffffffu, live);
      float m = -INFINITY, l = 0.f;
      const int n = x.n[i];
      for (int j = 0; j < n; ++j) {
        if (ok) ok = WARP_WAIT(&sh.s_full[i], tiles & 1, 630 + i);
        ++tiles;
        if (!ok) continue;
        if (!idle) {
          tc_fence_after();
          const int place0 = (u.tile0 + (x.turns ? 2 * j + i : j)) * kRtTile;
          if ((place0 < b_all || place0 + kRtTile > e_all) && place0 + kRtTile > a_all) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t v[32];
              tmem_ld_32x32(s_t + 32 * c, v);
              const int at = place0 + 32 * c;
              const uint32_t seen = low_bits(a - at) | (low_bits(e - at) & ~low_bits(b - at));
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = seen >> k & 1 ? v[k] : 0xff800000u;
              tmem_st_32x32(s_t + 32 * c, v);
            }
            tmem_wait_st();
          }
          float v[kRtTile];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_t + 32 * c, reinterpret_cast<uint32_t(&)[32]>(v[32 * c]));
          tmem_wait_ld();
          float top4[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            top4[c] = max3_nan(v[c], v[4 + c], v[8 + c]);
#pragma unroll
            for (int k = 12; k + 4 < kRtTile; k += 8) top4[c] = max3_nan(top4[c], v[k + c], v[k + 4 + c]);
            top4[c] = max3_nan(top4[c], top4[c], v[kRtTile - 4 + c]);
          }
          const float top = max3_nan(max3_nan(top4[0], top4[1], top4[2]), top4[3], top4[3]) * t.scale_log2;
          const bool grow = !(top <= m + 8.f);           // a NaN as well
          if (__any_sync(0xffffffffu, grow)) {
            const float m_new = grow ? top : m;
            const float keep = grow ? (m == -INFINITY ? 0.f : ex2_approx(m - m_new)) : 1.f;
            l *= keep;
            m = m_new;
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < vp; c += 16) {
                uint32_t o[16];
                tmem_ld_32x16(o_t + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                tmem_st_32x16(o_t + c, o);
              }
            }
          }
          const float neg = m == -INFINITY ? 0.f : -m;
          const float2 scale2 = make_float2(t.scale_log2, t.scale_log2), neg2 = make_float2(neg, neg);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              float2 y = fma2(make_float2(v[64 * h + 2 * k], v[64 * h + 2 * k + 1]), scale2, neg2);
              y.x = ex2_approx(y.x);
              y.y = ex2_approx(y.y);
              sum[k & 1] = add2(sum[k & 1], y);
              const __nv_bfloat162 q = __floats2bfloat162_rn(y.x, y.y);
              w[k] = *reinterpret_cast<const uint32_t*>(&q);
            }
            tmem_st_32x32(s_t + 32 * h, w);              // columns whose S this thread has read
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[i]);
      }
      if (n > 0) {
        if (ok) ok = WARP_WAIT(&sh.o_full[i], outputs & 1, 632 + i);
        ++outputs;
        tc_fence_after();
      }
      if (x.turns && i == 1) {
        // this half goes to the first tile's warps
        if (u.tiles > 1) {
          if (halves > 0 && ok) ok = WARP_WAIT(&sh.half_read[(halves - 1) & 1], ((halves - 1) >> 1) & 1, 634);
          if (!idle) {
            float4* to = reinterpret_cast<float4*>(s_q + q_bytes) + mine * (vp / 4);
#pragma unroll 1
            for (int c = 0; c < vp; c += 16) {
              uint32_t o[16];
              __syncwarp();
              tmem_ld_32x16(o_t + c, o);
              tmem_wait_ld();
              if (live)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  to[(c / 4 + k + mine) % (vp / 4)] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                                                  __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
            }
            if (live) sh.half_ml[mine] = make_float2(m, l);
          }
          tc_fence_before();
          ++halves;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.half_full);
        }
        continue;
      }
      float w_own = 1.f, w_half = 0.f;                   // factors of both halves
      const float4* half = reinterpret_cast<const float4*>(s_q + q_bytes) + mine * (vp / 4);
      const bool joined = x.turns && u.tiles > 1;
      if (joined) {
        if (ok) ok = WARP_WAIT(&sh.half_full, halves & 1, 635);
        if (live) {
          const float2 ml = sh.half_ml[mine];
          const float top = max3_nan(m, ml.x, ml.x), base = top == -INFINITY ? 0.f : top;
          w_own = ex2_approx(m - base);
          w_half = ex2_approx(ml.x - base);
          l = l * w_own + ml.y * w_half;
          m = top;
        }
      }
      const int row = u.row0 + first_tok + mine_tok, h = u.head * t.group + mine_head;
      float f = 1.f;
      long long cell = 0;
      if (u.pieces > 1) {
        cell = 1ll * u.cell + 1ll * u.piece * u.step + first_tok * t.group + mine;
        if (live) *reinterpret_cast<float2*>(t.p.part_ml + 2 * cell) = make_float2(m, l);
      } else if (live) {
        const float sink = t.a.sink != nullptr ? t.a.sink[h] * kLog2E : -INFINITY;
        const float top = max3_nan(m, sink, sink), base = top == -INFINITY ? 0.f : top;
        const float w = ex2_approx(m - base), den = l * w + (t.a.sink != nullptr ? ex2_approx(sink - base) : 0.f);
        f = den != 0.f ? w / den : 0.f;
        if (t.a.gate != nullptr) f *= sigmoid_f32(t.a.gate[row * t.a.gate_row + h]);
      }
      w_own *= f;
      w_half *= f;
      if (!idle && n > 0) {
#pragma unroll 1
        for (int c = 0; c < vp; c += 16) {
          uint32_t o[16];
          __syncwarp();
          tmem_ld_32x16(o_t + c, o);
          tmem_wait_ld();
          float y[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) y[k] = __uint_as_float(o[k]) * w_own;
          if (live && joined) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float4 z = half[(c / 4 + k + mine) % (vp / 4)];
              y[4 * k] += z.x * w_half;
              y[4 * k + 1] += z.y * w_half;
              y[4 * k + 2] += z.z * w_half;
              y[4 * k + 3] += z.w * w_half;
            }
          }
          if (live && u.pieces > 1) {
            float4* to = reinterpret_cast<float4*>(t.p.part_o + cell * vp + c);
#pragma unroll
            for (int k = 0; k < 4; ++k) to[k] = make_float4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
          } else if (live) {
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const __nv_bfloat162 q = __floats2bfloat162_rn(y[2 * k], y[2 * k + 1]);
              w[k] = *reinterpret_cast<const uint32_t*>(&q);
            }
            uint4* to = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(t.a.out) + row * t.a.out_row + 1ll * h * vp + c);
            to[0] = make_uint4(w[0], w[1], w[2], w[3]);
            to[1] = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      if (joined) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.half_read[halves & 1]);
        ++halves;
      }
      if (u.pieces > 1 && ragged_last(t.p.counters + u.counter + i, u.pieces, tid == 0, 1 + i, kRtTile, &sh.flag[i]))
        ragged_join<__nv_bfloat16>(t.p, t.a, u, first_tok * t.group + quad, (first_tok + toks) * t.group, 4);
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Stages of the rings and the launch's shared memory; 0: the sizes do not fit.
inline int tiled_smem(TiledParams& t) {
  t.kd = (t.p.dim + 63) / 64;
  t.vc = (t.p.vdim + 63) / 64;
  const int qk = t.kd * kRtChunk, v = t.vc * kRtChunk;
  constexpr int kFixed = 1024 + static_cast<int>(sizeof(TiledShared)), kLimit = 227 * 1024;
  t.k_stages = t.v_stages = 1;
  if (kFixed + 3 * qk + v > kLimit) return 0;
  while (true) {                                         // keys first: they are needed earlier
    const int left = kLimit - kFixed - 2 * qk - t.k_stages * qk - t.v_stages * v;
    if (t.k_stages <= t.v_stages && t.k_stages < kRtStages && left >= qk) ++t.k_stages;
    else if (t.v_stages < kRtStages && left >= v) ++t.v_stages;
    else if (t.k_stages < kRtStages && left >= qk) ++t.k_stages;
    else break;
  }
  return kFixed + 2 * qk + t.k_stages * qk + t.v_stages * v;
}

cudaError_t launch_ragged_tiled(const ds41_ragged_attend_args& a, const ds41_ragged_pass& p, cudaStream_t stream) {
  TiledParams t{};
  t.a = a;
  t.p = p;
  t.group = p.heads / p.kv_heads;
  if (p.f32 || t.group > kRtTile || p.vdim > 128 || p.page_tokens < 16 || (p.page_tokens < kRtTile ? kRtTile % p.page_tokens : p.page_tokens % kRtTile))
    return cudaErrorInvalidValue;
  t.per_tile = kRtTile / t.group;
  if (p.unit_tokens != 2 * t.per_tile) return cudaErrorInvalidValue;
  const int smem = tiled_smem(t);
  if (smem == 0) return cudaErrorInvalidValue;
  t.box = p.page_tokens < kRtTile ? p.page_tokens : kRtTile;
  if (kRtTile / t.box * (t.kd > t.vc ? t.kd : t.vc) > 32) return cudaErrorInvalidValue;
  t.slot_rows = t.kd * kRtChunk / (4 * p.vdim);          // their results have to fit the second tile's place
  if (t.slot_rows > kRtSlotRows) t.slot_rows = kRtSlotRows;
  t.hidden_row = a.n_pages * p.page_tokens;
  t.scale_log2 = a.scale * kLog2E;
  const int row_len = p.kv_heads * (p.dim + p.vdim);
  CUtensorMap queries, pool;
  cudaError_t e = make_tensor_map_3d(&queries, a.q, TmaDtype::kBF16, p.dim, p.heads, a.q_rows, 2 * a.q_head, 2 * a.q_row, 64, t.group, true,
                                     t.per_tile);
  if (e != cudaSuccess) return e;
  e = make_tensor_map_3d(&pool, a.pool, TmaDtype::kBF16, row_len, t.hidden_row, 1, 2ull * row_len, 0, 64, t.box, true);
  if (e != cudaSuccess) return e;
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(ragged_tiled_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  return launch_pdl(ragged_tiled_kernel, dim3(p.grid), dim3(kRtThreads), smem, stream, queries, pool, t);
}

}  // namespace ds41
