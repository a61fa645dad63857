// Attention of a ragged pass on tcgen05: bf16, up to 256 values of a key and of a value, pages of 16, 32, 64 or 128 tokens or whole 128s.
// Values of more than 128 columns are two units' each, which both make the scores: beside two tiles' scores tensor memory has no place for
// two results of 256.  (It has for one tile's, with two places for its scores: a form that is not built.)  Copies are as high as a page,
// or 128; pages of other sizes could come in copies of their greatest common divisor with 128, which is not built either.
//
// The queries of one key/value head are packed: the (token, head) pairs of a block's tokens are the rows of a tensor-core tile, so that a
// tile of keys and values is read once for all of them.  A CTA has two tiles of 128 rows.  A block of many tokens fills both, which then
// walk the same keys; a block of a few rows (decode) has them twice, and its two copies take the key tiles in turn.  Either way one
// tile's softmax runs while the tensor core works on the other's products.
//   warps 0-3, 4-7 : softmax of tile 0 / 1 (one thread per row), results
//   warp 8         : TMA producer: queries, keys and values, 128 positions at a time, page by page, a lane per copy
//   warps 9, 10    : tcgen05.mma issue for tile 0 / 1: S = Q K^T into TMEM, O += P V with P read from TMEM where it replaces its S, the
//                    first 96 keys' share while the others' weights are made
//   warp 11        : zeros in place of values that no row of the unit sees: their weights are zeros, but they may hold anything
//
// With x = scale * log2(e) * q.k a row's result is sum 2^(x - m) v / sum 2^(x - m) over the keys that it sees.
// The running maximum is raised when it grew by more than 2^8 only, so the accumulated output is rarely rescaled, and a tile's weights
// need not wait for its maximum.  P is rounded to bf16 as the operand of the second product; the sums take the unrounded weights.
//
// A CTA walks the units blockIdx.x, 2 * grid - 1 - blockIdx.x, ... of a list with the longest first; all roles but the softmax run ahead.
//
// What bounds it.  A pair of tiles takes 128 keys of 128 and 128 values in 3400 cycles, where the tensor core needs 2048, the exponentials
// 2048 and shared memory 2048: S and P share a place in tensor memory, which holds no second one beside two results of 128 columns, so that
// a tile's scores, softmax (2000), weights and products (600), and what tells one of the other (400) are a chain.  8192 tokens of 32 and 8
// heads: 490 us at 1.66 GHz, 550 to 575 at the 1.5 that the power limit leaves (1.0 PFLOP/s; tensor pipe 51 %, exponentials 51 %).  Decode over
// long contexts is bound by memory: 64 requests of up to 8192, 1.6 GB, 272 to 290 us, 5.6 to 6.0 TB/s; 16 x 16384 161 to 165 us, 6.5 to
// 6.7 TB/s; one of 131072 88 us.  Of fewer or shorter ones units' begin and end are a larger share: 40 x 4000, 655 MB, 137 us, 4.8 TB/s;
// 16 x 4000, 262 MB, 49 to 59 us.
// A unit begins and ends with 4.5 us (256 rows) or 2 us (decode), which short windows pay: 200 requests with 1024 + 4 positions 183 us,
// 846 MB, 12 % more than these for pages' ends.  4 requests of 300: 9.7 us.
//
// Two tiles of 128 rows x 128 keys, not 64 keys with two places for S: the products of 64 keys read the queries twice as often, and the
// tensor core alone took 3280 cycles a pair instead of 2554.  Decode as rows of a tile, not with the keys along its rows: those took 0.80 instead of
// 0.92 us a tile on a quiet machine and as long as the memory on a busy one, 2 us more a unit, and the registers that it needs slowed the
// other units down by 8 %; with warp-level products (16 rows, a warp's 16 keys of each tile) 642 instead of 300 us.
#include <cuda.h>

#include <atomic>

#include "ds41_prefix.cuh"
#include "ds41_ragged.cuh"
#include "ds41_tma.h"

namespace ds41 {

constexpr int kRtThreads = 384;
constexpr int kRtTile = 128, kRtKeys = 128;    // rows of a tile, keys of a tile
constexpr int kRtChunk = kRtTile * 128;        // bytes of 128 rows x 64 bf16 columns
constexpr int kRtKeyChunk = kRtKeys * 128;     // of its keys
constexpr int kRtStages = 4, kRtTurnRows = 64;

struct TiledParams {
  ds41_ragged_attend_args a;
  ds41_ragged_pass p;
  int group, per_tile;       // query heads of a key/value head, tokens of a tile
  int kd, vc;                // 64-column chunks of a key and a value
  int k_stages, v_stages;
  int box;                   // rows of a copy
  bool wide_out;             // a row of the result begins at 32 bytes
  int hidden_row;            // beyond the pool: reads as zeros
  float scale_log2;
};

struct TiledShared {
  uint64_t q_full, q_free;                     // queries are there; the unit's last scores are done
  uint64_t k_full[kRtStages], k_empty[kRtStages], v_full[kRtStages], v_empty[kRtStages];
  uint64_t v_clean[kRtStages];                 // places that nobody sees are zeros
  // per tile:
  uint64_t s_full[2];                          // S complete, and every product before it
  uint64_t p_full[2][2];                       // P written, O rescaled: of the first 96 keys, of the others
  uint64_t o_full[2];                          // the unit's last product is complete
  uint64_t half_full, half_read[2];            // the second tile's half of a unit whose keys were taken in turn
  float2 half_ml[kRtTurnRows];
  uint32_t tmem;
  int flag[2];
  int busy[4];                                 // per scheduler: one of its two softmax warps is at its exponentials
};

// Two products of 16 columns of K each (see umma4_ts).
template <int BSTEP>
__device__ __forceinline__ void umma2_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b32 x;\n\t.reg .b64 y;\n\t"
      "setp.eq.b32 q, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, q;\n\t"
      "add.s32 x, %1, 8;\n\tadd.s64 y, %2, %4;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "n"(BSTEP)
      : "memory");
}
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
  if (i + static_cast<int>(gridDim.x) < t.p.max_units)   // one of the next ones, or near it
    asm volatile("prefetch.global.L2 [%0];" ::"l"(t.p.units + 1ll * (i + static_cast<int>(gridDim.x)) * kRaggedInts));
  x.u = ragged_unit(t.p, i);
  const RaggedUnit& u = x.u;
  x.turns = u.tokens * t.group <= t.p.turn_rows;
  x.tok0 = x.turns ? u.tokens : (u.tokens + 1) / 2;
  x.walk = ragged_walk(u.pos0, u.pos0 + u.tokens - 1, t.p.window, t.p.first, Runs{t.box - 1});
  if (x.turns) {
    x.n[0] = (u.tiles + 1) / 2;
    x.n[1] = u.tiles / 2;
  } else {
    const int seen = u.pos0 + x.tok0 - x.walk.shift;                     // places up to tile 0's last row
    x.n[0] = min(max((seen + kRtKeys - 1) / kRtKeys - u.tile0, 0), u.tiles);
    x.n[1] = u.tokens > x.tok0 ? u.tiles : 0;
  }
  return x;
}

// The unit of a CTA's turn: the list goes back and forth.
__device__ __forceinline__ int unit_at(int turn) {
  return turn * static_cast<int>(gridDim.x) +
         (turn & 1 ? static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float largest(const uint32_t (&v)[32]) {
  auto f = [&](int k) { return __uint_as_float(v[k]); };
  float x[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    x[c] = max3(f(c), f(2 + c), f(4 + c));
#pragma unroll
    for (int k = 6; k + 2 < 32; k += 4) x[c] = max3(x[c], f(k + c), f(k + 2 + c));
  }
  return fmaxf(max3(x[0], f(30), f(31)), x[1]);
}
// The wait as something that the loaded registers depend on.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29])
               :: "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void mbar_arrive_if(bool issue, uint64_t* bar) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}"
               ::"r"(smem_u32(bar)), "r"(static_cast<uint32_t>(issue))
               : "memory");
}
// The lowest n bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// A scheduler's two softmax warps take turns at the exponentials: at the same time they would take each as long as both after one another,
// and the tensor core would have both tiles' products at once, and none afterwards.  Who has waited long enough goes on without.
__device__ __forceinline__ void take_turn(int* busy, int lane) {
  if (lane == 0) {
    const uint32_t at = smem_u32(busy);
    for (int i = 0, was = 1; i < 1024 && was != 0; ++i) asm volatile("atom.shared.cas.b32 %0, [%1], 0, 1;" : "=r"(was) : "r"(at) : "memory");
  }
  __syncwarp();
}
__device__ __forceinline__ void end_turn(int* busy, int lane) {
  __syncwarp();
  asm volatile("{\n\t.reg .pred q;\n\tsetp.eq.b32 q, %1, 0;\n\t@q st.shared.b32 [%0], 0;\n\t}" ::"r"(smem_u32(busy)), "r"(lane) : "memory");
}
// All lanes, or one thread by itself.
#define WARP_WAIT(bar, parity, where) (__all_sync(0xffffffffu, mbar_wait(bar, parity, t.p.status, where)) != 0)

__global__ void __launch_bounds__(kRtThreads, 1)
ragged_tiled_kernel(const __grid_constant__ CUtensorMap queries, const __grid_constant__ CUtensorMap pool,
                    const __grid_constant__ TiledParams t) {
  extern __shared__ uint8_t rt_raw[];
  uint8_t* smem = rt_raw + ((1024u - (smem_u32(rt_raw) & 1023u)) & 1023u);
  const int q_bytes = t.kd * kRtChunk, k_bytes = t.kd * kRtKeyChunk, v_bytes = t.vc * kRtKeyChunk;
  uint8_t* s_q = smem;                                   // two tiles
  uint8_t* s_k = s_q + 2 * q_bytes;
  uint8_t* s_v = s_k + t.k_stages * k_bytes;
  TiledShared& sh = *reinterpret_cast<TiledShared*>(s_v + t.v_stages * v_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int dp = t.p.dim, vp = t.p.vdim / t.p.v_parts;

  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_free, 2);                            // the products of either tile
    for (int i = 0; i < kRtStages; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 2);                      // the products of either tile, or that they do not take it
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_clean[i], 1);
      mbar_init(&sh.v_empty[i], 3);                      // the same, and the cleaner
    }
    mbar_init(&sh.half_full, 4);
    for (int i = 0; i < 4; ++i) sh.busy[i] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i][0], 4);
      mbar_init(&sh.p_full[i][1], 4);
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
    // Not before the allocation: a CTA of the next kernel with tensor memory of its own could take some here first, and would then wait for
    // this kernel's end, which waits for the memory.
    pdl_launch_dependents();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  pdl_wait();
  asm volatile("prefetch.global.L1 [%0];" ::"l"(t.p.units + 1ll * min(static_cast<int>(blockIdx.x), t.p.max_units - 1) * kRaggedInts));
  const int units = t.p.header[0];

  if (warp == 8) {
    // this lane's copies of a tile of keys and of one of values: some rows of one chunk of columns
    const int boxes = kRtKeys / t.box, k_box = lane / t.kd, k_chunk = lane - k_box * t.kd, v_box = lane / t.vc, v_chunk = lane - v_box * t.vc;
    const bool k_copies = k_box < boxes, v_copies = v_box < boxes;
    uint8_t *const k_to = s_k + k_chunk * kRtKeyChunk + k_box * t.box * 128, *const v_to = s_v + v_chunk * kRtKeyChunk + v_box * t.box * 128;
    int k_count = 0, v_count = 0, ks = 0, vs = 0, done = 0, halves = 0, v_row = 0, v_col = 0;
    uint32_t k_phase = 1, v_phase = 1;
    bool ok = true, behind = false;
    // values follow the keys one tile behind: by then their place is free as well
    auto values = [&]() {
      ok = WARP_WAIT(&sh.v_empty[vs], v_phase, 603);
      if (!ok) return;
      if (lane == 0) mbar_expect_tx(&sh.v_full[vs], v_bytes);
      __syncwarp();
      if (v_copies) tma_load_3d(v_to + vs * v_bytes, &pool, &sh.v_full[vs], v_col, v_row, 0);
      ++v_count;
      if (++vs == t.v_stages) {
        vs = 0;
        v_phase ^= 1;
      }
    };
    for (int turn = 0; unit_at(turn) < units && ok; ++turn) {
      const TiledUnit x = tiled_unit(t, unit_at(turn));
      const int n = x.u.tiles;
      auto locate = [&](int s, int box, bool copies) {
        const int place = (x.u.tile0 + s) * kRtKeys + box * t.box, pos = place < x.walk.lead ? place : place + x.walk.shift;
        const int pg = pos / t.p.page_tokens;
        const int id = copies && place < x.walk.places && pg < t.a.max_pages
                           ? __ldg(t.a.page_table + 1ll * x.u.slot * t.a.max_pages + pg) : -1;
        return static_cast<unsigned>(id) < static_cast<unsigned>(t.a.n_pages) ? id * t.p.page_tokens + (pos - pg * t.p.page_tokens)
                                                                              : t.hidden_row;
      };
      auto load_queries = [&]() {
        ok = WARP_WAIT(&sh.q_free, (done & 1) ^ 1, 600);
        // the second tile's place holds halves of units that went in turns
        for (int h = max(0, halves - 2); h < halves && ok && !x.turns; ++h) ok = WARP_WAIT(&sh.half_read[h & 1], (h >> 1) & 1, 601);
        if (!ok) return;
        const bool second = !x.turns && x.u.tokens > x.tok0;
        if (lane == 0) mbar_expect_tx(&sh.q_full, (second ? 2 : 1) * t.kd * t.per_tile * t.group * 128);
        __syncwarp();
        if (lane < (second ? 2 : 1) * t.kd) {
          const int k = lane / t.kd, c = lane - k * t.kd;
          tma_load_3d(s_q + k * q_bytes + c * kRtChunk, &queries, &sh.q_full, 64 * c, x.u.head * t.group, x.u.row0 + k * x.tok0);
        }
        ++done;
        if (x.turns && n > 1) ++halves;
      };
      // The first unit's queries before its keys; later ones behind as many key tiles as there are places for, as those do not wait for
      // the last unit's queries.
      const int q_after = done == 0 ? 0 : min(n, t.k_stages);
      if (n > 0 && q_after == 0) load_queries();
      int k_next = n > 0 ? locate(0, k_box, k_copies) : 0, v_next = n > 0 ? locate(0, v_box, v_copies) : 0;
      for (int s = 0; s < n && ok; ++s) {
        const int k_row = k_next, v_later = v_next;
        if (s + 1 < n) {
          k_next = locate(s + 1, k_box, k_copies);
          v_next = locate(s + 1, v_box, v_copies);
        }
        ok = WARP_WAIT(&sh.k_empty[ks], k_phase, 602);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&sh.k_full[ks], k_bytes);
        __syncwarp();
        if (k_copies) tma_load_3d(k_to + ks * k_bytes, &pool, &sh.k_full[ks], x.u.head * dp + 64 * k_chunk, k_row, 0);
        ++k_count;
        if (++ks == t.k_stages) {
          ks = 0;
          k_phase ^= 1;
        }
        if (behind) values();
        if (!ok) break;
        behind = true;
        v_row = v_later;
        v_col = t.p.kv_heads * dp + x.u.head * t.p.vdim + x.u.v0 + 64 * v_chunk;
        if (s + 1 == q_after) load_queries();
      }
    }
    if (ok && behind) values();
    if (!ok && lane == 0) {                              // something gave up: the copies under way land before the memory goes away
      auto drain = [](uint64_t* bar, uint32_t parity) {
        for (int i = 0; i < (1 << 18) && !mbar_test_wait(bar, parity); ++i) {
        }
      };
      if (done > 0) drain(&sh.q_full, (done - 1) & 1);
      for (int b = max(0, k_count - t.k_stages); b < k_count; ++b) drain(&sh.k_full[b % t.k_stages], (b / t.k_stages) & 1);
      for (int b = max(0, v_count - t.v_stages); b < v_count; ++b) drain(&sh.v_full[b % t.v_stages], (b / t.v_stages) & 1);
    }
  } else if (warp == 9 || warp == 10) {
    // one thread: votes and the like between two products cost as much as the products
    if (elect_one()) {
      const int i = warp - 9;
      const uint32_t idesc_s = umma_idesc(kRtTile, kRtKeys, 1u, 1u), idesc_pv = umma_idesc_bmn(kRtTile, vp, 1u, 1u);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q)), k_desc = umma_desc_sw128(smem_u32(s_k));
      const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(s_v), kRtKeyChunk, 1024);
      const uint64_t k_step = k_bytes / 16, v_step = v_bytes / 16;
      const int whole = dp / 64, rest = dp / 16 - 4 * whole;
      const uint32_t o_t = tmem + 256 + i * 128;
      int begun = 0, done = 0;                           // units, tiles
      int ks = 0, vs = 0;                                // places of the next keys and values, and their phases
      uint32_t k_phase = 0, v_phase = 0;
      bool ok = true;
      auto next_k = [&]() {
        if (++ks == t.k_stages) {
          ks = 0;
          k_phase ^= 1;
        }
      };
      auto next_v = [&]() {
        if (++vs == t.v_stages) {
          vs = 0;
          v_phase ^= 1;
        }
      };
      // tiles of the other one's, up to `upto`: every place of the rings is watched, or its phases could be mistaken
      auto skip_k = [&](int& at, int upto) {
        for (; at < upto && ok; ++at) {
          ok = mbar_wait(&sh.k_full[ks], k_phase, t.p.status, 610);
          if (ok) mbar_arrive(&sh.k_empty[ks]);
          next_k();
        }
      };
      auto skip_v = [&](int& at, int upto) {
        for (; at < upto && ok; ++at) {
          ok = mbar_wait(&sh.v_full[vs], v_phase, t.p.status, 611);
          if (ok) mbar_arrive(&sh.v_empty[vs]);
          next_v();
        }
      };
      for (int turn = 0; unit_at(turn) < units && ok; ++turn) {
        const TiledUnit x = tiled_unit(t, unit_at(turn));
        const int n = x.n[i], first = x.turns ? i : 0, step = x.turns ? 2 : 1;
        if (x.u.tiles == 0) continue;
        const int low = ragged_low(x.u.pos0, t.p.window) - x.walk.shift;
        const uint64_t q = q_desc + (i && !x.turns ? static_cast<uint64_t>(q_bytes / 16) : 0u);
        const uint32_t s_t = tmem + i * 128;
        int k_at = 0, v_at = 0;
        auto keys = [&](int j) {                         // of its tile j
          skip_k(k_at, first + j * step);
          if (ok) ok = mbar_wait(&sh.k_full[ks], k_phase, t.p.status, 612);
        };
        auto scores = [&](int j) {
          uint64_t a = q, b = k_desc + ks * k_step;
#pragma unroll 1
          for (int c = 0; c < whole; ++c, a += kRtChunk / 16, b += kRtKeyChunk / 16) umma4_ss<2, 2>(s_t, a, b, idesc_s, c);
#pragma unroll 1
          for (int k = 0; k < rest; ++k) umma_bf16(s_t, a + 2 * k, b + 2 * k, idesc_s, whole > 0 || k > 0);
          tc_commit(&sh.s_full[i]);
          tc_commit(&sh.k_empty[ks]);
          ++k_at;
          next_k();
          if (j == n - 1) tc_commit(&sh.q_free);
        };
        ok = mbar_wait(&sh.q_full, begun & 1, t.p.status, 613);
        ++begun;
        if (ok && n == 0) mbar_arrive(&sh.q_free);
        if (ok && n > 0) {
          keys(0);
          if (!ok) break;
          tc_fence_after();
          scores(0);
        }
        for (int j = 0; j < n && ok; ++j) {
          const int s = first + j * step, place0 = (x.u.tile0 + s) * kRtKeys;
          const bool unseen = place0 + kRtKeys > x.walk.places || max(place0, t.p.first) < min(place0 + kRtKeys, low);
          skip_v(v_at, s);
          // they have landed, so that the cleaner is past the ones before them in this place; only then can its phase be told
          if (ok) ok = mbar_wait(&sh.v_full[vs], v_phase, t.p.status, 614);
          if (ok && unseen) ok = mbar_wait(&sh.v_clean[vs], v_phase, t.p.status, 617);
          if (j + 1 < n) keys(j + 1);
          const uint64_t v = v_desc + vs * v_step;
          if (ok) ok = mbar_wait(&sh.p_full[i][0], done & 1, t.p.status, 615);
          if (!ok) break;
          tc_fence_after();
          umma4_ts<128>(o_t, s_t, v, idesc_pv, j > 0);
          umma2_ts<128>(o_t, s_t + 32, v + 512, idesc_pv);
          ok = mbar_wait(&sh.p_full[i][1], done & 1, t.p.status, 616);
          if (!ok) break;
          tc_fence_after();
          umma2_ts<128>(o_t, s_t + 48, v + 768, idesc_pv);
          if (j + 1 < n) scores(j + 1);                  // over the P that these products read
          else tc_commit(&sh.o_full[i]);
          tc_commit(&sh.v_empty[vs]);
          ++done;
          ++v_at;
          next_v();
        }
        for (int s = min(k_at, v_at); s < x.u.tiles && ok; ++s) {
          skip_k(k_at, s + 1);
          skip_v(v_at, s + 1);
        }
      }
    }
    __syncwarp();
  } else if (warp == 11) {
    int vs = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int turn = 0; unit_at(turn) < units && ok; ++turn) {
      const TiledUnit x = tiled_unit(t, unit_at(turn));
      const int low = ragged_low(x.u.pos0, t.p.window) - x.walk.shift;
      for (int s = 0; s < x.u.tiles; ++s) {
        const int place0 = (x.u.tile0 + s) * kRtKeys;
        ok = WARP_WAIT(&sh.v_full[vs], phase, 620);
        if (!ok) break;
        // places [a, b) and [c, 128) of the tile are seen by nobody
        const int a = max(0, t.p.first - place0), b = min(kRtKeys, low - place0), c = min(kRtKeys, x.walk.places - place0);
        if (a < b || c < kRtKeys) {
          for (int k = 0; k < t.vc; ++k) {
            uint8_t* v = s_v + vs * v_bytes + k * kRtKeyChunk + 16 * (lane & 7);
            for (int r = a + (lane >> 3); r < b; r += 4) *reinterpret_cast<uint4*>(v + r * 128) = make_uint4(0, 0, 0, 0);
            for (int r = c + (lane >> 3); r < kRtKeys; r += 4) *reinterpret_cast<uint4*>(v + r * 128) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sh.v_clean[vs]);
          mbar_arrive(&sh.v_empty[vs]);
        }
        if (++vs == t.v_stages) {
          vs = 0;
          phase ^= 1;
        }
      }
    }
  } else {
    // Where a wait gave up, `ok` stays false and later ones are left out, but every barrier that warps share is reached.
    const int i = warp >> 2, quad = warp & 3, mine = quad * 32 + lane, tid = mine;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_t = tmem + lanes + i * 128, o_t = tmem + lanes + 256 + i * 128;
    const int mine_tok = mine / t.group, mine_head = mine - mine_tok * t.group;
    const float2 scale2 = make_float2(t.scale_log2, t.scale_log2);
    // a row of the second tile's half, each beginning at another column, so that neighbours do not meet in a bank
    float4* const half = reinterpret_cast<float4*>(s_q + q_bytes) + mine * (vp / 4);
    const int turned = mine % (vp / 4);
    int tiles = 0, outputs = 0, halves = 0;
    bool ok = true;
    for (int turn = 0; unit_at(turn) < units; ++turn) {
      // Of this thread's row: visible are the places [0, a) and [b, e); of all of its warp's rows up to a_all, from b_all to e_all.
      int n, a, b, e, a_all, b_all, e_all, place0, place_step;
      bool live;
      float sink = -INFINITY, gate = 0.f;                // asked for long before they are needed
      {
        const TiledUnit x = tiled_unit(t, unit_at(turn));
        const RaggedUnit& u = x.u;
        if (unit_at(turn + 1) < units) {                 // the next one, which may lie in two lines
          const int* next = t.p.units + 1ll * unit_at(turn + 1) * kRaggedInts;
          asm volatile("prefetch.global.L1 [%0];" ::"l"(next));
          asm volatile("prefetch.global.L1 [%0];" ::"l"(next + kRaggedInts - 1));
        }
        if (u.tiles == 0) {
          for (int r = threadIdx.x; r < u.tokens * t.group; r += 256) {
            uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(t.a.out) + (u.row0 + r / t.group) * t.a.out_row +
                                                  1ll * (u.head * t.group + r % t.group) * t.p.vdim + u.v0);
            for (int c = 0; c < vp / 8; ++c) out[c] = make_uint4(0, 0, 0, 0);
          }
          continue;
        }
        const int toks = x.turns ? u.tokens : (i ? u.tokens - x.tok0 : x.tok0);
        live = mine_tok < toks;
        const int pos = u.pos0 + (i && !x.turns ? x.tok0 : 0) + min(mine_tok, toks - 1);
        e = pos + 1 - x.walk.shift;
        b = ragged_low(pos, t.p.window) - x.walk.shift;
        a = min(t.p.first, e);
        b_all = __shfl_sync(0xffffffffu, b, 31);
        e_all = __shfl_sync(0xffffffffu, e, 0);
        a_all = min(t.p.first, e_all);
        n = x.n[i];
        place0 = (u.tile0 + (x.turns ? i : 0)) * kRtKeys;
        place_step = x.turns ? 2 * kRtKeys : kRtKeys;
        const int h = u.head * t.group + mine_head, row = u.row0 + (i && !x.turns ? x.tok0 : 0) + mine_tok;
        if (live && t.a.sink != nullptr) sink = t.a.sink[h] * kLog2E;
        if (live && t.a.gate.data != nullptr) gate = proj_at(t.a.gate, row, h);
      }
      const bool idle = !__any_sync(0xffffffffu, live);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, ++tiles, place0 += place_step) {
        if (ok) ok = WARP_WAIT(&sh.s_full[i], tiles & 1, 630 + i);
        const bool work = ok && !idle;
        // Weights are relative to the maximum so far.  Where the tile's is above it by more than 2^8, it is raised and they are taken once
        // more.
        uint32_t x[2][32], w[32];
        float2 sums[2], neg2;
        auto begin = [&]() {
          const float neg = m == -INFINITY ? 0.f : -m;
          neg2 = make_float2(neg, neg);
          sums[0] = sums[1] = make_float2(0.f, 0.f);
        };
        auto weights = [&](const uint32_t (&v)[32], int from, int to, int at) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            if (k < from || k >= to) continue;
            float2 y = fma2(make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), scale2, neg2);
            y.x = ex2_approx(y.x);
            y.y = ex2_approx(y.y);
            sums[k & 1] = add2(sums[k & 1], y);
            const __nv_bfloat162 q = __floats2bfloat162_rn(y.x, y.y);
            w[at + k] = *reinterpret_cast<const uint32_t*>(&q);
          }
        };
        if (work) {
          tc_fence_after();
          const bool edge = (place0 < b_all || place0 + kRtKeys > e_all) && place0 + kRtKeys > a_all;
          if (edge) {
            float top = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < kRtKeys; c += 32) {
              const int at = place0 + c;
              if (j > 0 && ((at >= b_all && at + 32 <= e_all) || at + 32 <= a_all)) continue;       // all of it is seen
              tmem_ld_32x32(s_t + c, x[0]);
              const uint32_t seen = low_bits(a - at) | (low_bits(e - at) & ~low_bits(b - at));
              tmem_wait_ld(x[0]);
#pragma unroll
              for (int k = 0; k < 32; ++k) x[0][k] = seen >> k & 1 ? x[0][k] : 0xff800000u;
              top = fmaxf(top, largest(x[0]));
              tmem_st_32x32(s_t + c, x[0]);
            }
            tmem_wait_st();
            if (j == 0) m = top * t.scale_log2;
          }
          tmem_ld_32x32(s_t, x[0]);
          tmem_ld_32x32(s_t + 32, x[1]);
          take_turn(&sh.busy[quad], lane);
          tmem_wait_ld(x[0]);
          tmem_wait_ld(x[1]);
          if (j == 0 && !edge) m = fmaxf(largest(x[0]), largest(x[1])) * t.scale_log2;      // of the first half: seldom much less
          begin();
          weights(x[0], 0, 16, 0);
          float top = largest(x[0]);
          tmem_ld_32x32(s_t + 64, x[0]);
          weights(x[1], 0, 16, 16);
          top = fmaxf(top, largest(x[1]));
          tmem_ld_32x32(s_t + 96, x[1]);
          tmem_wait_ld(x[0]);
          tmem_wait_ld(x[1]);
          top = fmaxf(top, fmaxf(largest(x[0]), largest(x[1]))) * t.scale_log2;
          const bool grow = top > m + 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            // O and the sum follow; the products before this tile's are complete
            const float m_new = grow ? top : m, keep = grow ? (m == -INFINITY ? 0.f : ex2_approx(m - m_new)) : 1.f;
            l *= keep;
            m = m_new;
#pragma unroll 1
            for (int c = 0; c < vp && j > 0; c += 16) {
              uint32_t o[16];
              tmem_ld_32x16(o_t + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
              tmem_st_32x16(o_t + c, o);
            }
            tmem_ld_32x32(s_t, x[0]);
            tmem_ld_32x32(s_t + 32, x[1]);
            tmem_wait_ld(x[0]);
            tmem_wait_ld(x[1]);
            begin();
            weights(x[0], 0, 16, 0);
            weights(x[1], 0, 16, 16);
            tmem_ld_32x32(s_t + 64, x[0]);
            tmem_ld_32x32(s_t + 96, x[1]);
            tmem_wait_ld(x[0]);
            tmem_wait_ld(x[1]);
          }
          tmem_st_32x32(s_t, w);                         // columns whose S this thread has read
          weights(x[0], 0, 16, 0);
          tmem_st_32x16(s_t + 32, reinterpret_cast<uint32_t(&)[16]>(w[0]));
          end_turn(&sh.busy[quad], lane);
          weights(x[1], 0, 8, 16);
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        mbar_arrive_if(ok && lane == 0, &sh.p_full[i][0]);
        if (work) {
          weights(x[1], 8, 16, 16);
          tmem_st_32x16(s_t + 48, reinterpret_cast<uint32_t(&)[16]>(w[16]));
          l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        mbar_arrive_if(ok && lane == 0, &sh.p_full[i][1]);
      }
      const TiledUnit x = tiled_unit(t, unit_at(turn));  // once more: it takes registers
      const RaggedUnit& u = x.u;
      const int first_tok = i && !x.turns ? x.tok0 : 0, toks = x.turns ? u.tokens : (i ? u.tokens - x.tok0 : x.tok0);
      const int row = u.row0 + first_tok + mine_tok, h = u.head * t.group + mine_head;
      const bool placed = live && t.p.row_place[row] >= 0;
      if (n > 0) {
        if (ok) ok = WARP_WAIT(&sh.o_full[i], outputs & 1, 634 + i);
        ++outputs;
        tc_fence_after();
      }
      if (x.turns && i == 1) {
        // this half goes to the first tile's warps
        if (u.tiles > 1) {
          if (halves > 0 && ok) ok = WARP_WAIT(&sh.half_read[(halves - 1) & 1], ((halves - 1) >> 1) & 1, 634);
          if (!idle) {
            int at = turned;
#pragma unroll 1
            for (int c = 0; c < vp; c += 32) {             // behind the last column lies something of no use
              uint32_t o[32];
              __syncwarp();
              tmem_ld_32x32(o_t + c, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                if (live && c + 4 * k < vp) half[at] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                                                   __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                at = at + 1 < vp / 4 ? at + 1 : 0;
              }
            }
            if (live) sh.half_ml[mine] = make_float2(m, l);
          }
          tc_fence_before();
          ++halves;
          __syncwarp();
          mbar_arrive_if(lane == 0, &sh.half_full);
        }
        continue;
      }
      float w_own = 1.f, w_half = 0.f;                   // factors of both halves
      const bool joined = x.turns && u.tiles > 1;
      if (joined) {
        if (ok) ok = WARP_WAIT(&sh.half_full, halves & 1, 635);
        if (live) {
          const float2 ml = sh.half_ml[mine];
          const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top;
          w_own = ex2_approx(m - base);
          w_half = ex2_approx(ml.x - base);
          l = l * w_own + ml.y * w_half;
          m = top;
        }
      }
      float f = 1.f;
      long long cell = 0;
      if (u.pieces > 1) {
        cell = 1ll * u.cell + 1ll * u.piece * u.step + first_tok * t.group + mine;
        if (live) *reinterpret_cast<float2*>(t.p.part_ml + 2 * cell) = make_float2(m, l);
      } else if (live) {
        const float top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
        const float w = ex2_approx(m - base), den = l * w + (t.a.sink != nullptr ? ex2_approx(sink - base) : 0.f);
        f = w / den;
        if (t.a.gate.data != nullptr) f *= sigmoid_f32(gate);
      }
      w_own *= f;
      w_half *= f;
      if (!idle && n > 0) {
        float4* part = reinterpret_cast<float4*>(t.p.part_o + cell * vp);
        uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(t.a.out) + row * t.a.out_row + 1ll * h * t.p.vdim + u.v0);
        int at = turned;
#pragma unroll 1
        for (int c = 0; c < vp; c += 32, part += 8, out += 4) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_32x32(o_t + c, o);
          tmem_wait_ld(o);
          if (joined) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 z = live ? half[at] : make_float4(0.f, 0.f, 0.f, 0.f);
              at = at + 1 < vp / 4 ? at + 1 : 0;
              o[4 * k] = __float_as_uint(__uint_as_float(o[4 * k]) * w_own + z.x * w_half);
              o[4 * k + 1] = __float_as_uint(__uint_as_float(o[4 * k + 1]) * w_own + z.y * w_half);
              o[4 * k + 2] = __float_as_uint(__uint_as_float(o[4 * k + 2]) * w_own + z.z * w_half);
              o[4 * k + 3] = __float_as_uint(__uint_as_float(o[4 * k + 3]) * w_own + z.w * w_half);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * w_own);
          }
          // a sector or two of L2 at a time
          if (!live) {
          } else if (u.pieces > 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c + 8 * k < vp) store8(reinterpret_cast<float*>(part + 2 * k), reinterpret_cast<const float(&)[8]>(o[8 * k]));
          } else {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const __nv_bfloat162 q = __floats2bfloat162_rn(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1]));
              w[k] = placed ? *reinterpret_cast<const uint32_t*>(&q) : 0u;
            }
            if (t.wide_out) {
              store8(reinterpret_cast<float*>(out), reinterpret_cast<const float(&)[8]>(w[0]));
              if (c + 16 < vp) store8(reinterpret_cast<float*>(out + 2), reinterpret_cast<const float(&)[8]>(w[8]));
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (c + 8 * k < vp) out[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      if (joined) {
        fence_async_smem();
        __syncwarp();
        mbar_arrive_if(lane == 0, &sh.half_read[halves & 1]);
        ++halves;
      }
      if (u.pieces > 1 && ragged_last(t.p.counters + u.counter + i, u.pieces, tid == 0, 1 + i, kRtTile, &sh.flag[i]))
        ragged_join<__nv_bfloat16>(t.p, t.a, u, first_tok * t.group, (first_tok + toks) * t.group, quad, 4);
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Places of the rings and the launch's shared memory; 0: the sizes do not fit.
inline int tiled_smem(TiledParams& t) {
  t.kd = (t.p.dim + 63) / 64;
  t.vc = (t.p.vdim / t.p.v_parts + 63) / 64;
  const int q = 2 * t.kd * kRtChunk, k = t.kd * kRtKeyChunk, v = t.vc * kRtKeyChunk;
  constexpr int kFixed = 1024 + static_cast<int>(sizeof(TiledShared)), kLimit = 227 * 1024;
  t.k_stages = t.v_stages = 1;
  int left = kLimit - kFixed - q - k - v;
  if (left < 0) return 0;
  while (true) {                                         // values first: they are held until their weights are there
    if (t.v_stages <= t.k_stages && t.v_stages < kRtStages && left >= v) ++t.v_stages, left -= v;
    else if (t.k_stages < kRtStages && left >= k) ++t.k_stages, left -= k;
    else if (t.v_stages < kRtStages && left >= v) ++t.v_stages, left -= v;
    else break;
  }
  return kLimit - left;
}

cudaError_t launch_ragged_tiled(const ds41_ragged_attend_args& a, const ds41_ragged_pass& p, cudaStream_t stream) {
  TiledParams t{};
  t.a = a;
  t.p = p;
  t.group = p.heads / p.kv_heads;
  if (p.f32 || t.group > kRtTile || p.vdim > 128 * p.v_parts || p.key_tile != kRtKeys || p.page_tokens < 16 ||
      (p.page_tokens < kRtKeys ? kRtKeys % p.page_tokens : p.page_tokens % kRtKeys))
    return cudaErrorInvalidValue;
  t.per_tile = kRtTile / t.group;
  if (p.unit_tokens != 2 * t.per_tile) return cudaErrorInvalidValue;
  const int smem = tiled_smem(t);
  if (smem == 0) return cudaErrorInvalidValue;
  t.box = p.page_tokens < kRtKeys ? p.page_tokens : kRtKeys;
  if (kRtKeys / t.box * (t.kd > t.vc ? t.kd : t.vc) > 32) return cudaErrorInvalidValue;
  // the results of tiles in turns have to fit the second tile's place
  if (p.turn_rows > kRtTurnRows || p.turn_rows * 4 * (p.vdim / p.v_parts) > t.kd * kRtChunk) return cudaErrorInvalidValue;
  t.wide_out = !((reinterpret_cast<uintptr_t>(a.out) | 2 * a.out_row) & 31);
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
