// Parts of grouped-query attention for rows that share prefixes, on tcgen05.
//
// The queries of one key/value head are packed: (row, head) pairs of a unit's rows are the 128 rows of a tensor-core tile, so that a
// tile of keys and values is read once for all of them and the products have the shape of a prompt's.  A CTA has two tiles: units
// come in twos, and where both of them walk the same keys each copy serves two tiles.  One tile's softmax runs while the tensor core
// works on the other's products, and nothing but the order of the copies ties the two together.
//   warps 0-3, 4-7 : softmax of tile 0 / 1 (one thread per query), partial results
//   warps 8, 12    : TMA producers: key / value tiles of 64 positions, page by page
//   warps 9, 14    : tcgen05.mma issue for tile 0 / 1: S = Q K^T, O += P V with P in TMEM where it replaces its S.  S has two places,
//                    and the next tile's are asked for before this one's values.  200 rows of 32 heads over 16000 shared keys and up to
//                    700 own ones take 129 us so, 138 with one place for 128 keys (a tile's S, softmax and values are then a chain), and 185 with
//                    two places whose products one thread asked for: every step took it 800 cycles
//   warps 10, 11   : queries of tile 0 / 1, and what each of them sees
//   warp 13        : what the next units are and where their keys lie, for everybody (a ring of four)
// A CTA walks its units, and every role but the softmax runs ahead into the next ones: a request's own keys are a few tiles, which the
// chain of loads that a unit begins with (its description, its rows' positions, their pages, their queries) would take as long as.
// The running maximum is raised when it grew by more than 2^8 only; what leaves is (m, l, unnormalised O) in 32 bits.  P is rounded
// to bf16 as the operand of the second product; l sums the unrounded weights.
//
// What bounds it: 64 keys of two tiles take 2000 cycles, of which the tensor core works 1300 (the scores' two operands from shared memory
// 48 per 128 x 64 x 16, the values' 64) and the 128 exponentials of a scheduler's two warps 1024; the softmax warps are the longest chain.
// Letting them take turns at the exponentials, or taking a quarter of these by a polynomial, made steps of 1900 cycles and no call
// shorter.  A unit costs 1.4 us beside its keys and 0.1 us per row (queries in, results out); requests' own keys are tiles of a few live
// queries at the same price, and almost half of the call above (124 us with units dealt by these costs).
#include <cuda.h>

#include "ds41_group.cuh"
#include "ds41_mma.cuh"
#include "ds41_prefix.cuh"
#include "ds41_tma.h"

namespace ds41 {

constexpr int kPgThreads = 480;
constexpr int kPgTile = 128, kPgKeys = 64;     // queries of a tile, keys of a tile
constexpr int kPgChunk = kPgTile * 128;        // bytes of 128 queries x 64 bf16 columns
constexpr int kPgKeyChunk = kPgKeys * 128;     // of 64 keys
constexpr int kPgInfos = 4, kPgStages = 8;

struct PrefixGroupParams {
  const __nv_bfloat16* q;
  const int *page_table, *row_pos, *row_slot;
  long long ld_q;
  int heads, kv_heads, n, dp, vp, kd, vc, stages, shift;             // tiles of keys and of values: 2^shift
  int chunk, max_pages, page_tokens, n_pages, box, hidden_row;      // a row beyond the pool: reads as zeros
  int deep;                                                // all chunks of a box in one copy
  float scale_log2;
  int* status;
};

// What a CTA's two tiles do next, as the producer found it: unit t walks `tiles[t]` key tiles from `first[t]` on, and nobody sees
// `end[t]` or what follows.  both: they walk the same ones.  Key tiles inside [safe[t], safe_end[t]) have no place that nobody sees; of
// the places outside all are unseen, or it takes a look at the rows (gaps).
struct __align__(16) GroupWork {
  PrefixUnit unit[2];
  int first[2], end[2], tiles[2], base, both;              // base: number of the first key tile in the order of the copies
  int safe[2], safe_end[2], gaps[2];
  int row[2][32];                                          // pool rows of the first 32 boxes of their keys
};

// Number of key tile j of tile t in the order of the copies: one after the other, or in turn as long as both have some.
__device__ __forceinline__ int copy_index(bool both, int base, int least, int t, int j) {
  return base + (both ? j : j < least ? 2 * j + t : least + j);
}

struct GroupShared {                           // behind the tiles
  uint64_t info_full[kPgInfos], info_empty[kPgInfos];
  uint64_t k_full[kPgStages], k_empty[kPgStages], v_full[kPgStages], v_empty[kPgStages];
  // per tile:
  uint64_t q_full[2], q_empty[2];
  uint64_t s_full[2][2];                       // by place of S: complete (and every earlier MMA of the issuing thread)
  uint64_t p_full[2][2];                       // P written, O rescaled
  uint64_t o_next[2];                          // the unit's last product but one
  uint64_t o_full[2];                          // the unit's last product
  uint64_t v_here[2];                          // the values of a key tile with places that nobody sees, for the softmax
  int k_asked, v_asked;                        // copies under way or done: a place's barrier is at the phase of the last of these
  int v_place[2];                              // where in the ring those are
  uint32_t tmem, pad[3];
  GroupWork info[kPgInfos];
  int4 row[2][kPgTile];                        // of a unit's row: pass row, visible keys [y, z), cell
};

__global__ void __launch_bounds__(kPgThreads, 1)
prefix_group_kernel(const __grid_constant__ CUtensorMap keys, const __grid_constant__ CUtensorMap values, const PrefixGroupParams p,
                    const ds41_prefix_plan plan) {
  extern __shared__ uint8_t pg_raw[];
  uint8_t* smem = pg_raw + ((1024u - (smem_u32(pg_raw) & 1023u)) & 1023u);
  const int q_bytes = p.kd * kPgChunk, k_bytes = p.kd * kPgKeyChunk, v_bytes = p.vc * kPgKeyChunk;
  uint8_t* s_q = smem;                                   // two tiles
  uint8_t* s_k = s_q + 2 * q_bytes;
  uint8_t* s_v = s_k + p.stages * k_bytes;
  GroupShared& sh = *reinterpret_cast<GroupShared*>(s_v + p.stages * v_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPgInfos; ++i) {
      mbar_init(&sh.info_full[i], 1);
      mbar_init(&sh.info_empty[i], 14);                  // eight softmax warps, two of queries, two of copies, the products of either tile
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.q_full[i], 1);
      mbar_init(&sh.q_empty[i], 5);                      // four softmax warps, the products
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sh.s_full[i][b], 1);
        mbar_init(&sh.p_full[i][b], 4);
      }
      mbar_init(&sh.o_next[i], 1);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.v_here[i], 1);
    }
    for (int i = 0; i < kPgStages; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 2);                      // the products of either tile, or twice those of one
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 2);
    }
    sh.k_asked = sh.v_asked = 0;
    mbar_init_fence();
    tma_prefetch_desc(&keys);
    tma_prefetch_desc(&values);
  }
  if (warp == 9) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // The plan was copied to the device, not computed there by a kernel: it may be read before the wait.  Places behind the last unit
  // are empty units.
  const PrefixUnit first_a = prefix_unit(plan, min(2 * static_cast<int>(blockIdx.x), plan.max_units - 2));
  const PrefixUnit first_b = prefix_unit(plan, min(2 * static_cast<int>(blockIdx.x) + 1, plan.max_units - 1));
  const int turns = plan.turns[blockIdx.x];
  pdl_wait();

  bool ok = true;

  // lane i: pool row of box i of the 32 boxes from box u of a walk on
  auto locate = [&](int slot, int first, int end, int u) {
    const int key = first + (u + lane) * p.box, pg = key / p.page_tokens;
    const int id = key < end && pg < p.max_pages ? p.page_table[1ll * slot * p.max_pages + pg] : -1;
    return static_cast<unsigned>(id) < static_cast<unsigned>(p.n_pages) ? id * p.page_tokens + (key - pg * p.page_tokens) : p.hidden_row;
  };

  if (warp == 13) {
    int base = 0;
    for (int turn = 0; turn < turns; ++turn) {
      const int at = 2 * (static_cast<int>(blockIdx.x) + turn * static_cast<int>(gridDim.x));
      const PrefixUnit a = turn == 0 ? first_a : prefix_unit(plan, at), b = turn == 0 ? first_b : prefix_unit(plan, at + 1);
      // without chunks a walk begins at its first key: its pages are looked up together with its rows' positions
      int row_a = locate(a.slot, a.key0, a.key1, 0), row_b = locate(b.slot, b.key0, b.key1, 0);
      PrefixRows rows_a = prefix_rows(plan, a, p.row_pos, p.row_slot, p.chunk), rows_b = prefix_rows(plan, b, p.row_pos, p.row_slot, p.chunk);
      int first[2], end[2];
      prefix_span(a, rows_a, p.chunk, p.page_tokens, first[0], end[0]);
      prefix_span(b, rows_b, p.chunk, p.page_tokens, first[1], end[1]);
      const bool seen[2] = {first[0] < end[0], first[1] < end[1]};
      const bool both = b.rows > 0 && !a.tail && !b.tail && a.slot == b.slot && a.key0 == b.key0 && a.key1 == b.key1 &&
                        a.head == b.head && seen[0] && seen[1];
      if (both) {
        first[0] = first[1] = min(first[0], first[1]);
        end[0] = end[1] = max(end[0], end[1]);
      }
      // without chunks every place before `end` is seen by the row that stands last; with them, a row's window vouches for its tiles
      int safe[2] = {first[0], first[1]}, safe_end[2] = {end[0], end[1]}, gaps[2] = {0, 0};
      if (p.chunk > 0) {
        prefix_widest(rows_a, safe[0], safe_end[0]);
        prefix_widest(rows_b, safe[1], safe_end[1]);
        int low[2] = {max(rows_a.low, a.key0), max(rows_b.low, b.key0)};
        if (both) {
          const int t = safe_end[1] - safe[1] > safe_end[0] - safe[0];
          safe[0] = safe[1] = t ? safe[1] : safe[0];
          safe_end[0] = safe_end[1] = t ? safe_end[1] : safe_end[0];
          low[0] = low[1] = min(low[0], low[1]);
        }
        gaps[0] = low[0] < safe[0] || end[0] > safe_end[0];
        gaps[1] = low[1] < safe[1] || end[1] > safe_end[1];
      }
      // what lies behind the unit's keys is read as zeros
      if (safe_end[0] == a.key1) safe_end[0] = 0x7fffffff;
      if (safe_end[1] == b.key1) safe_end[1] = 0x7fffffff;
      if (first[0] != a.key0) row_a = locate(a.slot, first[0], end[0], 0);
      if (first[1] != b.key0) row_b = locate(b.slot, first[1], end[1], 0);
      if (first[0] + lane * p.box >= end[0]) row_a = p.hidden_row;
      if (first[1] + lane * p.box >= end[1]) row_b = p.hidden_row;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_empty[turn % kPgInfos], ((turn / kPgInfos) & 1) ^ 1, p.status, 459)) != 0;
      if (!ok) break;
      GroupWork& w = sh.info[turn % kPgInfos];
      const int tiles[2] = {(end[0] - first[0] + kPgKeys - 1) / kPgKeys, (end[1] - first[1] + kPgKeys - 1) / kPgKeys};
      w.row[0][lane] = row_a;
      w.row[1][lane] = row_b;
      if (lane < 2) {
        w.unit[lane] = lane ? b : a;
        w.first[lane] = lane ? first[1] : first[0];
        w.end[lane] = lane ? end[1] : end[0];
        w.tiles[lane] = lane ? tiles[1] : tiles[0];
        w.safe[lane] = lane ? safe[1] : safe[0];
        w.safe_end[lane] = lane ? safe_end[1] : safe_end[0];
        w.gaps[lane] = lane ? gaps[1] : gaps[0];
        w.base = base;
        w.both = both;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.info_full[turn % kPgInfos]);
      base += both ? tiles[0] : tiles[0] + tiles[1];
    }
  } else if (warp == 8 || warp == 12) {
    const bool second = warp == 12;                      // values
    const int boxes = kPgKeys / p.box, chunks = second ? p.vc : p.kd, stages = p.stages;
    const int bytes = chunks * kPgKeyChunk;
    const CUtensorMap* map = second ? &values : &keys;
    uint64_t *full = second ? sh.v_full : sh.k_full, *empty = second ? sh.v_empty : sh.k_empty;
    uint8_t* tiles = second ? s_v : s_k;
    int* asked = second ? &sh.v_asked : &sh.k_asked;
    int count = 0, stage = 0;
    uint32_t free_phase = 1;
    for (int turn = 0; turn < turns && ok; ++turn) {
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_full[turn % kPgInfos], (turn / kPgInfos) & 1, p.status, 462)) != 0;
      if (!ok) break;
      const GroupWork& w = sh.info[turn % kPgInfos];
      const int n0 = w.tiles[0], n1 = w.both ? 0 : w.tiles[1], most = max(n0, n1);
      int row0 = w.row[0][lane], row1 = w.row[1][lane];
      const int x0 = second ? p.kv_heads * p.dp + w.unit[0].head * p.vp : w.unit[0].head * p.dp;
      const int x1 = second ? p.kv_heads * p.dp + w.unit[1].head * p.vp : w.unit[1].head * p.dp;
      for (int j = 0; j < most && ok; ++j) {
        const int u = j * boxes;
        if (u > 0 && (u & 31) == 0) {                    // boxes divides 32
          row0 = locate(w.unit[0].slot, w.first[0], w.end[0], u);
          row1 = locate(w.unit[1].slot, w.first[1], w.end[1], u);
        }
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          if (j >= (t ? n1 : n0)) continue;
          const int row = t ? row1 : row0, x = t ? x1 : x0;
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], free_phase, p.status, second ? 461 : 460)) != 0;
          if (!ok) break;
          uint8_t* dst = tiles + stage * bytes;
          if (lane == 0) {
            mbar_expect_tx(&full[stage], bytes);
            *reinterpret_cast<volatile int*>(asked) = count + 1;
          }
#pragma unroll 1
          for (int i = 0; i < boxes; ++i, dst += p.box * 128) {
            const int at = __shfl_sync(0xffffffffu, row, (u + i) & 31);
            if (lane == 0) {
              // a copy costs its thread 50 to 100 cycles: all chunks of a page's rows in one where they lie side by side in whole chunks
              if (p.deep) {
                tma_load_3d(dst, map, &full[stage], 0, at, x >> 6);
              } else {
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) tma_load_3d(dst + c * kPgKeyChunk, map, &full[stage], x + 64 * c, at, 0);
              }
            }
            __syncwarp();
          }
          ++count;
          if (++stage == stages) {
            stage = 0;
            free_phase ^= 1;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.info_empty[turn % kPgInfos]);
    }
    if (!ok && lane == 0)                                // something gave up: let the copies under way land before the memory goes away
      for (int b = max(0, count - stages); b < count; ++b)
        for (int i = 0; i < (1 << 18) && !mbar_test_wait(&full[b % stages], (b / stages) & 1); ++i) {
        }
  } else if (warp == 9 || warp == 14) {
    // one thread: votes and the like between two products cost as much as the products
    if (elect_one()) {
      const int t = warp == 14;
      const uint32_t idesc_s = umma_idesc(kPgTile, kPgKeys, 1u, 1u);
      const uint32_t idesc_pv = umma_idesc_bmn(kPgTile, p.vp, 1u, 1u);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q + t * q_bytes)), k_desc = umma_desc_sw128(smem_u32(s_k));
      const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(s_v), kPgKeyChunk, 1024);
      const int whole = p.dp / 64, rest = p.dp / 16 - 4 * whole, mask = p.stages - 1;
      int begun = 0, tiles = 0, done = 0, k_seen = 0, v_seen = 0;        // units, tiles of S, products so far; copies known to be asked for
      // Copy `at` of a ring has landed.  Its place's barrier alone does not say so: while the copy before it in this place, the other
      // tile's, is under way, the one before that shows the same parity.
      auto landed = [&](const int* asked, int& seen, uint64_t* full, int at, int where) {
        if (seen <= at) {
          const long long start = clock64();
          for (uint32_t spins = 1; (seen = *reinterpret_cast<const volatile int*>(asked)) <= at; ++spins)
            if ((spins & 0x3ff) == 0 && (clock64() - start > DS41_WAIT_LIMIT_CYCLES ||
                                         (p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != kStatusOk))) {
              if (p.status != nullptr && atomicCAS(p.status, kStatusOk, kStatusMbarTimeout) == kStatusOk) {
                p.status[1] = where;
                p.status[2] = static_cast<int>(blockIdx.x);
                p.status[3] = at;
              }
              return false;
            }
        }
        return mbar_wait(&full[at & mask], (at >> p.shift) & 1, p.status, where);
      };
      for (int turn = 0; turn < turns && ok; ++turn) {
        ok = mbar_wait(&sh.info_full[turn % kPgInfos], (turn / kPgInfos) & 1, p.status, 470);
        if (!ok) break;
        const GroupWork& w = sh.info[turn % kPgInfos];
        const int n = w.tiles[t], base = w.base, least = min(w.tiles[0], w.tiles[1]);
        const int first = w.first[t], safe = w.safe[t], safe_end = w.safe_end[t];
        const bool both = w.both != 0;
        mbar_arrive(&sh.info_empty[turn % kPgInfos]);
        if (n == 0) continue;
        auto scores = [&](int j) {
          const int at = copy_index(both, base, least, t, j), stage = at & mask, place = tiles & 1;
          if (!landed(&sh.k_asked, k_seen, sh.k_full, at, 471)) return false;
          tc_fence_after();
          const uint32_t to = tmem + t * 128 + 64 * place;
          uint64_t a = q_desc, b = k_desc + static_cast<uint64_t>(stage * k_bytes / 16);
#pragma unroll 1
          for (int c = 0; c < whole; ++c, a += kPgChunk / 16, b += kPgKeyChunk / 16) umma4_ss<2, 2>(to, a, b, idesc_s, c);
#pragma unroll 1
          for (int k = 0; k < rest; ++k) umma_bf16(to, a + 2 * k, b + 2 * k, idesc_s, whole > 0 || k > 0);
          tc_commit(&sh.s_full[t][place]);
          if (!both) mbar_arrive(&sh.k_empty[stage]);
          tc_commit(&sh.k_empty[stage]);
          ++tiles;
          if (j + 1 == n) tc_commit(&sh.q_empty[t]);
          return true;
        };
        ok = mbar_wait(&sh.q_full[t], begun & 1, p.status, 472) && scores(0);
        ++begun;
        for (int j = 0; j < n && ok; ++j) {
          // they overwrite the P that the values before this tile's read
          if (j + 1 < n) ok = scores(j + 1);
          if (!ok) break;
          const int at = copy_index(both, base, least, t, j), stage = at & mask, place = done & 1;
          ok = landed(&sh.v_asked, v_seen, sh.v_full, at, 473);
          if (!ok) break;
          const int key0 = first + j * kPgKeys;
          if (key0 < safe || key0 > safe_end - kPgKeys) {
            sh.v_place[t] = stage;
            mbar_arrive(&sh.v_here[t]);
          }
          ok = mbar_wait(&sh.p_full[t][place], (done >> 1) & 1, p.status, 474);
          if (!ok) break;
          tc_fence_after();
          umma4_ts<128>(tmem + 256 + t * 128, tmem + t * 128 + 64 * place, v_desc + static_cast<uint64_t>(stage * v_bytes / 16), idesc_pv,
                        j > 0);
          ++done;
          if (!both) mbar_arrive(&sh.v_empty[stage]);
          tc_commit(&sh.v_empty[stage]);
          if (j + 2 == n) tc_commit(&sh.o_next[t]);
          if (j + 1 == n) tc_commit(&sh.o_full[t]);
        }
      }
    }
    __syncwarp();
  } else {
    // the roles that follow one tile: its work at a turn, once it is known; whole warps
    auto work = [&](int turn, int t, PrefixUnit& unit, int& first, int& safe, int& safe_end, bool& gaps) {
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_full[turn % kPgInfos], (turn / kPgInfos) & 1, p.status, 462)) != 0;
      if (!ok) return 0;
      const GroupWork& w = sh.info[turn % kPgInfos];
      unit = w.unit[t];
      first = w.first[t];
      safe = w.safe[t];
      safe_end = w.safe_end[t];
      gaps = w.gaps[t] != 0;
      return w.tiles[t];
    };
    auto work_read = [&](int turn) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.info_empty[turn % kPgInfos]);
    };
    PrefixUnit unit;
    int first, safe, safe_end;
    bool gaps;
    if (warp >= 10) {
      // A row's queries lie side by side: pieces of 16 bytes by neighbouring lanes, or whole rows where they are shorter than a warp.
      const int t = warp - 10, pieces = p.n * p.dp / 8, per = max(1, 32 / pieces), sub = pieces < 32 ? lane / pieces : 0;
      const int piece0 = pieces < 32 ? lane % pieces : lane;
      int filled = 0;
      for (int turn = 0; turn < turns; ++turn) {
        // everything is asked for before it is known whether the unit has keys
        unit = turn == 0 ? (t ? first_b : first_a) : prefix_unit(plan, 2 * (static_cast<int>(blockIdx.x) + turn * static_cast<int>(gridDim.x)) + t);
        int row[4], pos[4], slot[4], cell[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (lane + 32 * k < unit.rows) {
            row[k] = prefix_row(plan, unit, lane + 32 * k);
            pos[k] = p.row_pos[row[k]];
            slot[k] = p.row_slot[row[k]];
            cell[k] = plan.cell[row[k]];
          }
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.q_empty[t], (filled & 1) ^ 1, p.status, 463)) != 0;
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (lane + 32 * k < unit.rows)
            sh.row[t][lane + 32 * k] = make_int4(row[k], slot[k] >= 0 ? chunk_start(pos[k], p.chunk) : 0,
                                                 slot[k] >= 0 ? min(pos[k] + 1, unit.key1) : 0, cell[k] + unit.part);
        __syncwarp();
        for (int piece = piece0; piece < pieces && sub < per; piece += 32) {
          const int head = piece * 8 / p.dp, c = piece - head * (p.dp / 8);
          const __nv_bfloat16* src = p.q + unit.head * p.n * p.dp + 8 * piece;
          uint8_t* dst = s_q + t * q_bytes + (c >> 3) * kPgChunk;
#pragma unroll 4
          for (int i = sub; i < unit.rows; i += per) {
            const int x = i * p.n + head;
            cp_async_16(dst + x * 128 + (((c & 7) ^ (x & 7)) << 4), src + sh.row[t][i].x * p.ld_q);
          }
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_full[turn % kPgInfos], (turn / kPgInfos) & 1, p.status, 464)) != 0;
        cp_async_wait_all();
        if (!ok) break;
        const int n = sh.info[turn % kPgInfos].tiles[t];
        work_read(turn);
        if (n == 0) continue;
        ++filled;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full[t]);
      }
    } else {
      const int t = warp >> 2, quad = warp & 3, mine = quad * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
      const uint32_t o_t = tmem + lanes + 256 + t * 128;
      const int mine_row = mine / p.n, mine_head = mine - mine_row * p.n;
      int tiles = 0, done = 0, pairs = 0, cut = 0;       // tiles of S; units with keys, with two tiles or more; key tiles with unseen places
      for (int turn = 0; turn < turns; ++turn) {
        const int n = work(turn, t, unit, first, safe, safe_end, gaps);
        if (!ok) break;
        work_read(turn);
        if (n == 0) {                                    // nothing for any of its rows
          if (mine_row < unit.rows) {
            const long long cell = (1ll * plan.cell[prefix_row(plan, unit, mine_row)] + unit.part) * p.heads + unit.head * p.n + mine_head;
            *reinterpret_cast<float2*>(plan.part_ml + 2 * cell) = make_float2(-INFINITY, 0.f);
          }
          continue;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.q_full[t], done & 1, p.status, 482 + t)) != 0;
        if (!ok) break;
        const int4 me = mine_row < unit.rows ? sh.row[t][mine_row] : make_int4(-1, 0, 0, 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_empty[t]);
        const int r = me.x, lo = me.y, hi = me.z;
        // limits of the warp's queries: tiles between them need no look at single keys
        int low = hi > lo ? lo : 0, high = hi > lo ? hi : 0x7fffffff;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          low = max(low, __shfl_xor_sync(0xffffffffu, low, o));
          high = min(high, __shfl_xor_sync(0xffffffffu, high, o));
        }
        const bool idle = high == 0x7fffffff;            // no query of this warp sees anything
        float m = -INFINITY, l = 0.f;
        for (int j = 0; j < n; ++j) {
          const int place = tiles & 1;
          const uint32_t s_t = tmem + lanes + t * 128 + 64 * place;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full[t][place], (tiles >> 1) & 1, p.status, 480 + t)) != 0;
          if (!ok) break;
          ++tiles;
          // the last tile: the product before it is complete; for the others the next scores say so
          if (j > 0 && j + 1 == n) {
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_next[t], pairs & 1, p.status, 486 + t)) != 0;
            if (!ok) break;
            ++pairs;
          }
          const int key0 = first + j * kPgKeys;
          if (!idle) {
            tc_fence_after();
            const bool edge = key0 < low || key0 + kPgKeys > high;
            const int shown = hi - key0, hidden = lo - key0;             // columns [hidden, shown) of this tile are visible
            // the code of this loop is short on purpose: instructions that run for the first time are waited for
            float2 v[kPgKeys / 2];
            {
              uint32_t(&raw)[64] = reinterpret_cast<uint32_t(&)[64]>(v);
              tmem_ld_32x32(s_t, reinterpret_cast<uint32_t(&)[32]>(raw[0]));
              tmem_ld_32x32(s_t + 32, reinterpret_cast<uint32_t(&)[32]>(raw[32]));
              tmem_wait_ld();
            }
            if (edge) {
#pragma unroll
              for (int i = 0; i < kPgKeys / 2; ++i) {
                v[i].x = 2 * i < shown && 2 * i >= hidden ? v[i].x : -INFINITY;
                v[i].y = 2 * i + 1 < shown && 2 * i + 1 >= hidden ? v[i].y : -INFINITY;
              }
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < kPgKeys / 2; ++i) tops[i & 3] = fmaxf(tops[i & 3], fmaxf(v[i].x, v[i].y));
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * p.scale_log2;
            const bool grow = hi > lo && (top > m + 8.f || (m == -INFINITY && top > m));
            if (__any_sync(0xffffffffu, grow)) {
              const float m_new = grow ? top : m;
              const float alpha = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
              if (grow) l *= alpha;
              m = m_new;
              if (j > 0) {
                if (j + 1 < n) {                         // the next scores were issued behind the last values
                  ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full[t][place ^ 1], (tiles >> 1) & 1, p.status, 488 + t)) != 0;
                  if (!ok) break;
                  tc_fence_after();
                }
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
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t e2[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float2 e = fma2(v[16 * h + i], by, off);
                e = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                sums[i & 1] = add2(sums[i & 1], e);
                const __nv_bfloat162 b = __floats2bfloat162_rn(e.x, e.y);
                e2[i] = *reinterpret_cast<const uint32_t*>(&b);
              }
              tmem_st_32x16(s_t + 16 * h, e2);           // this thread has read all of its S
            }
            sums[0] = add2(sums[0], sums[1]);
            l += sums[0].x + sums[0].y;
          }
          if (key0 < safe || key0 > safe_end - kPgKeys) {
            // Places that no row sees may hold anything, and a weight of zero does not take a NaN or an infinity away: their values
            // become zeros, two threads to a place.  Where rows stand in different chunks, those of whoever walks these keys are asked.
            uint32_t seen[2];
            if (gaps) {
              const PrefixUnit other = prefix_unit(plan, 2 * (static_cast<int>(blockIdx.x) + turn * static_cast<int>(gridDim.x)) + (t ^ 1));
              unsigned long long mask = prefix_seen(plan, unit, p.row_pos, p.row_slot, p.chunk, key0);
              if (!unit.tail && !other.tail && other.slot == unit.slot && other.key0 == unit.key0 && other.key1 == unit.key1 &&
                  other.head == unit.head)
                mask |= prefix_seen(plan, other, p.row_pos, p.row_slot, p.chunk, key0);
              seen[0] = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(mask));
              seen[1] = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(mask >> 32));
            } else {
              const int from = max(safe - key0, 0), to = min(safe_end - key0, kPgKeys);
              const unsigned long long mask = from < to ? (~0ull >> (64 - (to - from))) << from : 0ull;
              seen[0] = static_cast<uint32_t>(mask);
              seen[1] = static_cast<uint32_t>(mask >> 32);
            }
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.v_here[t], cut & 1, p.status, 484 + t)) != 0;
            if (!ok) break;
            ++cut;
            const int key = mine & (kPgKeys - 1), at = sh.v_place[t];
            if (!((key < 32 ? seen[0] : seen[1]) >> (key & 31) & 1))
              for (int i = 8 * (mine / kPgKeys); i < 8 * p.vc; i += (i & 7) == 7 ? 9 : 1)
                *reinterpret_cast<uint4*>(s_v + at * v_bytes + (i >> 3) * kPgKeyChunk + key * 128 + (i & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
            fence_async_smem();
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[t][place]);
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_full[t], done & 1, p.status, 490 + t)) != 0;
        if (!ok) break;
        ++done;
        tc_fence_after();
        if (hi <= lo) {                                  // a query that sees nothing here: tiles without an edge did not look
          m = -INFINITY;
          l = 0.f;
        }
        const bool write = r >= 0;
        const long long cell = write ? 1ll * me.w * p.heads + unit.head * p.n + mine_head : 0;
        if (write) *reinterpret_cast<float2*>(plan.part_ml + 2 * cell) = make_float2(m, l);
        if (!idle) {                                     // whole warps: tensor memory is read by all lanes
          float* dst = plan.part_o + cell * p.vp;
#pragma unroll 1
          for (int c = 0; c < p.vp; c += 32) {             // a last half piece reads columns that nobody stores
            uint32_t a[32];
            tmem_ld_32x32(o_t + c, a);
            tmem_wait_ld();
            if (write) {
#pragma unroll
              for (int i = 0; i < 32; i += 8)
                if (c + i < p.vp) store8(dst + c + i, reinterpret_cast<const float(&)[8]>(a[i]));
            }
            __syncwarp();
          }
        }
        tc_fence_before();
      }
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
  if (a.f32 || a.n_pages <= 0 || a.vdim_pad > 128 || (a.ld_q & 7) || plan.rows_per_unit * p.n > kPgTile ||
      ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.pool)) & 15) ||
      1ll * a.n_pages * a.page_tokens >= (1ll << 31) - 1)
    return false;
  if (a.page_tokens % kPgKeys == 0) p.box = kPgKeys;
  else if (kPgKeys % a.page_tokens == 0 && a.page_tokens >= 8) p.box = a.page_tokens;
  else return false;
  p.kd = (a.dim_pad + 63) / 64;
  p.vc = (a.vdim_pad + 63) / 64;
  p.deep = p.box == kPgKeys && a.dim_pad % 64 == 0 && a.vdim_pad % 64 == 0;
  const int q = p.kd * kPgChunk, k = p.kd * kPgKeyChunk, v = p.vc * kPgKeyChunk;
  constexpr int kExtra = 1024 + static_cast<int>(sizeof(GroupShared)), kLimit = 227 * 1024 - kExtra;
  const int fit = (kLimit - 2 * q) / (k + v);
  if (fit < 1) return false;
  while (p.shift < 3 && 2 << p.shift <= fit) ++p.shift;  // kPgStages at most
  p.stages = 1 << p.shift;
  smem = 2 * q + p.stages * (k + v) + kExtra;
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
  p.chunk = a.chunk; p.max_pages = a.max_pages; p.page_tokens = a.page_tokens; p.n_pages = a.n_pages;
  p.hidden_row = a.n_pages * a.page_tokens;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = a.status;
  const int row_len = a.kv_heads * (a.dim_pad + a.vdim_pad);
  // keys and values are columns of the same rows; deep: as chunks of 64 columns, all of a head's in one box
  CUtensorMap keys, values;
  for (int i = 0; i < 2; ++i) {
    const cudaError_t e =
        p.deep ? make_tensor_map_3d(i ? &values : &keys, a.pool, TmaDtype::kBF16, 64, p.hidden_row, row_len / 64, 2ull * row_len, 128, 64, p.box,
                                    true, i ? p.vc : p.kd)
               : make_tensor_map_3d(i ? &values : &keys, a.pool, TmaDtype::kBF16, row_len, p.hidden_row, 1, 2ull * row_len, 0, 64, p.box, true);
    if (e != cudaSuccess) return e;
  }
  const cudaError_t e = cudaFuncSetAttribute(prefix_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(prefix_group_kernel, dim3(plan.grid), dim3(kPgThreads), smem, st, keys, values, p, plan);
}

}  // namespace ds41
