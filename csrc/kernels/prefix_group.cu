// Parts of grouped-query attention for rows that share prefixes, on tcgen05.
//
// The queries of one key/value head are packed: (row, head) pairs of a unit's rows are the 128 rows of a tensor-core tile, so that a
// tile of keys and values is read once for all of them and the products have the shape of a prompt's.  A CTA has two tiles: units
// come in twos, and where both of them walk the same keys each copy serves two tiles.  One tile's softmax runs while the tensor core
// works on the other's products, and nothing but the order of the copies ties the two together.
//   warps 0-3, 4-7 : softmax of tile 0 / 1 (one thread per query), partial results
//   warps 8, 12    : TMA producers: key / value tiles of 128 positions, page by page
//   warp 9         : tcgen05.mma issue, in whichever order their inputs come: S = Q K^T, O += P V with P in TMEM where it replaces its S
//   warps 10, 11   : queries of tile 0 / 1, and what each of them sees
//   warp 13        : what the next units are and where their keys lie, for everybody (a ring of four)
// A CTA walks its units, and every role but the softmax runs ahead into the next ones: a request's own keys are a few tiles, which the
// chain of loads that a unit begins with (its description, its rows' positions, their pages, their queries) would take as long as.
// The running maximum is raised when it grew by more than 2^8 only; what leaves is (m, l, unnormalised O) in 32 bits.  P is rounded
// to bf16 as the operand of the second product; l sums the unrounded weights.
#include <cuda.h>

#include "ds41_group.cuh"
#include "ds41_mma.cuh"
#include "ds41_prefix.cuh"
#include "ds41_tma.h"

namespace ds41 {

constexpr int kPgThreads = 448;
constexpr int kPgTile = 128;                   // queries per tile, keys per tile
constexpr int kPgChunk = kPgTile * 128;        // bytes of 128 rows x 64 bf16 columns
constexpr int kPgInfos = 4;

struct PrefixGroupParams {
  const __nv_bfloat16* q;
  const int *page_table, *row_pos, *row_slot;
  long long ld_q;
  int heads, kv_heads, n, dp, vp, kd, vc, k_stages, v_stages;
  int chunk, max_pages, page_tokens, box, hidden_row;      // a row beyond the pool: reads as zeros
  float scale_log2;
  int* status;
};

// What a CTA's two tiles do next, as the producer found it: unit t walks `tiles[t]` key tiles from `first[t]` on, and nobody sees
// `end[t]` or what follows.  both: they walk the same ones.
struct __align__(16) GroupWork {
  PrefixUnit unit[2];
  int first[2], end[2], tiles[2], base, both;              // base: number of the first key tile in the order of the copies
  int row[2][32];                                          // pool rows of the first 32 boxes of their keys
};

// Number of key tile j of tile t in the order of the copies: one after the other, or in turn as long as both have some.
__device__ __forceinline__ int copy_index(const GroupWork& w, int t, int j) {
  if (w.both) return w.base + j;
  const int least = min(w.tiles[0], w.tiles[1]);
  return w.base + (j < least ? 2 * j + t : least + j);
}

struct GroupShared {                           // behind the tiles
  uint64_t info_full[kPgInfos], info_empty[kPgInfos];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  // per tile:
  uint64_t q_full[2], q_empty[2];
  uint64_t s_full[2];                          // S complete (and every earlier MMA of the issuing thread)
  uint64_t p_full[2];                          // P written, O rescaled
  uint64_t o_full[2];                          // the unit's last product
  uint64_t v_here[2];                          // the values of a tail's last tile, for the softmax
  uint32_t tmem, pad[3];
  GroupWork info[kPgInfos];
  int4 row[2][kPgTile];                        // of a unit's row: pass row, visible keys [y, z), cell
};

__global__ void __launch_bounds__(kPgThreads, 1)
prefix_group_kernel(const __grid_constant__ CUtensorMap pool, const PrefixGroupParams p, const ds41_prefix_plan plan) {
  extern __shared__ uint8_t pg_raw[];
  uint8_t* smem = pg_raw + ((1024u - (smem_u32(pg_raw) & 1023u)) & 1023u);
  const int q_bytes = p.kd * kPgChunk, k_bytes = q_bytes, v_bytes = p.vc * kPgChunk;
  uint8_t* s_q = smem;                                   // two tiles
  uint8_t* s_k = s_q + 2 * q_bytes;
  uint8_t* s_v = s_k + p.k_stages * k_bytes;
  GroupShared& sh = *reinterpret_cast<GroupShared*>(s_v + p.v_stages * v_bytes);
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
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.v_here[i], 1);
    }
    mbar_init_fence();
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
    return id >= 0 ? id * p.page_tokens + (key - pg * p.page_tokens) : p.hidden_row;
  };

  if (warp == 13) {
    int base = 0;
    for (int turn = 0; turn < turns; ++turn) {
      const int at = 2 * (static_cast<int>(blockIdx.x) + turn * static_cast<int>(gridDim.x));
      const PrefixUnit a = turn == 0 ? first_a : prefix_unit(plan, at), b = turn == 0 ? first_b : prefix_unit(plan, at + 1);
      // without chunks a walk begins at its first key: its pages are looked up together with its rows' positions
      int row_a = locate(a.slot, a.key0, a.key1, 0), row_b = locate(b.slot, b.key0, b.key1, 0);
      const PrefixRows rows_a = prefix_rows(plan, a, p.row_pos, p.row_slot, p.chunk), rows_b = prefix_rows(plan, b, p.row_pos, p.row_slot, p.chunk);
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
      if (first[0] != a.key0) row_a = locate(a.slot, first[0], end[0], 0);
      if (first[1] != b.key0) row_b = locate(b.slot, first[1], end[1], 0);
      if (first[0] + lane * p.box >= end[0]) row_a = p.hidden_row;
      if (first[1] + lane * p.box >= end[1]) row_b = p.hidden_row;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_empty[turn % kPgInfos], ((turn / kPgInfos) & 1) ^ 1, p.status, 459)) != 0;
      if (!ok) break;
      GroupWork& w = sh.info[turn % kPgInfos];
      const int tiles[2] = {(end[0] - first[0] + kPgTile - 1) / kPgTile, (end[1] - first[1] + kPgTile - 1) / kPgTile};
      w.row[0][lane] = row_a;
      w.row[1][lane] = row_b;
      if (lane < 2) {
        w.unit[lane] = lane ? b : a;
        w.first[lane] = lane ? first[1] : first[0];
        w.end[lane] = lane ? end[1] : end[0];
        w.tiles[lane] = lane ? tiles[1] : tiles[0];
        w.base = base;
        w.both = both;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.info_full[turn % kPgInfos]);
      base += both ? tiles[0] : tiles[0] + tiles[1];
    }
  } else if (warp == 8 || warp == 12) {
    const bool values = warp == 12;
    const int boxes = kPgTile / p.box, chunks = values ? p.vc : p.kd, stages = values ? p.v_stages : p.k_stages;
    const int bytes = chunks * kPgChunk;
    uint64_t *full = values ? sh.v_full : sh.k_full, *empty = values ? sh.v_empty : sh.k_empty;
    uint8_t* tiles = values ? s_v : s_k;
    int count = 0, stage = 0;
    uint32_t free_phase = 1;
    for (int turn = 0; turn < turns && ok; ++turn) {
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_full[turn % kPgInfos], (turn / kPgInfos) & 1, p.status, 462)) != 0;
      if (!ok) break;
      const GroupWork& w = sh.info[turn % kPgInfos];
      const int n0 = w.tiles[0], n1 = w.both ? 0 : w.tiles[1], most = max(n0, n1);
      int row0 = w.row[0][lane], row1 = w.row[1][lane];
      const int x0 = values ? p.kv_heads * p.dp + w.unit[0].head * p.vp : w.unit[0].head * p.dp;
      const int x1 = values ? p.kv_heads * p.dp + w.unit[1].head * p.vp : w.unit[1].head * p.dp;
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
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], free_phase, p.status, values ? 461 : 460)) != 0;
          if (!ok) break;
          uint8_t* dst = tiles + stage * bytes;
          if (lane == 0) mbar_expect_tx(&full[stage], bytes);
#pragma unroll 1
          for (int i = 0; i < boxes; ++i, dst += p.box * 128) {
            const int at = __shfl_sync(0xffffffffu, row, (u + i) & 31);
            if (lane == 0)
#pragma unroll 1
              for (int c = 0; c < chunks; ++c) tma_load_3d(dst + c * kPgChunk, &pool, &full[stage], x + 64 * c, at, 0);
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
  } else if (warp == 9) {
    // one thread: votes and the like between two products cost as much as the products
    if (elect_one()) {
      const uint32_t idesc_s = umma_idesc(kPgTile, kPgTile, 1u, 1u);
      const uint32_t idesc_pv = umma_idesc_bmn(kPgTile, p.vp, 1u, 1u);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q)), k_desc = umma_desc_sw128(smem_u32(s_k));
      const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(s_v), kPgChunk, 1024);
      const int whole = p.dp / 64, rest = p.dp / 16 - 4 * whole;
      // per tile: the turn it is at, its key tiles (0: not begun), the next scores and values of that turn, and counts of units and
      // products for the barriers' phases.  Scores overwrite the P that the values before them read.
      int turn[2] = {0, 0}, n[2] = {0, 0}, sj[2] = {0, 0}, pj[2] = {0, 0}, begun[2] = {0, 0}, done[2] = {0, 0};
      bool told[2] = {false, false};
      // A tile's place in its ring has been filled at most as often as its last tenants were used: one tile may ask for copies far ahead
      // of the other's, whose barrier would still show a phase of the same parity.
      int k_used[2] = {-p.k_stages, 1 - p.k_stages}, v_used[2] = {-p.v_stages, 1 - p.v_stages};
      auto key_here = [&](int at) {
        const int stage = p.k_stages == 2 ? at & 1 : 0;
        return (stage ? k_used[1] : k_used[0]) == at - p.k_stages &&
               mbar_test_wait(&sh.k_full[stage], p.k_stages == 2 ? (at >> 1) & 1 : at & 1);
      };
      auto value_here = [&](int at) {
        const int stage = p.v_stages == 2 ? at & 1 : 0;
        return (stage ? v_used[1] : v_used[0]) == at - p.v_stages &&
               mbar_test_wait(&sh.v_full[stage], p.v_stages == 2 ? (at >> 1) & 1 : at & 1);
      };
      uint32_t idle = 0;
      long long since = 0;
      while (ok && (turn[0] < turns || turn[1] < turns)) {
        bool moved = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (turn[t] >= turns) continue;
          const GroupWork& w = sh.info[turn[t] % kPgInfos];
          uint64_t* read = &sh.info_empty[turn[t] % kPgInfos];
          if (n[t] == 0) {
            if (!mbar_test_wait(&sh.info_full[turn[t] % kPgInfos], (turn[t] / kPgInfos) & 1)) continue;
            moved = true;
            n[t] = w.tiles[t];
            if (n[t] == 0) {
              mbar_arrive(read);
              ++turn[t];
              continue;
            }
          }
          const bool both = w.both != 0;
          const int o = t ^ 1;
          if (pj[t] < sj[t]) {
            const int at = copy_index(w, t, pj[t]), stage = p.v_stages == 2 ? at & 1 : 0;
            if (!told[t] && pj[t] + 1 == n[t] && w.unit[t].tail && value_here(at)) {
              mbar_arrive(&sh.v_here[t]);
              told[t] = moved = true;
            }
            if (mbar_test_wait(&sh.p_full[t], done[t] & 1) && value_here(at)) {
              tc_fence_after();
              const uint64_t vd = v_desc + static_cast<uint64_t>(stage * v_bytes / 16);
              const uint32_t to = tmem + 256 + t * 128, a = tmem + t * 128;
              umma4_ts<128>(to, a, vd, idesc_pv, pj[t] > 0);
              umma4_ts<128>(to, a + 32, vd + 512, idesc_pv, 1u);
              ++done[t];
              if (!both || turn[o] > turn[t] || (turn[o] == turn[t] && pj[o] > pj[t])) {      // its last reader
                tc_commit_if(true, &sh.v_empty[stage]);
                if (stage) v_used[1] = at;
                else v_used[0] = at;
              }
              ++pj[t];
              moved = true;
              if (pj[t] == n[t]) {
                tc_commit_if(true, &sh.o_full[t]);
                mbar_arrive(read);
                ++turn[t];
                n[t] = sj[t] = pj[t] = 0;                // the other tile compares itself with these
                told[t] = false;
                continue;
              }
            }
          }
          if (sj[t] < n[t] && sj[t] == pj[t]) {
            const int at = copy_index(w, t, sj[t]), stage = p.k_stages == 2 ? at & 1 : 0;
            if (key_here(at) && (sj[t] > 0 || mbar_test_wait(&sh.q_full[t], begun[t] & 1))) {
              tc_fence_after();
              uint64_t a = q_desc + static_cast<uint64_t>(t * q_bytes / 16), b = k_desc + static_cast<uint64_t>(stage * k_bytes / 16);
#pragma unroll 1
              for (int c = 0; c < whole; ++c, a += kPgChunk / 16, b += kPgChunk / 16) umma4_ss<2, 2>(tmem + t * 128, a, b, idesc_s, c);
#pragma unroll 1
              for (int k = 0; k < rest; ++k) umma_bf16(tmem + t * 128, a + 2 * k, b + 2 * k, idesc_s, whole > 0 || k > 0);
              tc_commit_if(true, &sh.s_full[t]);
              if (!both || turn[o] > turn[t] || (turn[o] == turn[t] && sj[o] > sj[t])) {
                tc_commit_if(true, &sh.k_empty[stage]);
                if (stage) k_used[1] = at;
                else k_used[0] = at;
              }
              if (sj[t] == 0) ++begun[t];
              ++sj[t];
              if (sj[t] == n[t]) tc_commit_if(true, &sh.q_empty[t]);
              moved = true;
            }
          }
        }
        if (moved) {
          idle = 0;
          since = 0;
        } else if ((++idle & 0x3ff) == 0) {              // as long as any other wait: see mbar_wait
          if (since == 0) since = clock64();
          if (clock64() - since > DS41_WAIT_LIMIT_CYCLES ||
              (p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != kStatusOk)) {
            if (p.status != nullptr && atomicCAS(p.status, kStatusOk, kStatusMbarTimeout) == kStatusOk) {
              p.status[1] = 471;
              p.status[2] = static_cast<int>(blockIdx.x);
              p.status[3] = turn[0];
            }
            ok = false;
          }
        }
      }
    }
    __syncwarp();
  } else {
    // the roles that follow one tile: its work at a turn, once it is known; whole warps
    auto work = [&](int turn, int t, PrefixUnit& unit, int& first, int& end, int& last) {
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_full[turn % kPgInfos], (turn / kPgInfos) & 1, p.status, 462)) != 0;
      if (!ok) return 0;
      const GroupWork& w = sh.info[turn % kPgInfos];
      unit = w.unit[t];
      first = w.first[t];
      end = w.end[t];
      last = copy_index(w, t, w.tiles[t] > 0 ? w.tiles[t] - 1 : 0);
      return w.tiles[t];
    };
    auto work_read = [&](int turn) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.info_empty[turn % kPgInfos]);
    };
    PrefixUnit unit;
    int first, end, last;                                // last: the last tile's number
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
      const uint32_t s_t = tmem + lanes + t * 128, o_t = tmem + lanes + 256 + t * 128;
      const int mine_row = mine / p.n, mine_head = mine - mine_row * p.n;
      int tiles = 0, done = 0, tails = 0;                // tiles of S, units with keys, tails among them so far
      for (int turn = 0; turn < turns; ++turn) {
        const int n = work(turn, t, unit, first, end, last);
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
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full[t], tiles & 1, p.status, 480 + t)) != 0;
          if (!ok) break;
          ++tiles;
          const int key0 = first + j * kPgTile;
          if (!idle) {
            tc_fence_after();
            const bool edge = key0 < low || key0 + kPgTile > high;
            const int shown = hi - key0, hidden = lo - key0;             // columns [hidden, shown) of this tile are visible
            // Two pieces of 64 columns, read twice.  The bodies of these loops are short on purpose: with the tile unrolled, 42 % of all cycles
            // were waits for instructions, and a small call, which runs all code for the first time, took 6400 cycles for its one tile.
            if (edge) {
#pragma unroll 1
              for (int c = 0; c < kPgTile; c += 32) {
                uint32_t v[32];
                tmem_ld_32x32(s_t + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = i < shown - c && i >= hidden - c ? v[i] : 0xff800000u;
                tmem_st_32x32(s_t + c, v);
              }
              tmem_wait_st();
            }
            float top = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < kPgTile; c += 64) {
              uint32_t v[64];
              tmem_ld_32x32(s_t + c, reinterpret_cast<uint32_t(&)[32]>(v[0]));
              tmem_ld_32x32(s_t + c + 32, reinterpret_cast<uint32_t(&)[32]>(v[32]));
              tmem_wait_ld();
              float tops[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int i = 0; i < 64; i += 2)
                tops[(i >> 1) & 3] = fmaxf(tops[(i >> 1) & 3], fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
              top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            }
            top *= p.scale_log2;
            const bool grow = hi > lo && (top > m + 8.f || (m == -INFINITY && top > m));
            if (__any_sync(0xffffffffu, grow)) {
              const float m_new = grow ? top : m;
              const float alpha = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
              if (grow) l *= alpha;
              m = m_new;
              if (j > 0) {
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
              uint32_t v[64];
              tmem_ld_32x32(s_t + c, reinterpret_cast<uint32_t(&)[32]>(v[0]));
              tmem_ld_32x32(s_t + c + 32, reinterpret_cast<uint32_t(&)[32]>(v[32]));
              tmem_wait_ld();
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t e2[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  float2 e = fma2(make_float2(__uint_as_float(v[32 * h + 2 * i]), __uint_as_float(v[32 * h + 2 * i + 1])), by, off);
                  e = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                  sums[i & 1] = add2(sums[i & 1], e);
                  const __nv_bfloat162 b = __floats2bfloat162_rn(e.x, e.y);
                  e2[i] = *reinterpret_cast<const uint32_t*>(&b);
                }
                tmem_st_32x16(s_t + c / 2 + 16 * h, e2);       // columns whose S this thread has read
              }
            }
            sums[0] = add2(sums[0], sums[1]);
            l += sums[0].x + sums[0].y;
          }
          if (unit.tail && j + 1 == n) {
            // Places behind the last position belong to nobody, and a weight of zero does not take a NaN or an infinity away: their
            // values become zeros, a thread to a place.
            const int stage = p.v_stages == 2 ? last & 1 : 0;
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.v_here[t], tails & 1, p.status, 484 + t)) != 0;
            if (!ok) break;
            ++tails;
            if (key0 + mine >= end)
              for (int i = 0; i < 8 * p.vc; ++i)
                *reinterpret_cast<uint4*>(s_v + stage * v_bytes + (i >> 3) * kPgChunk + mine * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
            fence_async_smem();
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[t]);
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
  if (a.page_tokens % kPgTile == 0) p.box = kPgTile;
  else if (kPgTile % a.page_tokens == 0 && a.page_tokens >= 8) p.box = a.page_tokens;
  else return false;
  p.kd = (a.dim_pad + 63) / 64;
  p.vc = (a.vdim_pad + 63) / 64;
  const int qk = p.kd * kPgChunk, v = p.vc * kPgChunk;
  constexpr int kExtra = 1024 + static_cast<int>(sizeof(GroupShared)), kLimit = 227 * 1024 - kExtra;
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
