// Parts of latent attention for rows that share prefixes, on tcgen05.
//
// Every head reads the same key rows, so the (row, head) pairs of a unit's rows are packed into the 128 rows of a tensor-core tile.
// A key row is [latent | rotated part], the latent being the value as well: with 512 latent values the result of 128 queries alone
// would fill the 512 columns of a CTA's tensor memory.  So two CTAs of a cluster divide the columns of queries, keys and values between
// them: each multiplies its half of the columns, S = S_0 + S_1, they exchange these partial scores through distributed shared memory,
// both compute the whole softmax (the sum of two numbers is the same in either order, so they agree bit for bit), and each
// accumulates its half of the values from the key tile that it has loaded.  No product and no load is made twice.  Up to 256 latent
// values fit one CTA.
//   tensor memory : O 256 columns, Q 160 (the first product's A operand: it never touches shared memory again), S 64, P 32
//   shared memory : a ring of tiles of 64 keys (up to five chunks of 64 columns), two buffers for the other CTA's scores
//   warps 0-7     : two sets of four take the tiles in turn, one thread per query: exchange, softmax, partial results.  A tile's way
//                   from S to P is a chain of latencies; two are under way, and hand the running maximum on as soon as a tile's
//                   own is known
//   warp 8        : TMA producer, page by page
//   warp 9        : tcgen05.mma issue, in whichever order their inputs come: S = Q K^T as soon as the last S is in registers, O += P V
//   warp 10       : tells the other CTA which of its scores have been read.  That takes a release that the whole cluster sees, which
//                   also waits for the scores that a softmax warp has just sent: calls of 128 rows of 32 heads over 16000 keys take
//                   236 us where those warps make it, 212 so
// The running maximum is raised when it grew by more than 2^8 only.  P is rounded to bf16 as the operand of the second product; sums
// stay in 32 bits.
//
// What bounds it: 64 keys take a pair 2600 cycles (128 rows of 32 heads over 16000 shared keys and up to 700 own ones: 207 us with the
// join), of which the tensor core works 1150.  Sending a tile's scores takes 1200 and they share the way into an SM with the next tiles,
// which need a deep ring: with three sets and a third exchange buffer in a place of the ring the call took 238 us, with three sets and
// two buffers 212, when with two sets it took 203.  In one CTA (256 latent values: 73 us) 64 keys take 1425: a tile's P waits for the
// values before it to let go of it.
#include <cuda.h>

#include "ds41_prefix.cuh"
#include "ds41_tma.h"

namespace ds41 {

constexpr int kPlSets = 2, kPlThreads = 128 * kPlSets + 96, kPlTma = 4 * kPlSets, kPlMma = kPlTma + 1, kPlRelay = kPlTma + 2;
constexpr int kPlQueries = 128, kPlKeys = 64;
constexpr int kPlChunk = kPlKeys * 128;        // bytes of a tile's keys x 64 bf16 columns
constexpr int kPlMost = 5;                     // chunks of columns of a CTA
constexpr int kPlStages = 8;
constexpr uint32_t kPlQ = 256, kPlS = 416, kPlP = 480;      // columns of tensor memory behind O

struct PrefixLatentParams {
  const __nv_bfloat16 *q_abs, *q_rot;
  const int *page_table, *row_pos, *row_slot;
  long long ld_q_abs, ld_q_rot;
  int q_rot_stride, heads, kvp, rp;
  int chunks, stages;                                       // of a stage, of the ring
  int v_col[3], rot_step[3];                                // CTA c: latent columns [v_col[c], v_col[c + 1]), rotated steps of 16 likewise
  int max_pages, page_tokens, n_pages, box, hidden_row;
  int deep;                                                 // a CTA's latent chunks of a box in one copy
  int wide;                                                 // queries may be read 32 bytes at a time
  float scale_log2;
  int* status;
};

// ------------------------------------------------------------------ cluster helpers
// Sixteen bytes into the other CTA's shared memory, counted by its barrier.
__device__ __forceinline__ void remote_store(uint32_t addr, uint32_t bar, float a, float b, float c, float d) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%2, %3, %4, %5}, [%1];" ::"r"(addr), "r"(bar),
               "f"(a), "f"(b), "f"(c), "f"(d)
               : "memory");
}
// The other CTA's barrier: what this thread knows to have been read may be overwritten from there.
__device__ __forceinline__ void remote_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// mbar_wait for what the other CTA arrives with: its release is met by an acquire of the same scope.
__device__ __forceinline__ bool cluster_wait(uint64_t* bar, uint32_t parity, int* status, int where) {
  if (!mbar_wait(bar, parity, status, where)) return false;
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool PAIR>
__global__ void __launch_bounds__(kPlThreads, 1)
prefix_latent_kernel(const __grid_constant__ CUtensorMap pool, const __grid_constant__ CUtensorMap chunks, const PrefixLatentParams p,
                     const ds41_prefix_plan plan) {
  extern __shared__ __align__(1024) uint8_t pl_smem[];       // no room to align it here: it is a multiple of 1024 as it is
  uint8_t* smem = pl_smem;
  const int stage_bytes = p.chunks * kPlChunk;
  uint8_t* s_kv = smem;
  float* s_x = reinterpret_cast<float*>(s_kv + p.stages * stage_bytes);      // [2][columns of four][128 queries][4]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_x + (PAIR ? 2 * kPlKeys * kPlQueries : 0));
  uint64_t* kv_full = bars;                                  // [stages]
  uint64_t* kv_empty = kv_full + kPlStages;
  uint64_t* q_full = kv_empty + kPlStages;
  uint64_t* s_free = q_full + 1;                             // S in registers
  // by tile % 2, so that each is waited for by one set (which sees every phase of it):
  uint64_t* p_full = s_free + 1;                             // [2] P written, O rescaled
  uint64_t* s_full = p_full + kPlSets;                       // [2] S complete
  uint64_t* pv_done = s_full + kPlSets;                      // [2] O += P V complete
  uint64_t* x_full = pv_done + kPlSets;                      // [2] the other CTA's scores are here
  uint64_t* x_free = x_full + kPlSets;                       // [2] this CTA's have been read there
  uint64_t* x_read = x_free + kPlSets;                       // [2] the other CTA's have been read here
  uint64_t* known = x_read + kPlSets;                        // [2][4] the maximum after a tile, by quadrant
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(known + 4 * kPlSets);
  float* s_top = reinterpret_cast<float*>(tmem_slot + 2);    // [128] the running maximum
  float* s_sum = s_top + kPlQueries;                         // [2][128] the sets' sums
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? static_cast<int>(blockIdx.x & 1) : 0;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPlStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(q_full, 4 * kPlSets);
    mbar_init(s_free, 4);
    for (int i = 0; i < kPlSets; ++i) {
      mbar_init(&p_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&pv_done[i], 1);
      mbar_init(&x_full[i], 1);
      mbar_init(&x_free[i], 1);
      mbar_init(&x_read[i], 4);
      for (int q = 0; q < 4; ++q) mbar_init(&known[4 * i + q], 1);
    }
    mbar_init_fence();
    tma_prefetch_desc(&pool);
    if (p.deep) tma_prefetch_desc(&chunks);
  }
  if (warp == kPlMma) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_meet();                                  // the other CTA's barriers are ready, too
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The plan was copied to the device, not computed there by a kernel: it may be read before the wait.
  const int first_unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, unit_step = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int units = first_unit + plan.turns[first_unit] * unit_step;      // one past the last one's place
  const PrefixUnit begin = prefix_unit(plan, first_unit);
  pdl_wait();

  const int v0 = p.v_col[rank], v1 = p.v_col[rank + 1], r0 = p.rot_step[rank], r1 = p.rot_step[rank + 1];
  const int v_chunks = (v1 - v0 + 63) / 64, r_chunk0 = r0 >> 2, r_chunks = r1 > r0 ? (r1 + 3) / 4 - r_chunk0 : 0;

  auto span = [&](const PrefixUnit& it, int& end) {            // the key tiles of a unit (whole warps)
    int first;
    PrefixRows rows = prefix_rows(plan, it, p.row_pos, p.row_slot, 0);
    prefix_span(it, rows, 0, p.page_tokens, first, end);
    return (end - first + kPlKeys - 1) / kPlKeys;
  };

  if (warp == kPlTma) {
    // A copy costs the issuing thread 50 to 100 cycles: where a tile lies in one page and the chunks in one row of them, all of a CTA's
    // latent chunks come in one (a box of 64 columns x 64 rows x chunks).
    const int boxes = kPlKeys / p.box, singles = p.deep ? r_chunks : v_chunks + r_chunks, first_single = p.deep ? v_chunks : 0;
    int stage = 0, kt = 0;
    uint32_t free_phase = 1;
    bool ok = true;
    for (int unit = first_unit; unit < units && ok; unit += unit_step) {
      const PrefixUnit it = unit == first_unit ? begin : prefix_unit(plan, unit);
      if (it.rows == 0) continue;
      int end;
      const int n = span(it, end);
      const int* table = p.page_table + 1ll * it.slot * p.max_pages;
      int row = 0, u = 0;                                    // lane i: pool row of box i of the walk, 32 boxes at a time
      for (int j = 0; j < n; ++j, ++kt) {
        ok = __all_sync(0xffffffffu, mbar_wait(&kv_empty[stage], free_phase, p.status, 500)) != 0;
        if (!ok) break;
        uint8_t* dst = s_kv + stage * stage_bytes;
        if (lane == 0) mbar_expect_tx(&kv_full[stage], (v_chunks + r_chunks) * kPlChunk);
#pragma unroll 1
        for (int i = 0; i < boxes; ++i, ++u, dst += p.box * 128) {
          if ((u & 31) == 0) {
            const int key = it.key0 + (u + lane) * p.box, pg = key / p.page_tokens;
            const int id = key < end && pg < p.max_pages ? table[pg] : -1;
            row = static_cast<unsigned>(id) < static_cast<unsigned>(p.n_pages) ? id * p.page_tokens + (key - pg * p.page_tokens) : p.hidden_row;
          }
          const int at = __shfl_sync(0xffffffffu, row, u & 31);
          if (lane == 0) {
            if (p.deep) tma_load_3d(dst, &chunks, &kv_full[stage], 0, at, v0 >> 6);
#pragma unroll 1
            for (int c = first_single; c < first_single + singles; ++c)
              tma_load_3d(dst + c * kPlChunk, &pool, &kv_full[stage],
                          c < v_chunks ? v0 + 64 * c : p.kvp + 64 * (r_chunk0 + c - v_chunks), at, 0);
          }
          __syncwarp();
        }
        if (++stage == p.stages) {
          stage = 0;
          free_phase ^= 1;
        }
      }
    }
    if (!ok && lane == 0)                                    // let the copies under way land before the shared memory goes away
      for (int b = max(0, kt - p.stages); b < kt; ++b)
        for (int i = 0; i < (1 << 18) && !mbar_test_wait(&kv_full[b % p.stages], (b / p.stages) & 1); ++i) {
        }
  } else if (warp == kPlMma) {
    const bool leader = elect_one();
    const uint32_t idesc_s = umma_idesc(kPlQueries, kPlKeys, 1u, 1u);
    const uint32_t idesc_pv = umma_idesc_bmn(kPlQueries, v1 - v0, 1u, 1u);
    const uint64_t k_desc = umma_desc_sw128(smem_u32(s_kv)), v_desc = umma_desc_sw128_mn(smem_u32(s_kv), kPlChunk, 1024);
    bool ok = true;
    int kt = 0, live = 0, s_stage = 0, p_stage = 0;            // tiles so far; the ring's places of the next scores and values
    uint32_t s_phase = 0;
    for (int unit = first_unit; unit < units && ok; unit += unit_step) {
      const PrefixUnit it = unit == first_unit ? begin : prefix_unit(plan, unit);
      if (it.rows == 0) continue;
      int end;
      const int n = span(it, end);
      if (n == 0) continue;
      if (leader) {                                            // one thread: votes and the like between two products cost as much as the products
        ok = mbar_wait(q_full, live & 1, p.status, 510);
        ++live;
        tc_fence_after();
        int sj = 0, pj = 0;                                    // next scores, next values
        uint32_t idle = 0;
        long long since = 0;
        while (ok && pj < n) {
          const int st = kt + sj, pt = kt + pj;
          if (pj < sj && mbar_test_wait(&p_full[pt % kPlSets], (pt / kPlSets) & 1)) {
            tc_fence_after();
            umma4_ts<128>(tmem, tmem + kPlP, v_desc + static_cast<uint64_t>(p_stage * stage_bytes / 16), idesc_pv, pj > 0);
            tc_commit_if(true, &kv_empty[p_stage]);
            tc_commit_if(true, &pv_done[pt % kPlSets]);
            ++pj;
            if (++p_stage == p.stages) p_stage = 0;
          } else if (sj < n && mbar_test_wait(&kv_full[s_stage], s_phase) && (st == 0 || mbar_test_wait(s_free, (st - 1) & 1))) {
            tc_fence_after();
            // steps of 16 columns, four to a chunk of 128 bytes; queries are zero behind the last latent column
            uint64_t b = k_desc + static_cast<uint64_t>(s_stage * stage_bytes / 16);
            uint32_t a = tmem + kPlQ;
#pragma unroll 1
            for (int c = 0; c < v_chunks; ++c, a += 32, b += kPlChunk / 16) umma4_ts<2>(tmem + kPlS, a, b, idesc_s, c);
#pragma unroll 1
            for (int k = r0 - 4 * r_chunk0; k < r1 - 4 * r_chunk0; ++k)
              umma_bf16_ts_if(true, tmem + kPlS, a + 8 * k, b + (k >> 2) * (kPlChunk / 16) + 2 * (k & 3), idesc_s, 1u);
            tc_commit_if(true, &s_full[st % kPlSets]);
            ++sj;
            if (++s_stage == p.stages) {
              s_stage = 0;
              s_phase ^= 1;
            }
          } else if ((++idle & 0x3ff) == 0) {                  // as long as any other wait: see mbar_wait
            if (since == 0) since = clock64();
            if (clock64() - since > DS41_WAIT_LIMIT_CYCLES ||
                (p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != kStatusOk)) {
              if (p.status != nullptr && atomicCAS(p.status, kStatusOk, kStatusMbarTimeout) == kStatusOk) {
                p.status[1] = 511;
                p.status[2] = static_cast<int>(blockIdx.x);
                p.status[3] = pj;
              }
              ok = false;
            }
            continue;
          } else {
            continue;
          }
          idle = 0;
          since = 0;
        }
        kt += n;
      }
      ok = __ballot_sync(0xffffffffu, leader && ok) != 0;
    }
  } else if (warp == kPlRelay) {
    if (PAIR) {
      uint32_t free_there[kPlSets];
#pragma unroll
      for (int i = 0; i < kPlSets; ++i) free_there[i] = cluster_addr(smem_u32(&x_free[i]), rank ^ 1);
      bool ok = true;
      int kt = 0;
      for (int unit = first_unit; unit < units && ok; unit += unit_step) {
        const PrefixUnit it = unit == first_unit ? begin : prefix_unit(plan, unit);
        if (it.rows == 0) continue;
        int end;
        const int n = span(it, end);
        if (lane == 0)
          for (int j = 0; j < n && ok; ++j, ++kt) {
            const int set = kt % kPlSets;
            ok = mbar_wait(&x_read[set], (kt / kPlSets) & 1, p.status, 530);
            if (ok) remote_arrive(set ? free_there[1] : free_there[0]);
          }
        ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
      }
    }
  } else {
    const int set = warp >> 2, quad = warp & 3, mine = quad * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t x_there = PAIR ? cluster_addr(smem_u32(s_x) + 16 * mine, rank ^ 1) : 0;
    const uint32_t full_there = PAIR ? cluster_addr(smem_u32(&x_full[set]), rank ^ 1) : 0;
    const int before = (set + kPlSets - 1) % kPlSets;              // the set of the last tile
    int kt = 0;
    bool ok = true;
    // What a thread has to know of a unit, found while the last product of the one before it is under way.
    PrefixUnit it = begin;
    int n = 0, end = 0, r = -1, hi = 0, cell = 0;
    const int my_row = mine / p.heads, h = mine - my_row * p.heads;
    auto look = [&](const PrefixUnit& next) {
      it = next;
      PrefixRows rows = prefix_rows(plan, it, p.row_pos, p.row_slot, 0);
      r = -1;
      hi = 0;
      if (my_row < it.rows) {
        r = prefix_row(plan, it, my_row);
        cell = plan.cell[r] + it.part;
        if (p.row_slot[r] >= 0) hi = min(p.row_pos[r] + 1, it.key1);
      }
      int first;
      prefix_span(it, rows, 0, p.page_tokens, first, end);
      n = (end - first + kPlKeys - 1) / kPlKeys;
    };
    if (first_unit < units) look(begin);
    // the loop runs to its end whatever happened: the warps of a quadrant meet at barriers
    for (int unit = first_unit; unit < units; unit += unit_step) {
      const PrefixUnit next = unit + unit_step < units ? prefix_unit(plan, unit + unit_step) : it;
      if (n == 0) {                                            // nothing for any of its rows
        if (r >= 0 && set == 0 && rank == 0)
          *reinterpret_cast<float2*>(plan.part_ml + 2 * (1ll * cell * p.heads + h)) = make_float2(-INFINITY, 0.f);
        look(next);
        continue;
      }
      // queries into tensor memory, the sets in turn: all of a thread's loads are under way together
      {
        constexpr int kMine = 2 * kPlMost / kPlSets;             // pieces of 32 values
        uint32_t v[kMine][16];
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          const int c = set + kPlSets * k;
          const bool lat = c < 2 * v_chunks;
          const int d0 = lat ? v0 + 32 * c : 64 * r_chunk0 + 32 * (c - 2 * v_chunks), width = lat ? v1 : p.rp;
          const __nv_bfloat16* src = lat ? p.q_abs + r * p.ld_q_abs + 1ll * h * p.kvp + d0
                                         : p.q_rot + r * p.ld_q_rot + 1ll * h * p.q_rot_stride + d0;
          const bool there = r >= 0 && c < 2 * (v_chunks + r_chunks);
          // neighbouring threads read rows far apart: a sector of 32 bytes each
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t(&to)[8] = reinterpret_cast<uint32_t(&)[8]>(v[k][8 * i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) to[e] = 0;
            if (there && d0 + 16 * i < width) {
              if (p.wide) {
                load32(src + 16 * i, to);
              } else {
                const uint4 a = *reinterpret_cast<const uint4*>(src + 16 * i), b = *reinterpret_cast<const uint4*>(src + 16 * i + 8);
                to[0] = a.x;
                to[1] = a.y;
                to[2] = a.z;
                to[3] = a.w;
                to[4] = b.x;
                to[5] = b.y;
                to[6] = b.z;
                to[7] = b.w;
              }
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          const int c = set + kPlSets * k;
          if (c < 2 * (v_chunks + r_chunks)) tmem_st_32x16(lanes + kPlQ + 16 * c, v[k]);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      int high = hi > 0 ? hi : 0x7fffffff;
#pragma unroll
      for (int o = 16; o; o >>= 1) high = min(high, __shfl_xor_sync(0xffffffffu, high, o));
      float m = -INFINITY, l = 0.f;                              // the maximum that l is relative to
      for (int j = (set + kPlSets - kt % kPlSets) % kPlSets; j < n && ok; j += kPlSets) {
        const int tile = kt + j, use = tile / kPlSets;
        float2 s[kPlKeys / 2];
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[set], use & 1, p.status, 520)) != 0;
        if (!ok) break;
        tc_fence_after();
        {
          uint32_t a[32], b[32];
          tmem_ld_32x32(lanes + kPlS, a);
          tmem_ld_32x32(lanes + kPlS + 32, b);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            s[i] = make_float2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1]));
            s[16 + i] = make_float2(__uint_as_float(b[2 * i]), __uint_as_float(b[2 * i + 1]));
          }
        }
        if (PAIR) {                                            // [column / 4][query]: neighbouring lanes, neighbouring 16 bytes
          const uint32_t buf = (tile & 1) * kPlKeys * kPlQueries;      // its last scores, of the tile before last, have been read
          if (tile > 1)
            ok = __all_sync(0xffffffffu, cluster_wait(&x_free[(tile - 2) % kPlSets], ((tile - 2) / kPlSets) & 1, p.status, 521)) != 0;
          if (!ok) break;
          if (quad == 0 && lane == 0) mbar_expect_tx(&x_full[set], 4 * kPlKeys * kPlQueries);
#pragma unroll
          for (int i = 0; i < kPlKeys / 4; ++i)
            remote_store(x_there + 4 * buf + 16 * kPlQueries * i, full_there, s[2 * i].x, s[2 * i].y, s[2 * i + 1].x, s[2 * i + 1].y);
          ok = __all_sync(0xffffffffu, mbar_wait(&x_full[set], use & 1, p.status, 522)) != 0;
          if (!ok) break;
          const float4* x = reinterpret_cast<const float4*>(s_x + buf) + mine;
#pragma unroll
          for (int i = 0; i < kPlKeys / 4; ++i) {
            const float4 y = x[i * kPlQueries];
            s[2 * i] = add2(s[2 * i], make_float2(y.x, y.y));
            s[2 * i + 1] = add2(s[2 * i + 1], make_float2(y.z, y.w));
          }
        }
        const int key0 = it.key0 + j * kPlKeys;
        if (key0 + kPlKeys > high) {                           // the tile holds keys that a query of this warp does not see
          const int shown = hi - key0;
#pragma unroll
          for (int i = 0; i < kPlKeys / 2; ++i) {
            s[i].x = 2 * i < shown ? s[i].x : -INFINITY;
            s[i].y = 2 * i + 1 < shown ? s[i].y : -INFINITY;
          }
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kPlKeys / 2; ++i) tops[i & 3] = fmaxf(tops[i & 3], fmaxf(s[i].x, s[i].y));
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * p.scale_log2;
        if (PAIR) {                                            // every lane's scores are in registers
          __syncwarp();
          if (lane == 0) mbar_arrive(&x_read[set]);
        }
        if (tile > 0) ok = __all_sync(0xffffffffu, mbar_wait(&known[4 * before + quad], ((tile - 1) / kPlSets) & 1, p.status, 523)) != 0;
        if (!ok) break;
        float now = j > 0 ? s_top[mine] : -INFINITY;           // what O is relative to
        const bool grow = top > now + 8.f || (now == -INFINITY && top > now);
        bool last_done = tile == 0;
        if (__any_sync(0xffffffffu, grow)) {
          const float next = grow ? top : now, keep = grow ? (now == -INFINITY ? 0.f : ex2_approx(now - next)) : 1.f;
          if (j > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[before], ((tile - 1) / kPlSets) & 1, p.status, 524)) != 0;
            if (!ok) break;
            last_done = true;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < v1 - v0; c += 16) {
              uint32_t o[16];
              tmem_ld_32x16(lanes + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st_32x16(lanes + c, o);
            }
            tmem_wait_st();
            tc_fence_before();
          }
          now = next;
        }
        s_top[mine] = now;
        __syncwarp();
        if (lane == 0) mbar_arrive(&known[4 * set + quad]);
        if (now > m) l *= m == -INFINITY ? 0.f : ex2_approx(m - now);
        m = now;
        const float neg = m == -INFINITY ? 0.f : -m;
        uint32_t w[kPlKeys / 2];
        float2 sums[2] = {};
        const float2 by = make_float2(p.scale_log2, p.scale_log2), off = make_float2(neg, neg);
#pragma unroll
        for (int i = 0; i < kPlKeys / 2; ++i) {
          float2 e = fma2(s[i], by, off);
          e = make_float2(ex2_approx(e.x), ex2_approx(e.y));
          sums[i & 1] = add2(sums[i & 1], e);
          const __nv_bfloat162 q = __floats2bfloat162_rn(e.x, e.y);
          w[i] = *reinterpret_cast<const uint32_t*>(&q);
        }
        sums[0] = add2(sums[0], sums[1]);
        l += sums[0].x + sums[0].y;
        // the last tile's P has been used
        if (!last_done) ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[before], ((tile - 1) / kPlSets) & 1, p.status, 525)) != 0;
        if (!ok) break;
        tc_fence_after();
        tmem_st_32x32(lanes + kPlP, w);
        if (key0 + kPlKeys > end && end < it.key1) {
          // Places behind the last position that a row sees may hold anything, and a weight of zero does not take a NaN or an
          // infinity away: their values become zeros, two threads to a place.
          const int key = mine & (kPlKeys - 1);
          if (key0 + key >= end)
            for (int i = 8 * (mine / kPlKeys); i < 8 * v_chunks; i += (i & 7) == 7 ? 9 : 1)
              *reinterpret_cast<uint4*>(s_kv + tile % p.stages * stage_bytes + (i >> 3) * kPlChunk + key * 128 + (i & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
          fence_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[set]);
      }
      kt += n;
      // the last maximum is there; and the set of the last tile has seen the products up to the one before the last complete, so that the
      // wait that follows cannot take an earlier phase for its own
      named_barrier(1 + quad, 32 * kPlSets);
      const int key0 = it.key0, this_r = r, this_hi = hi, queries = it.rows * p.heads;
      const long long this_cell = 1ll * cell * p.heads + h;
      if (unit + unit_step < units) look(next);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[(kt - 1) % kPlSets], ((kt - 1) / kPlSets) & 1, p.status, 526)) != 0;
      tc_fence_after();
      const float all = s_top[mine];
      s_sum[set * kPlQueries + mine] = m == -INFINITY ? l : l * ex2_approx(m - all);      // without a maximum: 0, or NaN
      named_barrier(1 + quad, 32 * kPlSets);
      l = s_sum[mine];
#pragma unroll
      for (int i = 1; i < kPlSets; ++i) l += s_sum[i * kPlQueries + mine];
      m = all;
      if (ok) {
        const bool write = this_r >= 0, seen = this_hi > key0;
        if (write && set == 0 && rank == 0)
          *reinterpret_cast<float2*>(plan.part_ml + 2 * this_cell) =
              make_float2(seen ? m : -INFINITY, seen ? l : 0.f);
        float* dst = plan.part_o + (write ? this_cell : 0) * p.kvp + v0;
        if (__any_sync(0xffffffffu, write)) {
#pragma unroll 1
          for (int c = 32 * set; c < v1 - v0; c += 32 * kPlSets) {
            uint32_t o[32];
            tmem_ld_32x32(lanes + c, o);
            tmem_wait_ld();
            if (queries > kPlQueries / 2 && c + 32 <= v1 - v0) {
              store_rows(plan.part_o + v0 + c, write ? this_cell * p.kvp : -1, o);
            } else if (write) {
#pragma unroll
              for (int i = 0; i < 32; i += 8)
                if (c + i < v1 - v0) store8(dst + c + i, reinterpret_cast<const float(&)[8]>(o[i]));
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      named_barrier(1 + quad, 32 * kPlSets);                     // O, the maxima and the sums may be written again
    }
  }
  __syncthreads();
  if (PAIR) cluster_meet();                                    // nothing of this CTA's memory is written or signalled any more
  if (warp == kPlMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool PAIR>
static int launch_form(const CUtensorMap& pool, const CUtensorMap& chunks, const PrefixLatentParams& p, const ds41_prefix_plan& plan, int smem,
                       cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(prefix_latent_kernel<PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (!PAIR) return launch_pdl(prefix_latent_kernel<PAIR>, dim3(plan.grid), dim3(kPlThreads), smem, st, pool, chunks, p, plan);
  return launch_pdl_cluster(prefix_latent_kernel<PAIR>, dim3(2 * plan.grid), dim3(kPlThreads), 2, smem, st, pool, chunks, p, plan);
}

// cudaErrorNotSupported: these sizes are for the simple form
int launch_prefix_latent(const ds41_latent_attend_args& a, const ds41_prefix_plan& plan, int n_pages, cudaStream_t st) {
  const int rp = a.row_len - a.kv_pad, v_chunks = (a.kv_pad + 63) / 64;
  if (a.f32 || (a.kv_pad & 15) || (rp & 15) || a.kv_pad > 512 || plan.rows_per_unit * a.heads > kPlQueries || (a.ld_q_abs & 7) ||
      (a.ld_q_rot & 7) || (a.q_rot_stride & 7) || 1ll * n_pages * a.page_tokens >= (1ll << 31) - 1 ||
      ((reinterpret_cast<uintptr_t>(a.q_abs) | reinterpret_cast<uintptr_t>(a.q_rot) | reinterpret_cast<uintptr_t>(a.pool)) & 15))
    return cudaErrorNotSupported;
  PrefixLatentParams p{};
  if (a.page_tokens % kPlKeys == 0) p.box = kPlKeys;
  else if (kPlKeys % a.page_tokens == 0 && a.page_tokens >= 8) p.box = a.page_tokens;
  else return cudaErrorNotSupported;
  const bool pair = v_chunks > 4 || v_chunks + (rp + 63) / 64 > kPlMost;
  const int r_steps = rp / 16;
  p.v_col[1] = pair ? (v_chunks + 1) / 2 * 64 : a.kv_pad;
  if (p.v_col[1] > a.kv_pad) p.v_col[1] = a.kv_pad;
  p.v_col[2] = a.kv_pad;
  // the rotated steps go where they balance the first product
  int first = (a.kv_pad / 16 + r_steps) / 2 - p.v_col[1] / 16;
  first = first < 0 ? 0 : (first > r_steps ? r_steps : first);
  p.rot_step[1] = pair ? first : r_steps;
  p.rot_step[2] = r_steps;
  for (int c = 0; c < (pair ? 2 : 1); ++c) {
    const int r0 = p.rot_step[c], r1 = p.rot_step[c + 1];
    const int n = (p.v_col[c + 1] - p.v_col[c] + 63) / 64 + (r1 > r0 ? (r1 + 3) / 4 - r0 / 4 : 0);
    if (n > kPlMost || p.v_col[c + 1] <= p.v_col[c]) return cudaErrorNotSupported;
    p.chunks = n > p.chunks ? n : p.chunks;
  }
  constexpr int kExtra = 8 * (2 * kPlStages + 2 + 10 * kPlSets) + 8 + 4 * (1 + kPlSets) * kPlQueries;
  const int room = 227 * 1024 - kExtra - (pair ? 2 * 4 * kPlKeys * kPlQueries : 0);
  p.stages = room / (p.chunks * kPlChunk);
  if (p.stages > kPlStages) p.stages = kPlStages;
  const int smem = kExtra + (pair ? 2 * 4 * kPlKeys * kPlQueries : 0) + p.stages * p.chunks * kPlChunk;
  p.q_abs = static_cast<const __nv_bfloat16*>(a.q_abs);
  p.q_rot = static_cast<const __nv_bfloat16*>(a.q_rot);
  p.page_table = a.page_table; p.row_pos = a.row_pos; p.row_slot = a.row_slot;
  p.ld_q_abs = a.ld_q_abs; p.ld_q_rot = a.ld_q_rot; p.q_rot_stride = a.q_rot_stride;
  p.heads = a.heads; p.kvp = a.kv_pad; p.rp = rp;
  p.max_pages = a.max_pages; p.page_tokens = a.page_tokens; p.n_pages = n_pages; p.hidden_row = n_pages * a.page_tokens;
  p.wide = !((a.ld_q_abs | a.ld_q_rot | a.q_rot_stride) & 15) &&
           !((reinterpret_cast<uintptr_t>(a.q_abs) | reinterpret_cast<uintptr_t>(a.q_rot)) & 31);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = a.status;
  CUtensorMap pool;
  const cudaError_t e = make_tensor_map_3d(&pool, a.pool, TmaDtype::kBF16, a.row_len, p.hidden_row, 1, 2ull * a.row_len, 0, 64, p.box, true);
  if (e != cudaSuccess) return e;
  CUtensorMap chunks = pool;
  p.deep = p.box == kPlKeys && a.row_len % 64 == 0 && a.kv_pad % 64 == 0 && (!pair || 2 * p.v_col[1] == a.kv_pad);
  if (p.deep) {
    const cudaError_t d = make_tensor_map_3d(&chunks, a.pool, TmaDtype::kBF16, 64, p.hidden_row, a.row_len / 64, 2ull * a.row_len, 128, 64,
                                             kPlKeys, true, p.v_col[1] / 64);
    if (d != cudaSuccess) return d;
  }
  return pair ? launch_form<true>(pool, chunks, p, plan, smem, st) : launch_form<false>(pool, chunks, p, plan, smem, st);
}

}  // namespace ds41
