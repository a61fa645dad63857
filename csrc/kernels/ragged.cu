// Ragged passes: several requests with any number of new tokens each over a paged cache.
//
//  ragged_describe : positions, slots and cache rows of all new tokens from the requests' lengths, and how the attention's work is
//                    divided; nothing of it comes to the host, so that a captured pass follows its requests
//  ragged_heads    : RMS norm of every query and key head, rotation, queries as a matrix, keys and values into their cache rows
//  ragged_simple   : attention of a described pass for every type and size (ragged_attend.cu: bf16 on tcgen05)
#include <algorithm>
#include <atomic>
#include <climits>

#include "ds41_prefix.cuh"
#include "ds41_ragged.cuh"
#include "ds41_tma.h"

namespace ds41 {

constexpr int kDescribeThreads = 256, kDescribeWarps = kDescribeThreads / 32;
constexpr int kMostRequests = 4096, kMostBlocks = 8192;
constexpr int kCandidates = 16, kBins = 256;

struct DescribeArgs {
  const int *slots, *news, *lengths, *page_table;       // news: NULL, where slots and lengths are the slots and positions of rows
  int n, n_slots, max_pages, n_pages;
  int dividers;              // CTAs that divide the work and each write their share of the units; the others describe rows
};

// Sum of the block's values before this thread's, and of all of them; two numbers of 32 bits in one.  `sums`: of two calls after one another.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long (&sums)[2][kDescribeWarps], int& turn,
                                                         unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  turn ^= 1;
  if (lane == 31) sums[turn][warp] = x;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kDescribeWarps; ++w) {
    const unsigned long long y = sums[turn][w];
    if (w < warp) before += y;
    total += y;
  }
  return before + x - v;
}

// Last entry of an ascending list that is not above x; list[0] <= x.
__device__ __forceinline__ int find_last(const int* list, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A tile's time in tenths of that of a tensor-core tile pair of 128 keys, and that of what a unit begins and ends with.  Above it pieces
// are too long for the grid (60: 4 requests at 2000 of 32 and 8 heads 22.1 us instead of 15.2), below it there are too many, and joins
// (20: 40 requests at 4000 141 us instead of 135, 64 at up to 8192 300 instead of 278).
constexpr int kPairTile = 10, kTurnTile = 7, kSimpleTile = 22, kUnitCost = 45;
__device__ __forceinline__ int tile_cost(const ds41_ragged_pass& p, int rows) {
  return !p.tiled ? kSimpleTile : rows > p.turn_rows ? kPairTile : kTurnTile;
}

// A request's first row and first block are the sums of tokens and of ceil(tokens / unit_tokens) before it; a row finds its request by
// search, and its cache row is page_table[slot][position / page] * page + position % page.  Blocks whose walk is longer than the chosen
// length come in pieces, and the units are sorted by their length by counting.  A chain of dependent steps, not bytes (2 KB to 300 KB),
// bounds it: 5.1 us for 4 requests, of which an empty kernel takes 2.2; 8.3 us for 240 requests of 20200 rows in 3648 units.  So the sums are
// made by every CTA for itself rather than by a kernel before it, candidates are a warp's each, and many blocks are several CTAs'.  From rows,
// every CTA first looks for where requests begin, 256 rows at a time: 5.6 us for 4 rows, 7.5 for 240, 21 for 8192 of few requests.
__global__ void __launch_bounds__(kDescribeThreads) ragged_describe_kernel(const ds41_ragged_pass p, const DescribeArgs a) {
  extern __shared__ int rd_smem[];
  __shared__ unsigned long long scans[2][kDescribeWarps];
  __shared__ float cost_of[kCandidates];
  __shared__ int units_of[kCandidates], cells_of[kCandidates], bins[kBins], earlier[kBins], bin_sums[kBins / 32], longest, chosen, bad, first_bad;
  int scan = 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = p.kv_heads * p.v_parts, group = p.heads / p.kv_heads;
  int* row_first = rd_smem;             // [n] of every request: its first row, its first block, tokens, first token's position, slot
  int* block_first = row_first + p.requests;
  int* tokens = block_first + p.requests;
  int* begin = tokens + p.requests;
  int* slot_of = begin + p.requests;
  int* owner = slot_of + p.requests;             // [blocks] request
  int* tiles = owner + p.max_blocks;    // [blocks] key tiles
  int* first = tiles + p.max_blocks;    // [blocks] first unit of the list by blocks, first cell
  int* cells = first + p.max_blocks;
  pdl_launch_dependents();
  for (int i = tid; i < kBins; i += kDescribeThreads) bins[i] = earlier[i] = 0;
  if (tid == 0) longest = 1, bad = 0, first_bad = INT_MAX;
  pdl_wait();
  __syncthreads();
  int n = a.n;
  const bool by_rows = a.news == nullptr;
  if (by_rows) {                        // where requests begin, then how many rows they have
    int begun = 0;
    for (int r0 = 0; r0 < a.n; r0 += kDescribeThreads) {
      const int r = r0 + tid;
      int slot = -1, pos = 0;
      bool first = false;
      if (r < a.n) {
        slot = a.slots[r];
        pos = a.lengths[r];
        const int last = r > 0 ? a.slots[r - 1] : 0;
        first = r == 0 || (slot < 0 ? last >= 0 : last != slot || a.lengths[r - 1] != pos - 1);      // rows without a slot stay together
      }
      unsigned long long total;
      const int i = begun + static_cast<int>(block_scan(first, scans, scan, total));
      begun += static_cast<int>(total);
      if (first && i < p.requests) {
        row_first[i] = r;
        begin[i] = pos;
        slot_of[i] = slot;
      }
    }
    __syncthreads();
    n = min(begun, p.requests);
    if (tid == 0 && begun > n) bad = begun - n, first_bad = n;
    for (int i = tid; i < n; i += kDescribeThreads) tokens[i] = (i + 1 < begun && i + 1 < p.requests ? row_first[i + 1] : a.n) - row_first[i];
    if (begun > n) {                    // the last request that has a place ends where the next one begins
      __syncthreads();
      if (tid == 0) {
        int r = row_first[n - 1] + 1;
        const int slot = slot_of[n - 1], from = begin[n - 1] - row_first[n - 1];
        while (r < a.n && (slot < 0 ? a.slots[r] < 0 : a.slots[r] == slot && a.lengths[r] == from + r)) ++r;
        tokens[n - 1] = r - row_first[n - 1];
      }
    }
    __syncthreads();
  }
  unsigned long long base = 0;          // rows, blocks
  for (int i0 = 0; i0 < n; i0 += kDescribeThreads) {
    const int i = i0 + tid;
    int slot = -1, count = 0, length = 0;
    bool wrong = false;
    if (i < n) {
      slot = by_rows ? slot_of[i] : a.slots[i];
      count = by_rows ? tokens[i] : a.news[i];
      length = !by_rows ? a.lengths[i] : slot < 0 ? 0 : begin[i] + count;
      wrong = count < 0 || (slot >= 0 && length < count) || slot >= a.n_slots || (slot >= 0 && length > 1ll * a.max_pages * p.page_tokens);
      if (wrong) slot = -1;
    }
    const int wanted = max(count, 0), most = min(wanted, p.rows);
    unsigned long long total;
    unsigned long long at = block_scan(static_cast<unsigned long long>(most) << 32 | (most + p.unit_tokens - 1) / p.unit_tokens, scans, scan, total);
    // rows beyond the pass's are left out
    const int row = static_cast<int>(min((base + at) >> 32, static_cast<unsigned long long>(p.rows))), kept = min(most, p.rows - row);
    if (wrong || kept < wanted) {
      atomicAdd(&bad, 1);
      atomicMin(&first_bad, i);
    }
    if (((base + total) >> 32) > static_cast<unsigned>(p.rows))
      at = block_scan(static_cast<unsigned long long>(kept) << 32 | (kept + p.unit_tokens - 1) / p.unit_tokens, scans, scan, total);
    if (i < n) {
      row_first[i] = row;
      block_first[i] = static_cast<int>((base + at) & 0xffffffffu);
      tokens[i] = kept;
      begin[i] = max(0, length - wanted);
      slot_of[i] = slot;
    }
    base += total;
  }
  const int rows = static_cast<int>(base >> 32), blocks = min(static_cast<int>(base & 0xffffffffu), p.max_blocks);
  __syncthreads();

  const int divider = blockIdx.x;
  if (divider >= a.dividers) {
    const int r = (divider - a.dividers) * kDescribeThreads + tid;
    if (r < p.rows) {
      int pos = 0, slot = -1, place = -1;
      if (r < rows) {
        const int i = find_last(row_first, n, r);
        pos = by_rows ? a.lengths[r] : begin[i] + r - row_first[i];
        slot = slot_of[i];
        if (slot >= 0) {
          const int pg = pos / p.page_tokens, id = a.page_table[1ll * slot * a.max_pages + pg];
          if (static_cast<unsigned>(id) < static_cast<unsigned>(a.n_pages)) {
            place = id * p.page_tokens + (pos - pg * p.page_tokens);
          } else {
            atomicAdd(&p.report[2], 1);
            atomicMax(&p.report[3], INT_MAX - r);
          }
        }
      }
      p.row_pos[r] = pos;
      p.row_slot[r] = slot;
      p.row_place[r] = place;
    }
    // counters of calls that gave up
    for (int i = r; i < 2 * p.max_blocks * G; i += (gridDim.x - a.dividers) * kDescribeThreads) p.counters[i] = 0;
    return;
  }

  // blocks: request, key tiles
  const int align = min(p.page_tokens, p.key_tile);
  int most = 0;
  for (int b = tid; b < blocks; b += kDescribeThreads) {
    const int i = find_last(block_first, n, b), t0 = (b - block_first[i]) * p.unit_tokens, count = min(p.unit_tokens, tokens[i] - t0);
    int k = 0;
    if (slot_of[i] >= 0) {
      const RaggedWalk w = ragged_walk(begin[i] + t0, begin[i] + t0 + count - 1, p.window, p.first, AnyRuns{align});
      k = (w.places + p.key_tile - 1) / p.key_tile;
    }
    owner[b] = i;
    tiles[b] = k;
    cells[b] = count * group;
    most = max(most, k * tile_cost(p, count * group));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0 && most > 0) atomicMax(&longest, most);
  __syncthreads();
  // How long a piece may be.  A CTA's time is its pieces' tiles and what they begin and end with, and for a part of `unit_tokens` tokens
  // that has to be joined as much again to write and read it; the join comes last.
  const int longest_walk = longest;
  auto limit = [&](int k) {
    constexpr int kDivide[kCandidates] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256};
    int d = 1;
#pragma unroll
    for (int j = 0; j < kCandidates; ++j) d = k == j ? kDivide[j] : d;
    return (longest_walk + d - 1) / d;
  };
  // the same number wherever it is asked for: a product that is rounded once
  auto pieces_of = [&](int tiles, int cells, float part) {
    return max(1, min(tiles, static_cast<int>(ceilf(__fmul_rn(static_cast<float>(tiles * tile_cost(p, cells)), part)))));
  };
  const float per_full = 1.f / (p.unit_tokens * group);
  static_assert(kCandidates % kDescribeWarps == 0, "some lengths to a warp");
  for (int k = warp; k < kCandidates; k += kDescribeWarps) {
    const float part = 1.f / limit(k);
    int units = 0, parts = 0;
    float cost = 0.f;                                   // added in one order: the choice is the same every time
    for (int b = lane; b < blocks; b += 32) {
      const int pieces = pieces_of(tiles[b], cells[b], part);
      units += pieces;
      cost += static_cast<float>(tiles[b] * tile_cost(p, cells[b]) + kUnitCost * pieces);
      if (pieces > 1) {
        parts += min(pieces * cells[b], 1 << 18);
        cost += kUnitCost * per_full * static_cast<float>(pieces * cells[b]);
      }
    }
    units = __reduce_add_sync(0xffffffffu, units);
    parts = __reduce_add_sync(0xffffffffu, min(parts, 1 << 25));
    cost = warp_sum(cost);
    if (lane == 0) {
      units_of[k] = units;
      cells_of[k] = parts;
      cost_of[k] = cost;
    }
  }
  __syncthreads();
  if (warp == 0) {
    float time = INFINITY;
    if (lane < kCandidates && (lane == 0 || (1ll * units_of[lane] * G <= p.max_units && 1ll * cells_of[lane] * G <= p.max_cells))) {
      const float units = static_cast<float>(units_of[lane]) * G, turns = ceilf(units / p.grid), cost = cost_of[lane] * G;
      time = fmaxf(static_cast<float>(limit(lane) + kUnitCost), turns * cost / fmaxf(units, 1.f)) + (cells_of[lane] > 0 ? 1.5f * kUnitCost : 0.f);
    }
    float best = time;
#pragma unroll
    for (int o = 16; o; o >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, o));
    const int who = __ffs(__ballot_sync(0xffffffffu, time == best)) - 1;
    if (lane == 0) chosen = limit(who);
  }
  __syncthreads();
  const int most_cost = chosen;
  const float part = 1.f / most_cost;
  // the longest pieces first
  const int widest = longest_walk < most_cost + kSimpleTile ? longest_walk : most_cost + kSimpleTile;
  const float per_cost = (kBins - 1) / static_cast<float>(widest);
  auto bin_of = [&](int cost) { return kBins - 1 - min(kBins - 1, static_cast<int>(cost * per_cost)); };
  // this CTA's blocks
  const int share = (blocks + a.dividers - 1) / a.dividers, b_first = min(blocks, divider * share), b_end = min(blocks, b_first + share);
  unsigned long long sums = 0;
  for (int b0 = 0; b0 < blocks; b0 += kDescribeThreads) {
    const int b = b0 + tid;
    int pieces = 0, parts = 0;
    if (b < blocks) {
      const int k = tiles[b], c = tile_cost(p, cells[b]);
      pieces = pieces_of(k, cells[b], part);
      parts = pieces > 1 ? pieces * cells[b] * G : 0;
      const int least = pieces > 1 ? k / pieces : k, more = k - least * pieces;             // pieces of one tile more than the others
      if (more) atomicAdd(&bins[bin_of((least + 1) * c)], more * G);
      atomicAdd(&bins[bin_of(least * c)], (pieces - more) * G);
      if (b < b_first) {
        if (more) atomicAdd(&earlier[bin_of((least + 1) * c)], more * G);
        atomicAdd(&earlier[bin_of(least * c)], (pieces - more) * G);
      }
    }
    unsigned long long total;
    const unsigned long long at = sums + block_scan(static_cast<unsigned long long>(pieces * G) << 32 | parts, scans, scan, total);
    sums += total;
    if (b < blocks) {
      first[b] = static_cast<int>(at >> 32);
      cells[b] = static_cast<int>(at & 0xffffffffu);
    }
  }
  const int units = static_cast<int>(sums >> 32);
  __syncthreads();
  // where a bin's units begin
  static_assert(kBins == kDescribeThreads, "a bin to a thread");
  const int count = bins[tid];
  int upto = count;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) bin_sums[warp] = upto;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < kDescribeWarps; ++w) before += w < warp ? bin_sums[w] : 0;
  bins[tid] = before + upto - count + earlier[tid];
  __syncthreads();
  const bool whole = units == blocks * G;                // no block in pieces
  const int u_first = b_first < blocks ? first[b_first] : units, u_end = b_end < blocks ? first[b_end] : units;
  for (int u = u_first + tid; u < u_end; u += kDescribeThreads) {
    const int b = whole ? u / G : find_last(first, blocks, u), i = owner[b], k = tiles[b];
    const int t0 = (b - block_first[i]) * p.unit_tokens, tk = min(p.unit_tokens, tokens[i] - t0), step = tk * group;
    const int pieces = whole ? 1 : pieces_of(k, step, part), x = u - first[b], head = pieces > 1 ? x / pieces : x, piece = x - head * pieces;
    const int least = pieces > 1 ? k / pieces : k, more = k - least * pieces;
    const int mine = least + (piece < more), tile0 = piece * least + min(piece, more);
    // one thread asks for all of its warp's of a bin
    const int bin = bin_of(mine * tile_cost(p, step));
    const unsigned same = __match_any_sync(__activemask(), bin);
    const int leader = __ffs(same) - 1;
    int at = lane == leader ? atomicAdd(&bins[bin], __popc(same)) : 0;
    at = __shfl_sync(same, at, leader) + __popc(same & ((1u << lane) - 1));
    int4* out = reinterpret_cast<int4*>(p.units + 1ll * at * kRaggedInts);
    out[0] = make_int4(slot_of[i], row_first[i] + t0, tk, begin[i] + t0);
    out[1] = make_int4(head, tile0, mine, piece);
    out[2] = make_int4(pieces, cells[b] + head * pieces * step, 2 * (b * G + head), step);
  }
  if (divider == 0 && tid == 0) {
    p.header[0] = units;
    p.header[1] = rows;
    p.header[2] = bad;
    p.header[3] = first_bad;
    if (bad > 0) {                      // stays until the host has seen it, whatever passes follow
      if (p.report[0] == 0) p.report[1] = first_bad;
      p.report[0] = min(p.report[0], INT_MAX - bad) + bad;
    }
  }
}

// ---------------------------------------------------------------------------------------------------- heads
inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

constexpr int kHeadsThreads = 256;
constexpr int kMostHeadValues = 50688, kHeadsSmem = 4 * (kMostHeadValues + 1024);      // of a row's queries and keys; with the turns of 1024

// Cosine and sine of pos * freq, pos >= 0.  In turns that is pos * (freq / 2 pi), of which only the fraction counts: with freq / 2 pi as
// a whole number of 2^-64 turns it is what 64 bits hold of a product of whole numbers, as exact for far positions as for near ones (with
// the product and its reduction in 64-bit floating point, which is slow here, the rotations of 8192 rows took 12 us).
__device__ __forceinline__ unsigned long long turns_of(float freq) {
  constexpr unsigned long long kInverse = 11743562013128004906ull;       // 2^66 / (2 pi)
  const uint32_t bits = __float_as_uint(freq), exponent = bits >> 23 & 0xff;
  const unsigned long long m = (bits & 0x7fffffu) | (exponent ? 0x800000u : 0u);
  const int right = 152 - static_cast<int>(exponent ? exponent : 1);       // freq = m 2^(exponent - 150)
  const unsigned long long low = m * kInverse, high = __umul64hi(m, kInverse);
  unsigned long long x;
  if (right <= 0) x = right > -64 ? low << -right : 0;
  else if (right < 64) x = low >> right | high << (64 - right);
  else x = right < 128 ? high >> (right - 64) : 0;
  return bits >> 31 ? 0ull - x : x;
}
__device__ __forceinline__ float2 turn_at(int pos, float freq) {
  if (!(fabsf(freq) < INFINITY)) return make_float2(NAN, NAN);
  const uint32_t part = static_cast<uint32_t>(static_cast<unsigned long long>(pos) * turns_of(freq) >> 32);       // of a turn, in 2^-32
  const uint32_t quarter = (part + 0x20000000u) >> 30;
  float s, c;
  sincospif(static_cast<float>(static_cast<int>(part - (quarter << 30))) * 4.6566128730773926e-10f, &s, &c);     // within an eighth; 2^-31
  const float x = quarter & 1 ? -s : c, y = quarter & 1 ? c : s;
  return quarter & 2 ? make_float2(-x, -y) : make_float2(x, y);
}

// Any sizes: one block per row, whose heads stay in shared memory between the norm and the rotation.  For heads that are not whole
// sixteens, and rows that do not begin at 16 bytes; 8192 rows of 32 and 8 heads of 128 take it 166 us, those of the form below 47.
// The turns come first, as pairs of 8 bytes: behind the heads they would lie at any multiple of 4.
template <typename T>
__global__ void __launch_bounds__(kHeadsThreads) ragged_heads_kernel(const ds41_ragged_heads_args p) {
  extern __shared__ __align__(16) float2 rh_turns[];     // [rot_dim / 2], then [(heads + kv_heads) * dim] values
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, half = p.rot_dim / 2;
  const int H = p.heads, G = p.kv_heads, D = p.dim, V = p.vdim;
  float* const rh_row = reinterpret_cast<float*>(rh_turns + half);
  pdl_launch_dependents();
  pdl_wait();
  const int place = p.row_place[r], pos = p.row_pos[r];
  if (place < 0 || place >= p.pool_rows) return;
  for (int i = tid; i < half; i += kHeadsThreads) rh_turns[i] = turn_at(pos, p.freq[i]);
  __syncthreads();
  T* row = static_cast<T*>(p.pool) + 1ll * place * (G * (D + V));
  T* q = static_cast<T*>(p.q_out) + r * p.ld_q;
  for (int h = warp; h < H + G; h += kHeadsThreads / 32) {
    const bool key = h >= H;
    const int g = key ? h - H : h;
    float* x = rh_row + h * D;
    float sum = 0.f;
    for (int d = lane; d < D; d += 32) {
      const float v = proj_at(key ? p.k : p.q, r, g * D + d);
      x[d] = v;
      sum += v * v;
    }
    const float* w = key ? p.k_norm : p.q_norm;
    const float f = w != nullptr ? 1.0f / sqrtf(warp_sum(sum) / p.width + p.eps) : 1.f;
    if (w != nullptr) w += 1ll * g * (key ? p.k_norm_stride : p.q_norm_stride);
    __syncwarp();
    T* dst = key ? row + g * D : q + g * D;
    for (int d = lane; d < D; d += 32) {
      float v = x[d] * f * (w != nullptr ? w[d] : 1.f);
      if (d < 2 * half) {
        const int e = d < half ? d + half : d - half;
        const float o = x[e] * f * (w != nullptr ? w[e] : 1.f);
        const float2 t = rh_turns[d < half ? d : e];
        v = d < half ? v * t.x - o * t.y : v * t.x + o * t.y;
      }
      dst[d] = from_f32<T>(v);
    }
  }
  for (int c = tid; c < G * V; c += kHeadsThreads) row[G * D + c] = from_f32<T>(proj_at(p.v, r, c));
}

// Heads of multiples of 16 values and rotations of multiples of 16, rows of whole 16 bytes.  A lane has 16 values of a head: in its rotated
// part eight and the eight that they turn with, else neighbours; as many lanes as a head has sixteens (or the next power of two) share
// it.  A warp takes `per` steps of one row, in each of which its lanes have neighbouring heads, and keeps its lanes' turns and weights.
// y = x / sqrt(mean x^2 + eps) * w, then (y_j, y_{j + n}) turned by pos * freq_j.  Bound by memory: what is read and written is read and
// written once, in whole lines.  8192 rows of 32 and 8 heads of 128 in bf16: 201 MB in 47 us, 4.3 TB/s, where a plain copy of as much takes
// 31: 24 warps a multiprocessor, whose loads wait behind their own arithmetic (issue slots 57 % busy).  Five further layouts, with
// 16 to 48 warps and loads one to three steps ahead, took 47 to 58.  16 rows: 3.0 us, the launch and three dependent loads.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
// Sixteen values as two rows of eight, in pairs.
struct Sixteen {
  float2 a[4], b[4];
};
template <bool PACKED>
struct RawSixteen {
  uint4 a, b;
  __device__ __forceinline__ void load(const ds41_proj& p, long long at, int ca, int cb) {
    const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(p.data) + at;
    a = *reinterpret_cast<const uint4*>(row + ca);
    b = *reinterpret_cast<const uint4*>(row + cb);
  }
  __device__ __forceinline__ Sixteen get() const {
    const uint32_t q[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    Sixteen x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x.a[i] = make_float2(__uint_as_float(q[i] << 16), __uint_as_float(q[i] & 0xffff0000u));
      x.b[i] = make_float2(__uint_as_float(q[4 + i] << 16), __uint_as_float(q[4 + i] & 0xffff0000u));
    }
    return x;
  }
};
template <>
struct RawSixteen<false> {
  float4 q[4];
  __device__ __forceinline__ void load(const ds41_proj& p, long long at, int ca, int cb) {
    ds41_proj row = p;
    row.col = 0;
    row.data = p.bf16 ? static_cast<const void*>(static_cast<const __nv_bfloat16*>(p.data) + at)
                      : static_cast<const void*>(static_cast<const float*>(p.data) + at);
    q[0] = proj_at4(row, 0, ca);
    q[1] = proj_at4(row, 0, ca + 4);
    q[2] = proj_at4(row, 0, cb);
    q[3] = proj_at4(row, 0, cb + 4);
  }
  __device__ __forceinline__ Sixteen get() const {
    Sixteen x;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x.a[2 * i] = make_float2(q[i].x, q[i].y);
      x.a[2 * i + 1] = make_float2(q[i].z, q[i].w);
      x.b[2 * i] = make_float2(q[2 + i].x, q[2 + i].y);
      x.b[2 * i + 1] = make_float2(q[2 + i].z, q[2 + i].w);
    }
    return x;
  }
};
__device__ __forceinline__ void store_eight(float* to, const float2 (&v)[4]) {
  store4(to, make_float4(v[0].x, v[0].y, v[1].x, v[1].y));
  store4(to + 4, make_float4(v[2].x, v[2].y, v[3].x, v[3].y));
}
__device__ __forceinline__ void store_eight(__nv_bfloat16* to, const float2 (&v)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 q = __float22bfloat162_rn(v[i]);
    w[i] = *reinterpret_cast<const uint32_t*>(&q);
  }
  *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct HeadsSteps {
  int q, qk, all;            // steps of queries, of queries and keys, and with the values
  int per, parts;            // steps of a warp, warps of a row
  float inverse;             // 1 / width
};

template <typename T, bool PACKED, int LANES>
__global__ void __launch_bounds__(kHeadsThreads, PACKED ? 3 : 2) ragged_heads_wide_kernel(const ds41_ragged_heads_args p, const HeadsSteps h) {
  extern __shared__ __align__(16) float2 rw_turns[];     // [warps][rot_dim / 2]
  constexpr int kStep = 32 / LANES;                      // heads of a step
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = p.rot_dim / 2;
  const int G = p.kv_heads, D = p.dim, unit = lane % LANES, own = lane / LANES;
  const unsigned w = blockIdx.x * (kHeadsThreads / 32) + warp;
  const int r = static_cast<int>(w / h.parts), s0 = static_cast<int>(w % h.parts) * h.per, s1 = min(h.all, s0 + h.per);
  const bool inside = 16 * unit < D, turned = 16 * unit < p.rot_dim;
  const int ca = turned ? 8 * unit : 16 * unit, cb = turned ? half + 8 * unit : ca + 8;
  pdl_launch_dependents();
  pdl_wait();
  if (r >= p.rows) return;
  const int place = p.row_place[r], pos = p.row_pos[r];
  const bool turns = half > 0 && s0 < h.qk;
  const float freq = turns && lane < half ? p.freq[lane] : 0.f;
  const long long q_at = 1ll * r * p.q.ld + p.q.col, k_at = 1ll * r * p.k.ld + p.k.col, v_at = 1ll * r * p.v.ld + p.v.col;
  // this lane's head at a step of queries or keys
  auto head = [&](int s) { return (s - (s < h.q ? 0 : h.q)) * kStep + own; };
  auto lives = [&](int s) { return inside && head(s) < (s < h.q ? p.heads : G); };
  auto fetch = [&](int s, RawSixteen<PACKED>& raw) {
    if (s < h.q) {
      if (lives(s)) raw.load(p.q, q_at + head(s) * D, ca, cb);
    } else if (s < h.qk) {
      if (lives(s)) raw.load(p.k, k_at + head(s) * D, ca, cb);
    } else {
      const int c = (s - h.qk) * 512 + 16 * lane;
      if (c < G * p.vdim) raw.load(p.v, v_at + c, 0, 8);
    }
  };
  // what the first step needs is asked for before any of it is looked at
  RawSixteen<PACKED> next;
  fetch(s0, next);
  Sixteen weight;
  auto weights = [&](int s) {
    const float* norm = s < h.q ? p.q_norm : p.k_norm;
    if (norm == nullptr || !lives(s)) return;
    norm += 1ll * head(s) * (s < h.q ? p.q_norm_stride : p.k_norm_stride);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      weight.a[e] = *reinterpret_cast<const float2*>(norm + ca + 2 * e);
      weight.b[e] = *reinterpret_cast<const float2*>(norm + cb + 2 * e);
    }
  };
  if (s0 < h.qk) weights(s0);
  if (place < 0 || place >= p.pool_rows) return;
  float2 cosine[4], sine[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) cosine[e] = make_float2(1.f, 1.f), sine[e] = make_float2(0.f, 0.f);
  if (turns) {
    float2* mine = rw_turns + warp * half;
    if (lane < half) mine[lane] = turn_at(pos, freq);
    for (int i = lane + 32; i < half; i += 32) mine[i] = turn_at(pos, p.freq[i]);
    __syncwarp();
    if (turned)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 t = *reinterpret_cast<const float4*>(mine + 8 * unit + 2 * e);
        cosine[e] = make_float2(t.x, t.z);
        sine[e] = make_float2(t.y, t.w);
      }
  }
  T* row = static_cast<T*>(p.pool) + 1ll * place * (G * (D + p.vdim));
  T* q = static_cast<T*>(p.q_out) + r * p.ld_q;
  for (int s = s0; s < s1; ++s) {
    Sixteen x = next.get();
    if (s + 1 < s1) fetch(s + 1, next);
    if (s >= h.qk) {
      const int c = (s - h.qk) * 512 + 16 * lane;
      if (c < G * p.vdim) {
        store_eight(row + G * D + c, x.a);
        store_eight(row + G * D + c + 8, x.b);
      }
      continue;
    }
    // the last queries' step may leave lanes without a head that have one among the keys
    if (s > s0 && (s == h.q || (s < h.q ? p.q_norm_stride : p.k_norm_stride) > 0)) weights(s);
    const bool live = lives(s);
    if ((s < h.q ? p.q_norm : p.k_norm) != nullptr) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fma2(x.b[e], x.b[e], fma2(x.a[e], x.a[e], sum));
      float all = live ? sum.x + sum.y : 0.f;
#pragma unroll
      for (int o = LANES / 2; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      const float f = rsqrtf(all * h.inverse + p.eps);
      const float2 f2 = make_float2(f, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x.a[e] = mul2(mul2(x.a[e], f2), weight.a[e]);
        x.b[e] = mul2(mul2(x.b[e], f2), weight.b[e]);
      }
    }
    if (turned) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 u = x.a[e], v = x.b[e], minus = make_float2(-sine[e].x, -sine[e].y);
        x.a[e] = fma2(u, cosine[e], mul2(v, minus));
        x.b[e] = fma2(v, cosine[e], mul2(u, sine[e]));
      }
    }
    if (live) {
      T* to = (s < h.q ? q : row) + head(s) * D;
      store_eight(to + ca, x.a);
      store_eight(to + cb, x.b);
    }
  }
}

template <typename T, bool PACKED, int LANES>
cudaError_t launch_heads_lanes(const ds41_ragged_heads_args& a, cudaStream_t st) {
  HeadsSteps h{};
  constexpr int kStep = 32 / LANES;
  h.q = (a.heads + kStep - 1) / kStep;
  h.qk = h.q + (a.kv_heads + kStep - 1) / kStep;
  h.all = h.qk + (a.kv_heads * a.vdim + 511) / 512;
  h.inverse = 1.f / a.width;
  // few rows: a warp for every step; many: half of a row, whose turns are made once (8192 rows of 32 and 8 heads: 47.1 us, whole rows 47.6,
  // thirds 50)
  h.per = static_cast<int>(std::min<long long>(h.all, std::max<long long>(1, 1ll * a.rows * h.all / (148 * 100))));
  h.parts = (h.all + h.per - 1) / h.per;
  const long long blocks = (1ll * a.rows * h.parts + kHeadsThreads / 32 - 1) / (kHeadsThreads / 32);
  if (blocks > INT_MAX / 8) return cudaErrorInvalidValue;
  const int smem = kHeadsThreads / 32 * a.rot_dim / 2 * static_cast<int>(sizeof(float2));
  return launch_pdl(ragged_heads_wide_kernel<T, PACKED, LANES>, dim3(static_cast<unsigned>(blocks)), dim3(kHeadsThreads), smem, st, a, h);
}
template <typename T, bool PACKED>
cudaError_t launch_heads_wide(const ds41_ragged_heads_args& a, cudaStream_t st) {
  if (a.dim <= 16) return launch_heads_lanes<T, PACKED, 1>(a, st);
  if (a.dim <= 32) return launch_heads_lanes<T, PACKED, 2>(a, st);
  if (a.dim <= 64) return launch_heads_lanes<T, PACKED, 4>(a, st);
  if (a.dim <= 128) return launch_heads_lanes<T, PACKED, 8>(a, st);
  if (a.dim <= 256) return launch_heads_lanes<T, PACKED, 16>(a, st);
  return launch_heads_lanes<T, PACKED, 32>(a, st);
}

inline bool packed_row(const ds41_proj& p) {
  return p.bf16 && !(p.ld & 7) && !(p.col & 7) && !(reinterpret_cast<uintptr_t>(p.data) & 15);
}

// ---------------------------------------------------------------------------------------------------- attention, any type and size
constexpr int kSimpleRows = 64, kSimpleKeyTile = 32, kRaggedThreads = 256, kRaggedWarps = kRaggedThreads / 32;

__device__ __forceinline__ float4 four_at(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four_at(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                     __uint_as_float(v.y & 0xffff0000u));
}

inline int ragged_simple_smem(const ds41_ragged_pass& p) {
  const int ds = p.dim + 4;
  return 4 * (kSimpleRows * ds + kSimpleKeyTile * ds + kSimpleKeyTile * p.vdim + kSimpleRows * (kSimpleKeyTile + 1) + 3 * kSimpleRows);
}

// A unit's (token, head) rows, 64 at a time, against its keys, 32 at a time, both through shared memory: scores of 2 x 4 a thread, four
// threads to a row's softmax, and RPT rows x 4 columns of the result in a thread's registers.  fp32 products, since the tensor core has none
// of 24 bits; bf16 takes it where pages are not of 16 to 128 tokens or whole 128s (16 x 1 over 4000: 738 us with pages of 48, 59 of 64).  Bound by latency
// in small calls (3 + 2 x 50 rows over 500, 6 heads of 32 and 48: 19 to 22 us, launch and loads 3.4, a tile 5.5, the join 9) and by shared
// memory's reads in large ones (32 and 8 heads of 128 in fp32: 1000 tokens 0.51 ms, 8 x 1000 3.3, 16 x 1 over 4000 0.68).
template <typename T, int RPT>
__global__ void __launch_bounds__(kRaggedThreads) ragged_simple_kernel(const ds41_ragged_attend_args a, const ds41_ragged_pass p) {
  extern __shared__ __align__(16) float rs_smem[];
  __shared__ int flag, places[kSimpleRows];
  const int D = p.dim, V = p.vdim, G = p.kv_heads, group = p.heads / G, ds = D + 4, nc = V / 4, row_len = G * (D + V);
  float* qs = rs_smem;                                 // [64][ds]
  float* ks = qs + kSimpleRows * ds;                   // [32][ds]
  float* vs = ks + kSimpleKeyTile * ds;                // [32][V]
  float* sc = vs + kSimpleKeyTile * V;                 // [64][33] scores, then weights
  float* ms = sc + kSimpleRows * (kSimpleKeyTile + 1); // [64] maxima, sums, factors on what was summed before
  float* ls = ms + kSimpleRows;
  float* keep = ls + kSimpleRows;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int units = p.header[0];
  const int align = min(p.page_tokens, p.key_tile);
  const float scale = a.scale * kLog2E;
  for (int it = blockIdx.x; it < units; it += gridDim.x) {
    const RaggedUnit u = ragged_unit(p, it);
    const int n = u.tokens * group;
    if (u.slot < 0) {
      for (int i = tid; i < n * nc; i += kRaggedThreads) {
        const int r = i / nc, row = u.row0 + r / group, h = u.head * group + r % group;
        store4(static_cast<T*>(a.out) + row * a.out_row + 1ll * h * V + 4 * (i - r * nc), make_float4(0.f, 0.f, 0.f, 0.f));
      }
      continue;
    }
    const RaggedWalk walk = ragged_walk(u.pos0, u.pos0 + u.tokens - 1, p.window, p.first, AnyRuns{align});
    const int v0 = u.tile0 * p.key_tile, v1 = min(walk.places, v0 + u.tiles * p.key_tile);
    for (int r0 = 0; r0 < n; r0 += kSimpleRows) {
      const int rows = min(kSimpleRows, n - r0);
      __syncthreads();
      for (int d = 4 * lane; d < D; d += 128) {          // a warp's rows together
        float4 x[kSimpleRows / kRaggedWarps];
#pragma unroll
        for (int i = 0; i < kSimpleRows / kRaggedWarps; ++i) {
          const int r = warp + i * kRaggedWarps, row = u.row0 + (r0 + r) / group, h = u.head * group + (r0 + r) % group;
          x[i] = r < rows ? four_at(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < kSimpleRows / kRaggedWarps; ++i) *reinterpret_cast<float4*>(qs + (warp + i * kRaggedWarps) * ds + d) = x[i];
      }
      if (tid < kSimpleRows) {
        ms[tid] = -INFINITY;
        ls[tid] = 0.f;
        places[tid] = tid < rows ? p.row_place[u.row0 + (r0 + tid) / group] : -1;
      }
      float4 acc[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      const int col = tid % nc, own = tid / nc * RPT;
      for (int t0 = v0; t0 < v1; t0 += kSimpleKeyTile) {
        __syncthreads();
        constexpr int kOwn = kSimpleKeyTile / kRaggedWarps;
        const T* src[kOwn];                              // a warp's keys together
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int place = t0 + warp + i * kRaggedWarps, pos = place < walk.lead ? place : place + walk.shift, pg = pos / p.page_tokens;
          // a key that some row sees; other places may hold anything
          const bool seen = place < v1 && (pos < p.first || pos >= ragged_low(u.pos0, p.window));
          const int id = seen && pg < a.max_pages ? a.page_table[1ll * u.slot * a.max_pages + pg] : -1;
          src[i] = static_cast<unsigned>(id) < static_cast<unsigned>(a.n_pages)
                       ? static_cast<const T*>(a.pool) + (1ll * id * p.page_tokens + (pos - pg * p.page_tokens)) * row_len : nullptr;
        }
        for (int d = 4 * lane; d < max(D, V); d += 128) {
          float4 x[kOwn], y[kOwn];
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            x[i] = src[i] != nullptr && d < D ? four_at(src[i] + u.head * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            y[i] = src[i] != nullptr && d < V ? four_at(src[i] + G * D + u.head * V + d) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            if (d < D) *reinterpret_cast<float4*>(ks + (warp + i * kRaggedWarps) * ds + d) = x[i];
            if (d < V) *reinterpret_cast<float4*>(vs + (warp + i * kRaggedWarps) * V + d) = y[i];
          }
        }
        __syncthreads();
        const int ty = tid >> 3, tx = tid & 7;
        if (2 * ty < rows) {
          float s[2][4] = {};
          for (int d = 0; d < D; d += 4) {
            const float4 q0 = *reinterpret_cast<const float4*>(qs + 2 * ty * ds + d);
            const float4 q1 = *reinterpret_cast<const float4*>(qs + (2 * ty + 1) * ds + d);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float4 x = *reinterpret_cast<const float4*>(ks + (tx + 8 * k) * ds + d);
              s[0][k] += q0.x * x.x + q0.y * x.y + q0.z * x.z + q0.w * x.w;
              s[1][k] += q1.x * x.x + q1.y * x.y + q1.z * x.z + q1.w * x.w;
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) sc[(2 * ty + j) * (kSimpleKeyTile + 1) + tx + 8 * k] = s[j][k] * scale;
        }
        __syncthreads();
        {
          const int r = tid >> 2, part = tid & 3, pos = u.pos0 + (r0 + r) / group, low = ragged_low(pos, p.window);
          float* mine = sc + r * (kSimpleKeyTile + 1);
          float v[8], top = -INFINITY;
          bool bad = false;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int place = t0 + part + 4 * k, at = place < walk.lead ? place : place + walk.shift;
            const bool seen = r < rows && place < v1 && at <= pos && (at >= low || at < p.first);
            v[k] = seen ? mine[part + 4 * k] : -INFINITY;
            bad |= v[k] != v[k];
            top = fmaxf(top, v[k]);
          }
          if (bad) top = NAN;
#pragma unroll
          for (int o = 1; o < 4; o *= 2) {
            const float y = __shfl_xor_sync(0xffffffffu, top, o);
            top = top != top || y != y ? NAN : fmaxf(top, y);
          }
          const float m = ms[r];
          const float m_new = top != top || m != m ? NAN : fmaxf(m, top), base = m_new == -INFINITY ? 0.f : m_new;
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float w = exp2f(v[k] - base);
            mine[part + 4 * k] = w;
            sum += w;
          }
#pragma unroll
          for (int o = 1; o < 4; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          __syncwarp();
          if (part == 0) {
            const float f = m == -INFINITY ? 0.f : exp2f(m - base);
            ms[r] = m_new;
            ls[r] = ls[r] * f + sum;
            keep[r] = f;
          }
        }
        __syncthreads();
        if (own < rows) {
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float f = keep[own + i];
            acc[i].x *= f;
            acc[i].y *= f;
            acc[i].z *= f;
            acc[i].w *= f;
          }
#pragma unroll 4
          for (int k = 0; k < kSimpleKeyTile; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(vs + k * V + 4 * col);
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
              const float w = sc[(own + i) * (kSimpleKeyTile + 1) + k];
              acc[i].x += w * v.x;
              acc[i].y += w * v.y;
              acc[i].z += w * v.z;
              acc[i].w += w * v.w;
            }
          }
        }
      }
      __syncthreads();
      if (own < kSimpleRows) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const int r = own + i;
          if (r >= rows) continue;
          const float m = ms[r], l = ls[r];
          const int row = u.row0 + (r0 + r) / group, h = u.head * group + (r0 + r) % group;
          if (u.pieces > 1) {
            const long long cell = 1ll * u.cell + 1ll * u.piece * u.step + r0 + r;
            store4(p.part_o + cell * V + 4 * col, acc[i]);
            if (col == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * cell) = make_float2(m, l);
            continue;
          }
          const float sink = a.sink != nullptr ? a.sink[h] * kLog2E : -INFINITY;
          const float whole = fmaxf(m, sink), base = whole == -INFINITY ? 0.f : whole;
          const float w = m == -INFINITY ? 0.f : exp2f(m - base);
          const float den = l * w + (a.sink != nullptr ? exp2f(sink - base) : 0.f);
          float f = w / den;
          if (a.gate.data != nullptr) f *= sigmoid_f32(proj_at(a.gate, row, h));
          store4(static_cast<T*>(a.out) + row * a.out_row + 1ll * h * V + 4 * col,
                 places[r] >= 0 ? make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f) : make_float4(0.f, 0.f, 0.f, 0.f));
        }
      }
    }
    if (u.pieces > 1 && ragged_last(p.counters + u.counter, u.pieces, tid == 0, 1, kRaggedThreads, &flag))
      ragged_join<T>(p, a, u, 0, n, warp, kRaggedWarps);
  }
}

template <typename T, int RPT>
cudaError_t launch_simple(const ds41_ragged_attend_args& a, const ds41_ragged_pass& p, cudaStream_t st) {
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(ragged_simple_kernel<T, RPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  return launch_pdl(ragged_simple_kernel<T, RPT>, dim3(p.grid), dim3(kRaggedThreads), ragged_simple_smem(p), st, a, p);
}

template <typename T>
cudaError_t launch_ragged_simple(const ds41_ragged_attend_args& a, const ds41_ragged_pass& p, cudaStream_t st) {
  const int groups = kRaggedThreads / (p.vdim / 4), need = (kSimpleRows + groups - 1) / groups;
  if (need <= 1) return launch_simple<T, 1>(a, p, st);
  if (need <= 2) return launch_simple<T, 2>(a, p, st);
  if (need <= 4) return launch_simple<T, 4>(a, p, st);
  if (need <= 8) return launch_simple<T, 8>(a, p, st);
  return launch_simple<T, 16>(a, p, st);
}

inline bool ragged_pass_ok(const ds41_ragged_pass* p) {
  if (p == nullptr || p->header == nullptr || p->row_pos == nullptr || p->row_slot == nullptr || p->row_place == nullptr ||
      p->units == nullptr || p->counters == nullptr || p->part_o == nullptr || p->part_ml == nullptr || p->status == nullptr || p->report == nullptr)
    return false;
  if (p->rows <= 0 || p->rows > 1 << 18 || p->requests <= 0 || p->requests > kMostRequests || p->heads <= 0 || p->kv_heads <= 0 ||
      p->heads % p->kv_heads || p->heads / p->kv_heads > 1024 || p->dim <= 0 || p->dim > 256 || (p->dim & 15) || p->vdim <= 0 ||
      p->vdim > 256 || (p->vdim & 15) || p->page_tokens <= 0 || p->window < 0 || p->first < 0 || p->unit_tokens <= 0 || p->grid <= 0 ||
      p->turn_rows < 0 || (p->v_parts != 1 && (p->v_parts != 2 || !p->tiled || p->vdim & 31)))
    return false;
  return p->max_blocks >= p->rows / p->unit_tokens + std::min(p->requests, p->rows) && p->max_blocks <= kMostBlocks &&
         p->max_units >= 1ll * p->max_blocks * p->kv_heads * p->v_parts && p->max_units < 1 << 22 && p->max_cells > 0 && p->max_cells < 1 << 22 &&
         aligned(p->units, 16) && aligned(p->part_o, 32) && aligned(p->part_ml, 8) && p->key_tile == (p->tiled ? 128 : 32);
}

}  // namespace ds41

using namespace ds41;

static int describe(const ds41_ragged_pass* p, const DescribeArgs& given, void* stream) {
  DescribeArgs a = given;
  if (a.n < 0 || a.n_slots <= 0 || a.max_pages <= 0 || a.n_pages <= 0 || a.page_table == nullptr ||
      (a.n > 0 && (a.slots == nullptr || a.lengths == nullptr)) || 1ll * a.n_pages * p->page_tokens > INT_MAX ||
      1ll * a.max_pages * p->page_tokens > 1 << 30)
    return cudaErrorInvalidValue;
  const int smem = 4 * (5 * p->requests + 4 * p->max_blocks);
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(ragged_describe_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * (5 * kMostRequests + 4 * kMostBlocks));
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  // 456 blocks in 3648 units: 14.1 us with one divider
  a.dividers = std::min(8, (p->max_blocks + 31) / 32);
  const int grid = a.dividers + (p->rows + kDescribeThreads - 1) / kDescribeThreads;
  return launch_pdl(ragged_describe_kernel, dim3(grid), dim3(kDescribeThreads), smem, static_cast<cudaStream_t>(stream), *p, a);
}

extern "C" int ds41_ragged_describe(const ds41_ragged_pass* p, const int* slots, const int* news, const int* lengths, int n,
                                    const int* page_table, int n_slots, int max_pages, int n_pages, void* stream) {
  static const int none = 0;
  if (!ragged_pass_ok(p) || n > p->requests || (n > 0 && news == nullptr)) return cudaErrorInvalidValue;
  return describe(p, DescribeArgs{slots, n > 0 ? news : &none, lengths, page_table, n, n_slots, max_pages, n_pages, 0}, stream);
}

extern "C" int ds41_ragged_describe_rows(const ds41_ragged_pass* p, const int* row_pos, const int* row_slot, int n, const int* page_table,
                                         int n_slots, int max_pages, int n_pages, void* stream) {
  if (!ragged_pass_ok(p) || n > p->rows) return cudaErrorInvalidValue;
  return describe(p, DescribeArgs{row_slot, nullptr, row_pos, page_table, n, n_slots, max_pages, n_pages, 0}, stream);
}

extern "C" int ds41_ragged_heads(const ds41_ragged_heads_args* a, void* stream) {
  if (a == nullptr || a->rows <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->dim <= 0 || a->vdim <= 0 || a->dim > 1024 ||
      a->heads > 4096 || a->kv_heads > 4096 || a->rot_dim < 0 || (a->rot_dim & 1) || a->rot_dim > a->dim || a->width <= 0 || a->width > a->dim ||
      !proj_ok(a->q) || !proj_ok(a->k) || !proj_ok(a->v) || (a->rot_dim > 0 && a->freq == nullptr) || a->row_pos == nullptr ||
      a->row_place == nullptr || a->q_out == nullptr || a->pool == nullptr || a->pool_rows <= 0 || a->ld_q < 1ll * a->heads * a->dim ||
      a->q_norm_stride < 0 || a->k_norm_stride < 0 || (a->heads + a->kv_heads) * a->dim > kMostHeadValues ||
      1ll * a->kv_heads * (1ll * a->dim + a->vdim) > INT_MAX)
    return cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!(a->dim & 15) && a->dim <= 512 && !(a->rot_dim & 15) && !(a->kv_heads * a->vdim & 15) && !(a->ld_q & 7) && aligned(a->q_out, 16) &&
      aligned(a->pool, 16) && (a->q_norm == nullptr || aligned(a->q_norm, 16)) && (a->k_norm == nullptr || aligned(a->k_norm, 16)) &&
      !(a->q_norm_stride & 3) && !(a->k_norm_stride & 3)) {
    if (packed_row(a->q) && packed_row(a->k) && packed_row(a->v))
      return a->f32 ? launch_heads_wide<float, true>(*a, st) : launch_heads_wide<__nv_bfloat16, true>(*a, st);
    if (proj_vec4(a->q) && proj_vec4(a->k) && proj_vec4(a->v))
      return a->f32 ? launch_heads_wide<float, false>(*a, st) : launch_heads_wide<__nv_bfloat16, false>(*a, st);
  }
  const int smem = (a->heads + a->kv_heads) * a->dim * 4 + a->rot_dim * 4;
  auto kernel = a->f32 ? ragged_heads_kernel<float> : ragged_heads_kernel<__nv_bfloat16>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeadsSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(a->rows), dim3(kHeadsThreads), smem, st, *a);
}

extern "C" int ds41_ragged_attend(const ds41_ragged_attend_args* a, const ds41_ragged_pass* p, void* stream) {
  if (!ragged_pass_ok(p) || a == nullptr || a->q == nullptr || a->pool == nullptr || a->page_table == nullptr || a->out == nullptr ||
      a->q_rows < p->rows || a->max_pages <= 0 || a->n_pages <= 0 || 1ll * a->n_pages * p->page_tokens > INT_MAX || !(a->scale > 0.f) ||
      a->q_head < p->dim || a->q_row < 0 || a->out_row < 1ll * p->heads * p->vdim || (a->gate.data != nullptr && !proj_ok(a->gate)))
    return cudaErrorInvalidValue;
  const int size = p->f32 ? 4 : 2;
  if (!aligned(a->q, 16) || !aligned(a->pool, 16) || !aligned(a->out, 16) || (a->q_row * size & 15) || (a->q_head * size & 15) ||
      (a->out_row * size & 15))
    return cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->tiled) return launch_ragged_tiled(*a, *p, st);
  return p->f32 ? launch_ragged_simple<float>(*a, *p, st) : launch_ragged_simple<__nv_bfloat16>(*a, *p, st);
}
