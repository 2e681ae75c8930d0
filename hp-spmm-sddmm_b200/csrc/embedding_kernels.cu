// Rows of a table by id, and the gradient of the table.
//   out[t]    = scale * table[id[t]]                       a row of zeros where id[t] lies outside [0, N)
//   dTable[v] = scale * sum over t with id[t] = v of dOut[t]
// It is the product of a pattern with one entry to a row, and the product of its transpose, without a CSR of either.
#include <algorithm>

#include "dense_types.cuh"
#include "device_utils.cuh"
#include "hpspmm_internal.h"

namespace {

using namespace hpspmm;

constexpr int kThreads = 256;

// A group of W lanes to a piece of 4 W vectors of one row, all of them in flight at once.  Bound by memory: 262,144 rows of
// 2048 bf16 out of as many 230 us, 5.8 TB/s; 32 rows 2.0 us.
template <typename T, int BYTES, int W>
__global__ void __launch_bounds__(kThreads)
lookup_kernel(int64_t groups, int pieces, int per_row, int N, const void* ids, int wide, const T* table, int64_t ld, float scale,
              T* __restrict__ out) {
  typedef dense_vec<T, BYTES> vec;
  chain_grid();
  const int64_t group = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / W;
  if (group >= groups) return;
  const int64_t t = pieces == 1 ? group : group / pieces;
  // (unsigned: a row may have nearly 2^31 vectors, and the last lanes step past its end)
  const unsigned first = (unsigned)(group - t * pieces) * (4 * W) + (threadIdx.x & (W - 1)), vectors = per_row;
  const int id = load_id(ids, wide, t, N);
  const T* src = table + (int64_t)id * ld;
  T* to = out + t * ((int64_t)per_row * vec::kCount);
  vec v[4];
  if (id >= 0) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (first + u * W < vectors) v[u].raw = *reinterpret_cast<const decltype(v[u].raw)*>(src + (int64_t)(first + u * W) * vec::kCount);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (first + u * W < vectors) {
#pragma unroll
      for (int e = 0; e < vec::kCount; ++e) v[u].at[e] = from_float<T>(id >= 0 ? scale * to_float(v[u].at[e]) : 0.f);
      reinterpret_cast<decltype(v[u].raw)*>(to)[first + u * W] = v[u].raw;
    }
}

// ---- positions sorted by id ----------------------------------------------------------------------------------------
//
// Key of a position: its id, N where that lies outside the table.  The sort is stable, so that every row of the gradient
// is a sum over ascending positions.

__device__ __forceinline__ int key_of(const void* ids, int wide, int64_t at, int N) {
  const int id = load_id(ids, wide, at, N);
  return id >= 0 ? id : N;
}

// Up to kRankMost positions: every one counts how many come before it in the order of (key, position).  n^2 / 8 comparisons
// of a thread's eighth of the keys, all in shared memory; one launch where the radix sort needs three or more.
constexpr int kRankMost = 8192;

__global__ void __launch_bounds__(kThreads)
rank_kernel(int T, int N, const void* ids, int wide, int* key_out, int* pos_out) {
  __shared__ int4 keys[kRankMost / 4];
  chain_grid();
  int* flat = reinterpret_cast<int*>(keys);
  const int vectors = (T + 3) / 4;
  for (int j = threadIdx.x; j < 4 * vectors; j += kThreads) flat[j] = j < T ? key_of(ids, wide, j, N) : 0x7fffffff;
  __syncthreads();
  const int t = blockIdx.x * (kThreads / 8) + (threadIdx.x >> 3), sub = threadIdx.x & 7;
  const int mine = flat[min(t, T - 1)], own = t / 4;
  int rank = 0;
  for (int v = sub; v < vectors; v += 8) {
    const int4 k = keys[v];
    const int below = v < own ? mine + 1 : mine;   // in front of the position equal keys count, behind it they do not
    rank += (k.x < below) + (k.y < below) + (k.z < below) + (k.w < below);
  }
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, d);
  if (t < T && sub == 0) {
    for (int j = own * 4; j < t; ++j) rank += flat[j] == mine;
    key_out[rank] = mine;
    pos_out[rank] = t;
  }
}

// Radix sort by digits of up to 10 bits, for more positions.  Block b of each pass has the positions [b * chunk, ...).
// Every block adds up the counts of all blocks itself, which costs blocks^2 * digits loads, so the blocks are few and
// large.  262,144 positions of as many rows: two passes of 17.4 us with digits of 10 bits, three of 13.2 with 9.
constexpr int kMaxDigitBits = 10;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;

// Counts of the first digit; the tables of the later ones, which the passes in front of them fill, are cleared.
__global__ void __launch_bounds__(kSortThreads)
digit_count_kernel(int64_t T, int N, const void* ids, int wide, int64_t chunk, int digits, int passes, int* tables) {
  __shared__ int count[1 << kMaxDigitBits];
  chain_grid();
  count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t end = min(T, (blockIdx.x + 1) * chunk);
  for (int64_t t = blockIdx.x * chunk + threadIdx.x; t < end; t += kSortThreads)
    atomicAdd(count + (key_of(ids, wide, t, N) & (digits - 1)), 1);
  __syncthreads();
  if (threadIdx.x < digits) {
    tables[blockIdx.x * digits + threadIdx.x] = count[threadIdx.x];
    for (int p = 1; p < passes; ++p) tables[((int64_t)p * gridDim.x + blockIdx.x) * digits + threadIdx.x] = 0;
  }
}

// One pass: positions to their places by one digit, in order within a digit.  keys_in is null in the first pass, which
// reads the ids.  next: the counts of the next digit by block of the new order, or null in the last pass.
__global__ void __launch_bounds__(kSortThreads)
digit_place_kernel(int64_t T, int N, const void* ids, int wide, const int* keys_in, const int* pos_in, int64_t chunk, int shift,
                   int bits, const int* table, int* next, int* keys_out, int* pos_out) {
  extern __shared__ int places[];      // [warp][digit]
  __shared__ int of_digit[1 << kMaxDigitBits], of_digit_before[1 << kMaxDigitBits];
  __shared__ int warp_sum[kSortWarps];
  chain_grid();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int digits = 1 << bits, mask = digits - 1;
  int* place = places + warp * digits;
  auto key_at = [&](int64_t t) { return keys_in ? keys_in[t] : key_of(ids, wide, t, N); };
  of_digit[threadIdx.x] = of_digit_before[threadIdx.x] = 0;
  for (int d = lane; d < digits; d += 32) place[d] = 0;
  __syncthreads();
  {   // of every digit: how many there are, and how many in the blocks in front of this one
    const int quads = digits / 4, quad = threadIdx.x & (quads - 1), group = threadIdx.x / quads, groups = kSortThreads / quads;
    int4 all = make_int4(0, 0, 0, 0), before = all;
#pragma unroll 8
    for (int b = group; b < gridDim.x; b += groups) {
      const int4 c = reinterpret_cast<const int4*>(table)[b * quads + quad];
      all.x += c.x, all.y += c.y, all.z += c.z, all.w += c.w;
      if (b < blockIdx.x) before.x += c.x, before.y += c.y, before.z += c.z, before.w += c.w;
    }
    int *to = of_digit + quad * 4, *to_before = of_digit_before + quad * 4;
    atomicAdd(to, all.x), atomicAdd(to + 1, all.y), atomicAdd(to + 2, all.z), atomicAdd(to + 3, all.w);
    atomicAdd(to_before, before.x), atomicAdd(to_before + 1, before.y), atomicAdd(to_before + 2, before.z), atomicAdd(to_before + 3, before.w);
  }
  const int64_t begin = blockIdx.x * chunk, end = min(T, begin + chunk);
  const int64_t sub = chunk / kSortWarps;
  const int64_t from = min(end, begin + warp * sub), to = min(end, from + sub);
  for (int64_t t = from + lane; t < to; t += 32) atomicAdd(place + (key_at(t) >> shift & mask), 1);
  __syncthreads();
  {   // places of every warp's digits
    const int d = threadIdx.x;
    const int all = d < digits ? of_digit[d] : 0;
    int sum = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    if (d < digits) {
      int at = sum - all + of_digit_before[d];
      for (int w = 0; w < warp; ++w) at += warp_sum[w];
      int n[kSortWarps];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) n[w] = places[w * digits + d];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        places[w * digits + d] = at;
        at += n[w];
      }
    }
  }
  __syncthreads();
  for (int64_t t0 = from; t0 < to; t0 += 32) {
    const int64_t t = t0 + lane;
    const bool have = t < to;
    const int key = have ? key_at(t) : 0;
    const int d = have ? key >> shift & mask : digits;
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const int before = __popc(same & ((1u << lane) - 1));
    int at = 0;
    if (have) at = place[d] + before;
    __syncwarp();
    if (have) {
      if (before == 0) place[d] = at + __popc(same);
      keys_out[at] = key;
      pos_out[at] = pos_in ? pos_in[t] : (int)t;
      if (next) atomicAdd(next + (int64_t)((unsigned)at / (unsigned)chunk) * digits + (key >> (shift + bits) & mask), 1);
    }
    __syncwarp();
  }
}

// ---- sums of sorted rows -------------------------------------------------------------------------------------------
//
// The work is the sorted positions (a row of dOut to read each) and the rows of the table (one to write each) in one
// sequence: the positions of row 0, the end of row 0, the positions of row 1, ...  Position j of the sorted order comes at
// place j + key[j], so a cut of the sequence into equal parts is found by a search, whatever the ids are: a table that is
// all but empty is cleared at the speed of its stores, and an id that half of the batch names is shared by as many groups
// of lanes as it has parts.  A group of W lanes takes one part of one slab of columns.  Rows that lie in several parts go to
// `split` in 32 bits ([part][0: end of a row that began earlier, 1: beginning of a row that ends later][column]) and are
// added up by the kernel behind, in the order of the parts.  Bound by memory: 262,144 positions of 262,144 x 2048 bf16 356 us,
// 6.0 TB/s; 16,384 of 131,072 x 1024 58 us, 5.2 TB/s.

// number of positions in the sequence's first `d` places
template <int W>
__device__ __forceinline__ int positions_before(const int* keys, int T, int64_t d) {
  const int lane = threadIdx.x & (W - 1);
  const unsigned mask = subwarp_mask<W>();
  const int shift = (threadIdx.x & 31) & ~(W - 1);
  int lo = 0, n = T;   // the answer lies in [lo, lo + n]
  while (n > 0) {
    const int step = n / (W + 1) + 1;   // probes at lo + step - 1, lo + 2 * step - 1, ...
    const int64_t j = (int64_t)lo + (int64_t)(lane + 1) * step - 1;
    const bool inside = j < (int64_t)lo + n && j + keys[j] < d;
    const int c = __popc(__ballot_sync(mask, inside) >> shift & (W == 32 ? 0xffffffffu : (1u << W) - 1));
    const int used = c * step;
    lo += used;
    n = min(n - used, step - 1);
  }
  return lo;
}

template <typename T, int BYTES, int R, int W>
__global__ void __launch_bounds__(kThreads)
sum_parts_kernel(int n, int N, int K, int64_t parts, int slabs, int length, const int* keys, const int* pos,
                 const T* __restrict__ dout, int64_t ld, float scale, T* __restrict__ dtable, int2* info, float* split) {
  typedef dense_vec<T, BYTES> vec;
  constexpr int E = vec::kCount;
  constexpr int U = R >= 4 ? 2 : 4;     // rows of dOut in flight
  chain_grid();
  const int lane = threadIdx.x & (W - 1);
  const unsigned mask = subwarp_mask<W>();
  const int64_t id = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / W;
  const int64_t part = id / slabs;
  const int slab = (int)(id - part * slabs);
  if (part >= parts) return;            // whole groups of lanes: nothing below reaches across them
  const int64_t d0 = part * length, d1 = d0 + length;
  int j = positions_before<W>(keys, n, d0);
  int row = (int)min(d0 - j, (int64_t)N);
  bool open = j > 0 && row < N && keys[j - 1] == row;     // the row began in an earlier part
  if (slab == 0 && lane == 0) info[part] = make_int2(row, open);
  int col[R];
#pragma unroll
  for (int r = 0; r < R; ++r) col[r] = (slab * R + r) * W * E + lane * E;
  float acc[R][E];
  auto clear = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[r][e] = 0.f;
  };
  auto to_split = [&](int which) {
    float* p = split + (2 * part + which) * K;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (col[r] < K) {
#pragma unroll
        for (int e = 0; e < E; ++e) p[col[r] + e] = acc[r][e];
      }
  };
  auto end_row = [&]() {
    if (open) {
      to_split(0);
      open = false;
    } else {
      T* p = dtable + (int64_t)row * K;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (col[r] < K) {
          vec v;
#pragma unroll
          for (int e = 0; e < E; ++e) v.at[e] = from_float<T>(scale * acc[r][e]);
          *reinterpret_cast<decltype(v.raw)*>(p + col[r]) = v.raw;
        }
    }
    clear();
    ++row;
  };
  clear();
  bool last_is_row = true;   // the part's last place is the end of a row
  while (true) {
    // up to W positions of this part
    const int64_t at = (int64_t)j + lane;
    int key = 0x7fffffff, p = 0;
    if (at < n) key = keys[at], p = pos[at];
    const bool mine = at < n && key < N && at + key < d1;
    const int have = __popc(__ballot_sync(mask, mine));    // the first ones: places ascend
    for (int i = 0; i < have; i += U) {
      vec v[U][R];
      int k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int l = min(i + u, have - 1);
        k[u] = __shfl_sync(mask, key, l, W);
        const T* src = dout + (int64_t)__shfl_sync(mask, p, l, W) * ld;
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (i + u < have && col[r] < K) v[u][r].raw = *reinterpret_cast<const decltype(v[u][r].raw)*>(src + col[r]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u < have) {
          while (row < k[u]) end_row();
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] += to_float(v[u][r].at[e]);
        }
      }
    }
    j += have;
    if (have) last_is_row = false;
    if (have < W) break;
  }
  const int last = (int)min(d1 - j, (int64_t)N);   // rows that end in front of the next part
  if (row < last) last_is_row = true;
  while (row < last) end_row();
  if (!last_is_row) to_split(1);
}

template <int E>
__device__ __forceinline__ void load_columns(const float* p, float (&v)[E]) {
  if (E == 4) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1 % E] = x.y, v[2 % E] = x.z, v[3 % E] = x.w;
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = p[i];
  }
}

// Rows that lie in several parts: a row that began earlier and ends in a part is the sum of the pieces before it and its own.
// A block has 16 parts and 512 columns, every gridDim.x-th part, since those with such rows lie together; those that end
// one are shared out among its warps, but for rows of many pieces, on which all of them work.  (With a block to 8 parts
// and 128 columns most of the time went into blocks without work: 81 us for 262,144 positions of 262,144 x 2048, now 17;
// with 32 neighbouring parts to a block a few blocks had all of it.)
constexpr int kJoinParts = 16;
constexpr int kJoinColumns = 512;
constexpr int kJoinMany = 32;

template <typename T, int E>   // E: columns that one load takes, 4 where all rows of `split` are aligned for it
__global__ void __launch_bounds__(kThreads)
join_parts_kernel(int N, int K, int64_t parts, const int2* info, const float* split, float scale, T* __restrict__ dtable) {
  constexpr int kWarps = kThreads / 32, kStep = 32 * E, kSteps = kJoinColumns / kStep;
  __shared__ int64_t first_of[kJoinParts];
  __shared__ int row_of[kJoinParts];
  __shared__ float sums[kWarps][kStep];
  chain_grid();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto part_of = [&](int i) { return (int64_t)i * gridDim.x + blockIdx.x; };
  {   // two parts to a warp
    const int i = warp * 2 + (lane >> 4), sub = lane & 15;
    const unsigned mask = 0xffffu << (lane & 16);
    const int64_t part = part_of(i);
    int row = -1;
    if (part < parts) {
      const int2 here = info[part];
      const int next = part + 1 < parts ? info[part + 1].x : N;
      if (here.y && here.x < N && next > here.x) row = here.x;
    }
    int64_t lo = 0, n = row >= 0 ? part : 0;   // first part that begins inside this row or at its first position: in [lo, lo + n]
    while (n > 0) {
      const int64_t step = n / 17 + 1, at = lo + (sub + 1) * step - 1;
      const bool before = at < lo + n && info[at].x < row;
      const int c = __popc(__ballot_sync(mask, before) & mask);
      lo += c * step;
      n = min(n - c * step, step - 1);
    }
    if (sub == 0) {
      row_of[i] = row;
      first_of[i] = row >= 0 && info[lo].y ? lo - 1 : lo;   // (open: its beginning is the part in front)
    }
  }
  __syncthreads();
  // pieces [b, e) in the E columns from `col` on
  auto add = [&](int64_t b, int64_t e, int col, float (&sum)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] = 0.f;
    if (col >= K) return;
    const float* p = split + (2 * b + 1) * K + col;
#pragma unroll 8
    for (int64_t s = b; s < e; ++s) {
      float v[E];
      load_columns<E>(p, v);
#pragma unroll
      for (int i = 0; i < E; ++i) sum[i] += v[i];
      p += 2 * (int64_t)K;
    }
  };
  auto load_own = [&](int i, int col, float (&own)[E]) {
    if (col < K) load_columns<E>(split + 2 * part_of(i) * K + col, own);
  };
  auto finish = [&](int i, int col, const float (&sum)[E], const float (&own)[E]) {
    if (col >= K) return;
    T* to = dtable + (int64_t)row_of[i] * K + col;
#pragma unroll
    for (int e = 0; e < E; ++e) to[e] = from_float<T>(scale * (sum[e] + own[e]));
  };
  const int col0 = blockIdx.y * kJoinColumns + lane * E;
  const int steps = min(kSteps, (K - (int)blockIdx.y * kJoinColumns + kStep - 1) / kStep);
  int turn = 0;
  for (int i = 0; i < kJoinParts; ++i) {
    if (row_of[i] < 0 || part_of(i) - first_of[i] > kJoinMany) continue;
    for (int c = 0; c < steps; ++c) {
      if (turn++ % kWarps != warp) continue;
      float sum[E], own[E];
      load_own(i, col0 + c * kStep, own);
      add(first_of[i], part_of(i), col0 + c * kStep, sum);
      finish(i, col0 + c * kStep, sum, own);
    }
  }
  for (int i = 0; i < kJoinParts; ++i) {
    const int64_t f = first_of[i], pieces = part_of(i) - f;
    if (row_of[i] < 0 || pieces <= kJoinMany) continue;
    for (int c = 0; c < steps; ++c) {
      float sum[E], own[E];
      load_own(i, col0 + c * kStep, own);
      add(f + pieces * warp / kWarps, f + pieces * (warp + 1) / kWarps, col0 + c * kStep, sum);
#pragma unroll
      for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = sum[e];
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 1; w < kWarps; ++w)
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] += sums[w][lane * E + e];
        finish(i, col0 + c * kStep, sum, own);
      }
      __syncthreads();
    }
  }
}

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// How a call of these sizes is cut up, and where its workspace lies.
struct backward_plan {
  int bits, passes;             // of the radix sort; passes = 0: the positions are ranked
  int64_t chunk;
  int blocks;
  int length;                   // places to a part
  int64_t parts;
  size_t keys, pos, tables, info, split, bytes;   // offsets
};

// Places to a part: 16 to 256, as many as leave 64 warps for every SM, two rounds of them, with slabs of 256 columns (16,384
// positions of 131,072 x 1024: 58 us, with 32 warps 65).  Longer parts mean fewer rows in several of them: 64 instead of 256
// cost 53 us instead of 17 in the join for 262,144 positions of 262,144 x 2048.  (Narrow rows, four groups of lanes to a
// warp, would sum faster in shorter parts, but their join takes more than that: 3 M positions, 16 columns 104 + 83 against
// 140 + 28 us.)
backward_plan plan_backward(int64_t T, int64_t N, int64_t K) {
  backward_plan p = {};
  while (p.bits < 31 && ((int64_t)1 << p.bits) <= N) ++p.bits;
  if (T > kRankMost) {
    p.passes = (p.bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.bits = std::max(5, (p.bits + p.passes - 1) / p.passes);
  }
  p.chunk = (T + 63) / 64;
  if (T > 1 << 20) p.chunk = (T + 147) / 148;
  p.chunk = std::max<int64_t>(1, (p.chunk + kSortThreads - 1) / kSortThreads) * kSortThreads;
  p.blocks = (int)((T + p.chunk - 1) / p.chunk);
  p.length = (int)std::min<int64_t>(256, std::max<int64_t>(16, ((T + N) * ((K + 255) / 256) / (148 * 64) + 15) / 16 * 16));
  p.parts = (T + N + p.length - 1) / p.length;
  const size_t b_t = align_up((size_t)T * 4, 256);
  p.keys = 0;
  p.pos = p.keys + b_t * (p.passes > 1 ? 2 : 1);
  p.tables = p.pos + b_t * (p.passes > 1 ? 2 : 1);
  p.info = p.tables + align_up((size_t)p.passes * p.blocks * ((size_t)4 << p.bits), 256);
  p.split = p.info + align_up((size_t)p.parts * sizeof(int2), 256);
  p.bytes = p.split + (size_t)p.parts * 2 * K * 4;
  return p;
}

// Sorts; *keys and *pos point to the result.
void launch_sort(hpspmm_ctx* ctx, const backward_plan& p, int64_t T, int64_t N, const void* ids, int wide, char* space,
                 const int** keys, const int** pos, cudaStream_t s) {
  const size_t b_t = align_up((size_t)T * 4, 256);
  int *k = (int*)(space + p.keys), *at = (int*)(space + p.pos);
  *keys = k, *pos = at;
  if (p.passes == 0) {
    hpspmm_launch(rank_kernel, dim3((unsigned)((T + kThreads / 8 - 1) / (kThreads / 8))), dim3(kThreads), 0, s, (int)T, (int)N, ids, wide,
                  k, at);
    ctx->launches++;
    return;
  }
  int* tables = (int*)(space + p.tables);
  const int digits = 1 << p.bits, smem = kSortWarps * digits * 4;
  cudaFuncSetAttribute(digit_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);   // (a refusal shows at the launch)
  hpspmm_launch(digit_count_kernel, dim3(p.blocks), dim3(kSortThreads), 0, s, T, (int)N, ids, wide, p.chunk, digits, p.passes, tables);
  ctx->launches++;
  for (int i = 0; i < p.passes; ++i) {
    // the last pass writes the first buffers
    int* to_k = (p.passes - 1 - i) % 2 ? (int*)((char*)k + b_t) : k;
    int* to_p = (p.passes - 1 - i) % 2 ? (int*)((char*)at + b_t) : at;
    const int* from_k = i == 0 ? nullptr : (to_k == k ? (int*)((char*)k + b_t) : k);
    const int* from_p = i == 0 ? nullptr : (to_p == at ? (int*)((char*)at + b_t) : at);
    const int64_t table = (int64_t)p.blocks * digits;
    hpspmm_launch(digit_place_kernel, dim3(p.blocks), dim3(kSortThreads), smem, s, T, (int)N, ids, wide, from_k, from_p, p.chunk, i * p.bits,
                  p.bits, tables + i * table, i + 1 < p.passes ? tables + (i + 1) * table : nullptr, to_k, to_p);
    ctx->launches++;
  }
}

template <typename T, int BYTES, int R, int W>
void launch_sums(hpspmm_ctx* ctx, const backward_plan& p, int64_t n, int64_t N, int64_t K, const int* keys, const int* pos,
                 const void* dout, int64_t ld, float scale, void* dtable, char* space, cudaStream_t s) {
  constexpr int kSlab = W * R * BYTES / (int)sizeof(T);
  const int64_t slabs = (K + kSlab - 1) / kSlab, lanes = p.parts * slabs * W;
  hpspmm_launch(sum_parts_kernel<T, BYTES, R, W>, dim3((unsigned)((lanes + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, (int)n, (int)N,
                (int)K, p.parts, (int)slabs, p.length, keys, pos, (const T*)dout, ld, scale, (T*)dtable, (int2*)(space + p.info),
                (float*)(space + p.split));
  const dim3 grid((unsigned)((p.parts + kJoinParts - 1) / kJoinParts), (unsigned)((K + kJoinColumns - 1) / kJoinColumns));
  const int2* info = (const int2*)(space + p.info);
  const float* split = (const float*)(space + p.split);
  if (K % 4 == 0)
    hpspmm_launch(join_parts_kernel<T, 4>, grid, dim3(kThreads), 0, s, (int)N, (int)K, p.parts, info, split, scale, (T*)dtable);
  else
    hpspmm_launch(join_parts_kernel<T, 1>, grid, dim3(kThreads), 0, s, (int)N, (int)K, p.parts, info, split, scale, (T*)dtable);
  ctx->launches += 2;
}

template <typename T>
void launch_sums_of(hpspmm_ctx* ctx, const backward_plan& p, int64_t n, int64_t N, int64_t K, const int* keys, const int* pos,
                    const void* dout, int64_t ld, float scale, void* dtable, char* space, cudaStream_t s) {
  const int bytes = dense_vector_bytes((uintptr_t)dout | (uintptr_t)dtable | (uintptr_t)(K * (int64_t)sizeof(T)) |
                                           (uintptr_t)(ld * (int64_t)sizeof(T)), (int)sizeof(T));
  // 8 lanes to a group for rows of up to 8 vectors; four vectors to a lane where they are short
  const bool narrow = K * (int64_t)sizeof(T) <= 8 * bytes;
#define HPSPMM_SUMS(B, R)                                                                               \
  (narrow ? launch_sums<T, B, 1, 8>(ctx, p, n, N, K, keys, pos, dout, ld, scale, dtable, space, s)     \
          : launch_sums<T, B, R, 32>(ctx, p, n, N, K, keys, pos, dout, ld, scale, dtable, space, s))
  if (bytes == 16)
    HPSPMM_SUMS(16, 1);
  else if (bytes == 8)
    HPSPMM_SUMS(8, 2);
  else if (bytes == 4 || sizeof(T) == 4)
    HPSPMM_SUMS(4, 4);
  else
    HPSPMM_SUMS(sizeof(T), 4);
#undef HPSPMM_SUMS
}

template <typename T, int BYTES>
void launch_lookup(int64_t T_, int64_t N, int64_t K, const void* ids, int wide, const void* table, int64_t ld, float scale, void* out,
                   cudaStream_t s) {
  const int per_row = (int)(K * (int64_t)sizeof(T) / BYTES);
  // rows of up to 32 (8) vectors: 8 (2) lanes with up to four each, so that as much is in flight as with wide rows
  const int W = per_row <= 8 ? 2 : (per_row <= 32 ? 8 : 32);
  const int64_t pieces = ((int64_t)per_row + 4 * W - 1) / (4 * W), groups = T_ * pieces;
  const dim3 grid((unsigned)((groups * W + kThreads - 1) / kThreads));
  if (W == 2)
    hpspmm_launch(lookup_kernel<T, BYTES, 2>, grid, dim3(kThreads), 0, s, groups, (int)pieces, per_row, (int)N, ids, wide, (const T*)table, ld,
                  scale, (T*)out);
  else if (W == 8)
    hpspmm_launch(lookup_kernel<T, BYTES, 8>, grid, dim3(kThreads), 0, s, groups, (int)pieces, per_row, (int)N, ids, wide, (const T*)table, ld,
                  scale, (T*)out);
  else
    hpspmm_launch(lookup_kernel<T, BYTES, 32>, grid, dim3(kThreads), 0, s, groups, (int)pieces, per_row, (int)N, ids, wide, (const T*)table,
                  ld, scale, (T*)out);
}

template <typename T>
void launch_lookup_of(int64_t T_, int64_t N, int64_t K, const void* ids, int wide, const void* table,
                      int64_t ld, float scale, void* out, cudaStream_t s) {
  const int bytes = dense_vector_bytes((uintptr_t)table | (uintptr_t)out | (uintptr_t)(K * (int64_t)sizeof(T)) |
                                           (uintptr_t)(ld * (int64_t)sizeof(T)), (int)sizeof(T));
  if (bytes == 16)
    launch_lookup<T, 16>(T_, N, K, ids, wide, table, ld, scale, out, s);
  else if (bytes == 8)
    launch_lookup<T, 8>(T_, N, K, ids, wide, table, ld, scale, out, s);
  else if (bytes == 4 || sizeof(T) == 4)
    launch_lookup<T, 4>(T_, N, K, ids, wide, table, ld, scale, out, s);
  else
    launch_lookup<T, sizeof(T)>(T_, N, K, ids, wide, table, ld, scale, out, s);
}

int check_embedding(hpspmm_ctx* ctx, int64_t T, int64_t N, int64_t K, int32_t type, int32_t id_bytes, int64_t ld) {
  HPSPMM_REQUIRE(ctx, ctx != nullptr, "null context");
  HPSPMM_REQUIRE(ctx, T >= 0 && N >= 0 && K >= 0, "negative size");
  HPSPMM_REQUIRE(ctx, hpspmm::dense_type_size(type) != 0, "unknown element type");
  HPSPMM_REQUIRE(ctx, id_bytes == 4 || id_bytes == 8, "ids must have 4 or 8 bytes");
  HPSPMM_REQUIRE(ctx, ld >= 0, "negative row stride");
  if (T > 2147483646ll || N > 2147483646ll || K > 2147483646ll)
    return hpspmm_unsupported(ctx, "more than 2^31 - 2 positions, rows or columns");
  return hpspmm_report_timeout(ctx);
}

}  // namespace

extern "C" {

int hpspmm_embedding_forward(hpspmm_ctx* ctx, int64_t T, int64_t N, int64_t K, int32_t type, const void* ids,
                             int32_t id_bytes, const void* table, int64_t ld_table, float scale, void* out,
                             hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_embedding_forward");
  const int st = check_embedding(ctx, T, N, K, type, id_bytes, ld_table);
  if (st != HPSPMM_OK) return st;
  HPSPMM_REQUIRE(ctx, ld_table >= K, "row stride below the number of columns");
  if (T == 0 || K == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, ids && out && (table || N == 0), "null pointer");
  const int size = dense_type_size(type);
  HPSPMM_REQUIRE(ctx, may_begin(ids, id_bytes) && may_begin(table, size) && may_begin(out, size),
                 "an array does not begin on a multiple of its elements' size");
  // a group of lanes moves at least four elements of each of its lanes, or a row of up to 32 vectors
  if (T > ((int64_t)1 << 33) / ((K + 127) / 128)) return hpspmm_unsupported(ctx, "more than 2^31 - 1 blocks");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  if (type == HPSPMM_TYPE_F32)
    launch_lookup_of<float>(T, N, K, ids, id_bytes == 8, table, ld_table, scale, out, s);
  else if (type == HPSPMM_TYPE_F16)
    launch_lookup_of<__half>(T, N, K, ids, id_bytes == 8, table, ld_table, scale, out, s);
  else
    launch_lookup_of<__nv_bfloat16>(T, N, K, ids, id_bytes == 8, table, ld_table, scale, out, s);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

int64_t hpspmm_embedding_backward_workspace(int64_t T, int64_t N, int64_t K) {
  if (T < 0 || N < 0 || K < 0 || T > 2147483646ll || N > 2147483646ll || K > 2147483646ll) return -1;
  return (int64_t)plan_backward(T, N, K).bytes;
}

int hpspmm_embedding_backward(hpspmm_ctx* ctx, int64_t T, int64_t N, int64_t K, int32_t type, const void* ids,
                              int32_t id_bytes, const void* dOut, int64_t ld_dout, float scale, void* dTable,
                              void* workspace, size_t workspace_bytes, hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_embedding_backward");
  const int st = check_embedding(ctx, T, N, K, type, id_bytes, ld_dout);
  if (st != HPSPMM_OK) return st;
  if (N == 0 || K == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, dTable && (T == 0 || (ids && dOut && workspace)), "null pointer");
  const int size = dense_type_size(type);
  HPSPMM_REQUIRE(ctx, may_begin(dTable, size) && (T == 0 || (may_begin(ids, id_bytes) && may_begin(dOut, size))),
                 "an array does not begin on a multiple of its elements' size");
  const backward_plan p = plan_backward(T, N, K);
  HPSPMM_REQUIRE(ctx, T == 0 || workspace_bytes >= p.bytes, "workspace too small");
  HPSPMM_REQUIRE(ctx, T == 0 || ((uintptr_t)workspace & 255) == 0, "workspace not aligned to 256 bytes");
  if (p.parts * ((K + 31) / 32) > (int64_t)2147483647 * 8 || K > (int64_t)65535 * kJoinColumns)
    return hpspmm_unsupported(ctx, "more than 2^31 - 1 blocks, or 33,553,920 columns");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  if (T == 0) {
    HPSPMM_CUDA_TRY(ctx, cudaMemsetAsync(dTable, 0, (size_t)(N * K) * hpspmm::dense_type_size(type), s));
    return HPSPMM_OK;
  }
  char* space = (char*)workspace;
  const int *keys, *pos;
  launch_sort(ctx, p, T, N, ids, id_bytes == 8, space, &keys, &pos, s);
  if (type == HPSPMM_TYPE_F32)
    launch_sums_of<float>(ctx, p, T, N, K, keys, pos, dOut, ld_dout, scale, dTable, space, s);
  else if (type == HPSPMM_TYPE_F16)
    launch_sums_of<__half>(ctx, p, T, N, K, keys, pos, dOut, ld_dout, scale, dTable, space, s);
  else
    launch_sums_of<__nv_bfloat16>(ctx, p, T, N, K, keys, pos, dOut, ld_dout, scale, dTable, space, s);
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

}  // extern "C"
