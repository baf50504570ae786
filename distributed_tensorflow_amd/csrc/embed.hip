// Table lookup by token, its gradient, and the sparse row update (an embedding in front of a dense stack).
//
//   lookup    out[t][:]   = scale * table[ids[t]][:]
//   gradient  grad[v][:]  = scale * sum over t with ids[t] = v of g[t][:]           (every row of the table is written)
//   update    table[v][:] -= lr * scale * sum over t with ids[t] = v of g[t][:]     (only rows that occur are touched)
//
// An id outside [0, rows) is padding: a row of zeros, no gradient.  Storage fp32, bf16 or fp16; sums in fp32, rounded once.
//
// All three are bound by memory.  The gradient must not depend on the order in which atomics land, and a frequent token
// must not serialise on its row.
//
// Few tokens and elements, where launches and trips to memory count (see few()): one launch, a block per token.  The block of an id's FIRST
// occurrence finds the others by comparing (T^2 / 64 wave steps in all), each wave in a range of tokens of its own, and the
// waves' sums meet in order; the other blocks end at once.  (3001 tokens x 101, the whole pass: sorting by one workgroup, summing and
// joining took 23.6 us, this takes 13.3.)
//
// More tokens are SORTED by id (stable, least significant digit first) and equal ids are summed as runs of the sorted order, in
// ascending t:
//
//   sort      digits of up to 10 bits (a vocabulary of 2^20 - 1 takes two), two launches per digit: counts of every block, then
//             the scatter, each block of which adds up the counts in front of it by itself (at most 64 blocks).  Ranks inside a
//             wave come from ballots over the digit's bits.  (One launch whose blocks each count all the items: 24 us a digit
//             instead of 12 at 32768 tokens.)
//   sums      a group of lanes owns a chunk of consecutive sorted positions and a slice of columns, walks the chunk with
//             the loads of four positions in flight, and stores each run that lies inside the chunk.  The pieces of a run
//             that crosses chunks go to an fp32 workspace row of their chunk.  Zeros of the rows that do not occur: see Clear;
//             of a large table's other rows further blocks of the sums' launch look up (binary search in the sorted ids) which
//             do not occur and store those.
//   joins     a wave per run that crosses chunks and slice of columns adds its pieces in order; all eight waves of a block
//             share a run of more than 32 pieces (a frequent token).  The chunk borders depend on the sizes alone: the result
//             is the same bits every time.
#include "dtf_api.h"
#include "dtf_types.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kSmall = 4096;        // tokens compared with each other instead of sorted, at most (see few())
constexpr int kSmallWaves = 8;
constexpr int kSortThreads = 1024;
constexpr int kWaves = kSortThreads / 64;
constexpr int kMaxDigit = 10;       // bits
constexpr int kMaxSortBlocks = 64;
constexpr int kThreads = 256;
constexpr int64_t kCaches = (int64_t)256 << 20;     // bytes: a result of more does not stay in the last cache anyway
constexpr int kFillRows = 32;       // rows of the table per zero-filling block
constexpr int kJoinWaves = 8;       // (32768 tokens x 256: 16 waves 12.0 us, 8 waves 8.0, 4 waves 9.7)
constexpr int kLongRun = 32;        // pieces

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t t) {
  return wide ? static_cast<const int64_t*>(ids)[t] : (int64_t) static_cast<const int32_t*>(ids)[t];
}
// Sort key: the row, or `rows` (behind every row) for padding.
__device__ __forceinline__ uint32_t load_key(const void* ids, int wide, int64_t t, uint32_t rows) {
  const int64_t id = load_id(ids, wide, t);
  return (id >= 0 && id < (int64_t)rows) ? (uint32_t)id : rows;
}

// A pack to memory, past the caches if `past`: results larger than they are.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T, int N>
__device__ __forceinline__ void put(T* at, const Pack<T, N>& p, bool past) {
  if constexpr (sizeof(T) * N == 16) {
    if (past) {
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4, p), reinterpret_cast<u32x4*>(at));
      return;
    }
  }
  *reinterpret_cast<Pack<T, N>*>(at) = p;
}

// The other way: a pack that is read once.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> get(const T* at, bool past) {
  if constexpr (sizeof(T) * N == 16) {
    if (past) return __builtin_bit_cast(Pack<T, N>, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at)));
  }
  return *reinterpret_cast<const Pack<T, N>*>(at);
}

// --- lookup ------------------------------------------------------------------------------------------------------------
// 1 << lanes_log2 lanes per row, as many rows per block as fit, U tokens at a time (their rows requested together); the grid
// strides over the tokens.
template <typename T, int N, int U>
__global__ __launch_bounds__(kThreads) void lookup_kernel(const T* __restrict__ table, int64_t ld, int64_t rows,
                                                          const void* __restrict__ ids, int wide, int64_t tokens, int packs,
                                                          int lanes_log2, float scale, T* __restrict__ out, int64_t ldo, bool past) {
  const int group = threadIdx.x >> lanes_log2, groups = kThreads >> lanes_log2;
  const int lane = threadIdx.x & ((1 << lanes_log2) - 1);
  for (int64_t t0 = ((int64_t)blockIdx.x * groups + group) * U; t0 < tokens; t0 += (int64_t)gridDim.x * groups * U) {
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = load_id(ids, wide, min(t0 + u, tokens - 1));
    for (int c = lane; c < packs; c += 1 << lanes_log2) {
      Pack<T, N> p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {       // (padding reads row 0 and forgets it)
        const bool inside = id[u] >= 0 && id[u] < rows;
        p[u] = *reinterpret_cast<const Pack<T, N>*>(table + (inside ? id[u] : 0) * ld + (int64_t)c * N);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool inside = id[u] >= 0 && id[u] < rows;
#pragma unroll
        for (int e = 0; e < N; ++e) p[u].v[e] = inside ? (T)(scale * (float)p[u].v[e]) : (T)0.0f;
        if (t0 + u < tokens) put(out + (t0 + u) * ldo + (int64_t)c * N, p[u], past);
      }
    }
  }
}

// --- sort --------------------------------------------------------------------------------------------------------------
// Lanes of the wave with the same digit as this one (among `valid` lanes).
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool valid) {
  uint64_t mask = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1u);
    mask &= ((digit >> b) & 1u) ? set : ~set;
  }
  return mask;
}

// Stable places of one batch of kSortThreads items.  `base[d]` is where the next item with digit d goes; it is advanced.
// `wave_at[w][d]` is zero on entry and on exit: only the entries of digits that wave w has are set, and its leaders clear them
// again after its lanes have read them (LDS accesses of a wave stay in order).  Every thread of the block calls it.
__device__ __forceinline__ uint32_t place(uint32_t digit, int bits, bool valid, uint32_t* base, uint32_t* wave_at) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << bits;
  const uint64_t mask = same_digit(digit, bits, valid);
  const uint32_t rank = __popcll(mask & ((1ull << lane) - 1));
  const bool leader = valid && rank == 0;
  volatile uint32_t* mine = wave_at + wave * digits + digit;
  if (leader) *mine = __popcll(mask);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) {
    uint32_t n[kWaves], at = base[d];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) n[w] = wave_at[w * digits + d];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (n[w]) wave_at[w * digits + d] = at;
      at += n[w];
    }
    base[d] = at;
  }
  __syncthreads();
  const uint32_t to = valid ? *mine + rank : 0;
  if (leader) *mine = 0;
  return to;
}

// Exclusive prefix sum over `digits` (<= 1024) totals, one per thread; every thread of the block calls it.
__device__ __forceinline__ uint32_t digit_prefix(uint32_t v, uint32_t* wave_sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t inc = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t up = __shfl_up(inc, s);
    if (lane >= s) inc += up;
  }
  if (lane == 63) wave_sum[wave] = inc;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += wave_sum[w];
  __syncthreads();
  return before + inc - v;
}

struct SortPass {
  const void* ids;         // first pass: the ids themselves
  const uint2* in;         // later passes: {key, position}
  int wide;
  uint32_t rows;
  int64_t tokens, tile;    // items per block, a multiple of kSortThreads
  int shift, bits;
  int blocks;              // of the sort; the blocks behind them clear rows
  char* clear;             // first row that this launch clears, rows of whole 16-byte packs
  int64_t clear_rows, clear_ld;
  int clear_packs;
  bool past;
};

// Rows of the gradient to zero, by the blocks of a sort's launch behind the sort's own.
__device__ __forceinline__ void clear_rows(const SortPass& a) {
  const uint32_t total = (uint32_t)(a.clear_rows * a.clear_packs), step = (gridDim.x - a.blocks) * kSortThreads;      // (kClearBytes)
  const Pack<float, 4> zero{};
  for (uint32_t i = (blockIdx.x - a.blocks) * kSortThreads + threadIdx.x; i < total; i += step) {
    const uint32_t row = i / (uint32_t)a.clear_packs;
    put(reinterpret_cast<float*>(a.clear + row * a.clear_ld + (i - row * a.clear_packs) * 16), zero, a.past);
  }
}

__device__ __forceinline__ uint2 sort_item(const SortPass& a, int64_t i) {
  return a.in ? a.in[i] : make_uint2(load_key(a.ids, a.wide, i, a.rows), (uint32_t)i);
}

// counts[block][digit]
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortPass a, uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[1 << kMaxDigit];
  if ((int)blockIdx.x >= a.blocks) return clear_rows(a);
  const int digits = 1 << a.bits, lane = threadIdx.x & 63;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * a.tile, last = min(first + a.tile, a.tokens);
  for (int64_t i0 = first; i0 < last; i0 += kSortThreads) {
    const int64_t i = i0 + threadIdx.x;
    const bool valid = i < last;
    const uint32_t digit = valid ? (sort_item(a, i).x >> a.shift) & (digits - 1) : 0;
    // one LDS atomic per distinct digit of the wave: a frequent token would make its lanes queue on one counter
    const uint64_t mask = same_digit(digit, a.bits, valid);
    if (valid && (mask & ((1ull << lane) - 1)) == 0) atomicAdd(&hist[digit], (uint32_t)__popcll(mask));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) counts[(int64_t)blockIdx.x * digits + d] = hist[d];
}

// `pairs` (not the last pass) or `keys` and `order` (the last pass) receive the items in order of this digit.
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortPass a, const uint32_t* __restrict__ counts,
                                                                    uint2* __restrict__ pairs, uint32_t* __restrict__ keys,
                                                                    uint32_t* __restrict__ order) {
  __shared__ uint32_t wave_at[kWaves << kMaxDigit];
  __shared__ uint32_t base[1 << kMaxDigit], wave_sum[kWaves];
  if ((int)blockIdx.x >= a.blocks) return clear_rows(a);
  const int blocks = a.blocks;
  const int digits = 1 << a.bits;
  const int64_t first = (int64_t)blockIdx.x * a.tile, last = min(first + a.tile, a.tokens);
  uint32_t total = 0, before = 0;
  if (threadIdx.x < digits) {
    for (int b0 = 0; b0 < blocks; b0 += 32) {
      uint32_t n[32];                     // (requested together; past the end the last block's again)
#pragma unroll
      for (int k = 0; k < 32; ++k) n[k] = counts[(int64_t)min(b0 + k, blocks - 1) * digits + threadIdx.x];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        total += b0 + k < blocks ? n[k] : 0;
        before += b0 + k < (int)blockIdx.x ? n[k] : 0;
      }
    }
  }
  for (int i = threadIdx.x; i < kWaves * digits; i += kSortThreads) wave_at[i] = 0;
  const uint32_t at = digit_prefix(total, wave_sum);
  if (threadIdx.x < digits) base[threadIdx.x] = at + before;
  __syncthreads();
  for (int64_t i0 = first; i0 < last; i0 += kSortThreads) {
    const int64_t i = i0 + threadIdx.x;
    const bool valid = i < last;
    const uint2 it = valid ? sort_item(a, i) : make_uint2(0, 0);
    const uint32_t to = place((it.x >> a.shift) & (digits - 1), a.bits, valid, base, wave_at);
    if (valid) {
      if (pairs) {
        pairs[to] = it;
      } else {
        keys[to] = it.x;
        order[to] = it.y;
      }
    }
  }
}

// --- sums --------------------------------------------------------------------------------------------------------------
struct SumArgs {
  const uint32_t* keys;      // sorted
  const uint32_t* order;     // token of every sorted position
  int64_t tokens;
  uint32_t rows;
  int chunk;                 // sorted positions per chunk
  int64_t chunks;
  int dim, packs, lanes_log2;
  int64_t ldg, ldt;          // row strides of g and of the table / gradient, in elements
  float scale;
  const float* lr;           // row update: device learning rate
  float* pieces;             // [chunks][2][piece_ld]: the run that began before the chunk, the run that goes on behind it
  int64_t piece_ld;
  int64_t sum_blocks;        // blocks past these write the zeros of rows that do not occur
  bool past, g_past;         // the gradient (the upstream gradient) is larger than the caches: 131072 x 4096 860 -> 811 us
  int join_chunks;           // chunks whose crossing runs one block joins (at most 64: one lane looks at each)
};

template <typename T, int N, bool UPDATE>
__device__ __forceinline__ void store_row(const SumArgs& a, T* table, uint32_t row, int pack, const float (&acc)[N], float f) {
  Pack<T, N>* at = reinterpret_cast<Pack<T, N>*>(table + (int64_t)row * a.ldt + (int64_t)pack * N);
  Pack<T, N> p;
  if (UPDATE) {
    p = *at;
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = (T)((float)p.v[e] - f * acc[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = (T)(f * acc[e]);
  }
  put(reinterpret_cast<T*>(at), p, !UPDATE && a.past);
}

template <typename T, int N, bool UPDATE>
__global__ __launch_bounds__(kThreads) void sum_kernel(SumArgs a, const T* __restrict__ g, T* __restrict__ table) {
  const int lanes = 1 << a.lanes_log2, groups = kThreads >> a.lanes_log2;
  const int group = threadIdx.x >> a.lanes_log2;
  const int pack = blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
  const bool in_row = pack < a.packs;
  if ((int64_t)blockIdx.x >= a.sum_blocks) {
    // Rows that do not occur: which of kFillRows rows are missing from the sorted ids, then their zeros.
    __shared__ int missing[kFillRows];
    const int64_t row0 = ((int64_t)blockIdx.x - a.sum_blocks) * kFillRows;
    if (threadIdx.x < kFillRows) {
      const int64_t row = row0 + threadIdx.x;
      int64_t low = 0, high = a.tokens;                    // first position whose key is >= row
      while (low < high) {
        const int64_t mid = (low + high) >> 1;
        if ((int64_t)a.keys[mid] < row) low = mid + 1; else high = mid;
      }
      missing[threadIdx.x] = row < (int64_t)a.rows && !(low < a.tokens && (int64_t)a.keys[low] == row);
    }
    __syncthreads();
    Pack<T, N> zero;
#pragma unroll
    for (int e = 0; e < N; ++e) zero.v[e] = (T)0.0f;
    for (int r = group; r < kFillRows; r += groups)
      if (missing[r] && in_row) put(table + (row0 + r) * a.ldt + (int64_t)pack * N, zero, a.past);
    return;
  }
  const int64_t chunk = (int64_t)blockIdx.x * groups + group;
  if (chunk >= a.chunks || !in_row) return;
  const float f = UPDATE ? a.lr[0] * a.scale : a.scale;
  const int64_t first = chunk * a.chunk, last = min(first + a.chunk, a.tokens);
  const T* column = g + (int64_t)pack * N;
  uint32_t run = a.keys[first];
  bool from_before = first > 0 && a.keys[first - 1] == run;
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  Pack<float, N>* piece = reinterpret_cast<Pack<float, N>*>(a.pieces + chunk * 2 * a.piece_ld + (int64_t)pack * N);
  Pack<float, N> sum;
  constexpr int kAhead = 4;        // (8: 889 us instead of 862 at 131072 x 4096)
  for (int64_t i0 = first; i0 < last && run < a.rows; i0 += kAhead) {
    uint32_t key[kAhead];
    Pack<T, N> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) key[j] = i0 + j < last ? a.keys[i0 + j] : a.rows;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (key[j] < a.rows) v[j] = get<T, N>(column + (int64_t)a.order[i0 + j] * a.ldg, a.g_past);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j >= last) break;
      if (key[j] != run) {
        if (from_before) {
#pragma unroll
          for (int e = 0; e < N; ++e) sum.v[e] = acc[e];
          *piece = sum;
        } else {
          store_row<T, N, UPDATE>(a, table, run, pack, acc, f);
        }
        from_before = false;
        run = key[j];
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.f;
      }
      if (run < a.rows) {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += (float)v[j].v[e];
      }
    }
  }
  if (run >= a.rows) return;                               // padding sits behind every row
  const bool goes_on = last < a.tokens && a.keys[last] == run;
  if (from_before || goes_on) {
#pragma unroll
    for (int e = 0; e < N; ++e) sum.v[e] = acc[e];
    *(from_before ? piece : reinterpret_cast<Pack<float, N>*>(reinterpret_cast<float*>(piece) + a.piece_ld)) = sum;
  } else {
    store_row<T, N, UPDATE>(a, table, run, pack, acc, f);
  }
}

// How many chunks from `c0` on begin with `run`.  They are the first ones or none (the ids are sorted): 64 places at a time, then
// 64 places between the last that does and the first that does not.
__device__ __forceinline__ int64_t run_of_chunks(const SumArgs& a, int64_t c0, uint32_t run, int lane) {
  int64_t low = c0, n = a.chunks - c0;         // chunks c0 .. low - 1 do, chunks from low + n on do not
  while (n > 0) {
    const int64_t step = (n + 63) / 64, c = low + lane * step;
    const int hits = __popcll(__ballot(c < low + n && a.keys[min(c, a.chunks - 1) * a.chunk] == run));
    if (hits == 0) break;
    const int64_t end = low + n;
    low += (hits - 1) * step + 1;
    n = min(step - 1, end - low);
  }
  return low - c0;
}

// Runs that cross chunks: the chunk a run begins in names it; its pieces are that chunk's second workspace row and the
// first rows of the chunks behind it.
template <typename T, int N, bool UPDATE>
__global__ __launch_bounds__(kJoinWaves * 64) void join_kernel(SumArgs a, T* __restrict__ table) {
  __shared__ f32x4 part[kJoinWaves][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = (blockIdx.y * 64 + lane) * 4;
  const float f = UPDATE ? a.lr[0] * a.scale : a.scale;
  // lane l looks at chunk chunk0 + l: its first key, and whether its last run is one that begins in it and goes on behind it
  const int64_t chunk0 = (int64_t)blockIdx.x * a.join_chunks, mine = min(chunk0 + lane, a.chunks - 1);
  const int64_t first = mine * a.chunk, last = min(first + a.chunk, a.tokens);
  const uint32_t first_key = a.keys[first], last_key = a.keys[last - 1];
  const uint32_t before = a.keys[max(first - 1, (int64_t)0)], behind = a.keys[min(last, a.tokens - 1)];
  const bool begins = lane < a.join_chunks && chunk0 + lane < a.chunks && last < a.tokens && last_key < a.rows && behind == last_key &&
                      !(first_key == last_key && first > 0 && before == last_key);
  uint64_t todo = __ballot(begins);
  auto add = [&](int64_t chunk, int64_t pieces, int64_t p, int step) {       // pieces p, p + step, ...; piece 0 in the run's own chunk
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (col >= a.dim) return sum;
    const float* src = a.pieces + chunk * 2 * a.piece_ld + col;
    for (; p <= pieces; p += 8 * step) {
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t q = min(p + k * step, pieces);
        v[k] = *reinterpret_cast<const f32x4*>(src + (q ? q * 2 : 1) * a.piece_ld);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (p + k * step <= pieces) sum += v[k];
    }
    return sum;
  };
  auto store = [&](uint32_t run, f32x4 sum) {
    T* row = table + (int64_t)run * a.ldt + col;
    if (N >= 4) {                            // whole, aligned quads
      if (col >= a.dim) return;
      Pack<T, 4> q;
      if (UPDATE) q = *reinterpret_cast<const Pack<T, 4>*>(row);
#pragma unroll
      for (int e = 0; e < 4; ++e) q.v[e] = UPDATE ? (T)((float)q.v[e] - f * sum[e]) : (T)(f * sum[e]);
      *reinterpret_cast<Pack<T, 4>*>(row) = q;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < a.dim) row[e] = UPDATE ? (T)((float)row[e] - f * sum[e]) : (T)(f * sum[e]);
  };
  for (int turn = 0; todo; ++turn, todo &= todo - 1) {
    const int l = __builtin_ctzll(todo);
    const uint32_t run = __shfl(last_key, l);
    const int64_t chunk = chunk0 + l;
    // the chunks behind this one that begin with the run; the ids are sorted, so the first that does not ends the count
    uint64_t same = __ballot(chunk0 + lane < a.chunks && first_key == run) >> (l + 1 < 64 ? l + 1 : 63);
    if (l == 63) same = 0;
    int64_t pieces = same == ~0ull ? 64 : __builtin_ctzll(~same);
    if (chunk + pieces + 1 == chunk0 + 64) pieces += run_of_chunks(a, chunk0 + 64, run, lane);       // past the chunks the lanes look at
    if (pieces <= kLongRun) {
      if (turn % kJoinWaves == wave) store(run, add(chunk, pieces, 0, 1));
      continue;
    }
    part[wave][lane] = add(chunk, pieces, wave, kJoinWaves);
    __syncthreads();
    if (wave == 0) {
      f32x4 sum = part[0][lane];
#pragma unroll
      for (int w = 1; w < kJoinWaves; ++w) sum += part[w][lane];
      store(run, sum);
    }
    __syncthreads();
  }
}

// --- few tokens ----------------------------------------------------------------------------------------------------------
// Block (t, s): slice s of the columns of the row ids[t], if t is its first occurrence.
constexpr int kSmallLoops = 4;      // packs of a lane
template <typename T, int N, bool UPDATE>
__global__ __launch_bounds__(kSmallWaves * 64) void few_kernel(SumArgs a, const void* __restrict__ ids, int wide,
                                                               const T* __restrict__ g, T* __restrict__ table) {
  __shared__ int earlier, others;
  __shared__ uint16_t list[kSmallWaves][kSmall / kSmallWaves];
  __shared__ float part[kSmallWaves][64 * N];
  const int t = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, tokens = (int)a.tokens;
  const int64_t id = load_id(ids, wide, t);
  if (id < 0 || id >= (int64_t)a.rows) return;
  if (threadIdx.x == 0) earlier = others = 0;
  __syncthreads();
  for (int j0 = 0; j0 < t; j0 += kSmallWaves * 64) {
    const int j = j0 + threadIdx.x;
    if (__ballot(j < t && load_id(ids, wide, min(j, t)) == id)) {
      if (lane == 0) earlier = 1;
      break;
    }
  }
  // this wave's range of the tokens from t on, and where the id occurs in it
  const int range = (tokens - t + kSmallWaves - 1) / kSmallWaves, from = t + wave * range, to = min(from + range, tokens);
  int count = 0;
  for (int j0 = from; j0 < to; j0 += 64) {
    const int j = j0 + lane;
    const bool hit = j < to && load_id(ids, wide, min(j, tokens - 1)) == id;
    const uint64_t mask = __ballot(hit);
    if (hit) list[wave][count + __popcll(mask & ((1ull << lane) - 1))] = (uint16_t)j;
    count += __popcll(mask);
  }
  if (wave > 0 && count > 0 && lane == 0) others = 1;
  __syncthreads();
  if (earlier) return;
  const bool alone = !others;              // the first wave has all of them
  if (alone && wave > 0) return;
  const float f = UPDATE ? a.lr[0] * a.scale : a.scale;
#pragma unroll 1
  for (int k = 0; k < kSmallLoops; ++k) {
    const int pack = (blockIdx.y * kSmallLoops + k) * 64 + lane;
    if ((blockIdx.y * kSmallLoops + k) * 64 >= a.packs) break;
    const T* column = g + (int64_t)min(pack, a.packs - 1) * N;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    for (int p = 0; p < count; p += 8) {
      Pack<T, N> v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const Pack<T, N>*>(column + (int64_t)list[wave][min(p + q, count - 1)] * a.ldg);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (p + q < count) {
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] += (float)v[q].v[e];
        }
    }
    if (!alone) {
#pragma unroll
      for (int e = 0; e < N; ++e) part[wave][e * 64 + lane] = acc[e];
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int w = 1; w < kSmallWaves; ++w)
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] += part[w][e * 64 + lane];
      }
      __syncthreads();
    }
    if (wave == 0 && pack < a.packs) store_row<T, N, UPDATE>(a, table, (uint32_t)id, pack, acc, f);
  }
}

// Zeros in front of few_kernel.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void zero_rows_kernel(T* __restrict__ table, int64_t rows, int packs, int64_t ldt, int lanes_log2,
                                                             bool past) {
  const int groups = kThreads >> lanes_log2, lane = threadIdx.x & ((1 << lanes_log2) - 1);
  Pack<T, N> zero;
#pragma unroll
  for (int e = 0; e < N; ++e) zero.v[e] = (T)0.0f;
  for (int64_t r = (int64_t)blockIdx.x * groups + (threadIdx.x >> lanes_log2); r < rows; r += (int64_t)gridDim.x * groups)
    for (int c = lane; c < packs; c += 1 << lanes_log2) put(table + r * ldt + (int64_t)c * N, zero, past);
}

inline int log2_lanes(int packs) {
  int l = 0;
  while ((1 << l) < packs && (1 << l) < kThreads) ++l;
  return l;
}

// Sorted positions per chunk: enough chunks for 256 CUs x 1024 threads, at least 4 and at most 64 positions.
inline int chunk_of(int64_t tokens, int64_t lanes) {
  const int64_t c = tokens * lanes / (256 * 1024);
  return c < 4 ? 4 : c > 64 ? 64 : (int)c;
}

// Whether tokens are compared with each other (one launch, 13 us while little is moved) or sorted (20 to 25 us, and the rows of a
// frequent token are shared out).  Measured with ids as words occur, row update, fp32: 4096 x 512 of 2000 rows 16 us against 27, 1000 x
// 2048 of 250 rows 13 against 20, 300 x 8192 13 against 24; but 2000 x 2048 of 30 rows 29 against 20, 4096 x 2048 of 2000 rows
// 42 against 36, 4096 x 8192 155 against 60; of four rows 2000 x 512 19 against 20, 4096 x 512 46 against 25.
inline bool few(int64_t tokens, int64_t packs, int64_t rows) {
  return tokens <= kSmall && tokens * packs <= (rows < 16 ? 1 << 18 : 3 << 18);
}
inline bool surely_few(int64_t tokens, int64_t dim) { return few(tokens, dim, 1); }      // whatever the alignment and the rows

struct Workspace {
  int64_t keys, order, pairs, counts, pieces, total;    // byte offsets
  int64_t chunks, piece_ld;
  int chunk;
};

// The chunk length goes by the element count of a row and not by the access width: the workspace does not depend on
// alignment.
Workspace plan(int64_t tokens, int dim) {
  Workspace w;
  auto up = [](int64_t n) { return (n + 255) & ~(int64_t)255; };
  w.chunk = chunk_of(tokens, (dim + 3) / 4);
  w.chunks = (tokens + w.chunk - 1) / w.chunk;
  w.piece_ld = (dim + 7) / 8 * 8;
  const int64_t big = surely_few(tokens, dim) ? 0 : 1;         // (these need no workspace)
  w.keys = 0;
  w.order = up(w.keys + big * 4 * tokens);
  w.pairs = up(w.order + big * 4 * tokens);
  w.counts = up(w.pairs + big * 16 * tokens);
  w.pieces = up(w.counts + big * 4 * kMaxSortBlocks * (1 << kMaxDigit));
  w.total = up(w.pieces + big * w.chunks * 2 * w.piece_ld * 4) + 256;
  return w;
}

// The gradient's last rows, as many as the memory can take while the sort's launches wait for their own trips, are zeroed by further
// blocks of those launches, before the sums store the rows that occur (16384 tokens, 50001 x 768 fp32: 85.4 -> 79.8 us; 131072
// tokens, 131072 x 4096 bf16: 799 -> 790).  The last rows: vocabularies are often in order of frequency, and a row that
// occurs is then written twice.  (480 blocks instead of 240, or a third instead of a quarter with the counts: 80 to 81 us.)
constexpr int64_t kClearBytes = (int64_t)20 << 20;      // per part
constexpr int kClearBlocks = 240;
constexpr int kParts = 4;               // of a digit: the counts' launch takes one, the scatter the others
struct Clear {
  char* table;
  int64_t rows, row_bytes, ld_bytes;
  bool past;
};

// Returns how many of the gradient's rows, counted from the last one, are zeros afterwards.
int64_t sort_tokens(const void* ids, int wide, int64_t tokens, uint32_t rows, const Workspace& w, char* ws, const Clear& c, hipStream_t s) {
  uint32_t* keys = reinterpret_cast<uint32_t*>(ws + w.keys);
  uint32_t* order = reinterpret_cast<uint32_t*>(ws + w.order);
  int key_bits = 1;
  while ((1ull << key_bits) <= (uint64_t)rows) ++key_bits;       // keys 0 .. rows
  uint2* pairs[2] = {reinterpret_cast<uint2*>(ws + w.pairs), reinterpret_cast<uint2*>(ws + w.pairs) + tokens};
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + w.counts);
  int64_t tile = (tokens + kMaxSortBlocks - 1) / kMaxSortBlocks;
  tile = (tile + kSortThreads - 1) / kSortThreads * kSortThreads;
  const int blocks = (int)((tokens + tile - 1) / tile);
  const int passes = (key_bits + kMaxDigit - 1) / kMaxDigit;
  const int bits = (key_bits + passes - 1) / passes;
  const int64_t most = c.row_bytes ? kClearBytes / c.row_bytes : 0, share = (c.rows + kParts * passes - 1) / (kParts * passes);
  int64_t cleared = 0;
  auto grid = [&](SortPass& a, int parts) {
    a.clear_rows = std::min({share * parts, most * parts, c.rows - cleared});
    cleared += a.clear_rows;
    a.clear = c.table + (c.rows - cleared) * c.ld_bytes;
    const int64_t packs = a.clear_rows * a.clear_packs;
    return (unsigned)(blocks + std::min<int64_t>((packs + kSortThreads - 1) / kSortThreads, kClearBlocks));
  };
  for (int p = 0; p < passes; ++p) {
    SortPass a{};
    a.ids = p == 0 ? ids : nullptr;
    a.in = p == 0 ? nullptr : pairs[(p - 1) & 1];
    a.wide = wide, a.rows = rows, a.tokens = tokens, a.tile = tile, a.shift = p * bits, a.bits = bits, a.blocks = blocks;
    a.clear_ld = c.ld_bytes, a.clear_packs = (int)(c.row_bytes / 16), a.past = c.past;
    const unsigned count_grid = grid(a, 1);
    sort_count_kernel<<<count_grid, kSortThreads, 0, s>>>(a, counts);
    const unsigned scatter_grid = grid(a, kParts - 1);
    sort_scatter_kernel<<<scatter_grid, kSortThreads, 0, s>>>(a, counts, p + 1 < passes ? pairs[p & 1] : nullptr, keys, order);
  }
  return cleared;
}

template <typename T, int N, bool UPDATE>
void launch_sums(SumArgs a, const void* ids, int wide, const T* g, T* table, int64_t fill_rows, hipStream_t s) {
  a.packs = a.dim / N;
  a.lanes_log2 = log2_lanes(a.packs);
  if (few(a.tokens, a.packs, a.rows)) {
    if (!UPDATE) {
      const int64_t blocks = (fill_rows + (kThreads >> a.lanes_log2) - 1) / (kThreads >> a.lanes_log2);
      zero_rows_kernel<T, N><<<(unsigned)(blocks > 16384 ? 16384 : blocks), kThreads, 0, s>>>(table, fill_rows, a.packs, a.ldt, a.lanes_log2, a.past);
    }
    if (a.tokens > 0)
      few_kernel<T, N, UPDATE><<<dim3((unsigned)a.tokens, (a.packs + 64 * kSmallLoops - 1) / (64 * kSmallLoops)), kSmallWaves * 64, 0, s>>>(
          a, ids, wide, g, table);
    return;
  }
  const int lanes = 1 << a.lanes_log2, groups = kThreads / lanes;
  a.sum_blocks = (a.chunks + groups - 1) / groups;
  const int64_t fill = (fill_rows + kFillRows - 1) / kFillRows;
  const dim3 grid((unsigned)(a.sum_blocks + fill), (a.packs + lanes - 1) / lanes);
  if (grid.x) sum_kernel<T, N, UPDATE><<<grid, kThreads, 0, s>>>(a, g, table);
  if (a.chunks > 1) {
    // few enough chunks per block that a thousand blocks share the runs: they are a chain of trips to memory each, and the
    // frequent tokens' runs lie side by side (32768 tokens x 256: 64 chunks a block 23 us, 4 to 16 chunks 8 us)
    const int64_t slices = (a.dim + 255) / 256, per = a.chunks * slices / 1024;
    a.join_chunks = per < 4 ? 4 : per > 64 ? 64 : (int)per;
    join_kernel<T, N, UPDATE><<<dim3((unsigned)((a.chunks + a.join_chunks - 1) / a.join_chunks), (unsigned)slices), kJoinWaves * 64, 0, s>>>(a, table);
  }
}

template <typename T>
int scatter_sums(bool update, const void* ids, int wide, int64_t tokens, const void* g, int64_t ldg, void* table, int64_t ldt,
                 int64_t rows, int dim, float scale, const float* lr, void* workspace, hipStream_t s) {
  const Workspace w = plan(tokens, dim);
  char* ws = static_cast<char*>(workspace);
  SumArgs a{};
  a.keys = reinterpret_cast<uint32_t*>(ws + w.keys);
  a.order = reinterpret_cast<uint32_t*>(ws + w.order);
  a.tokens = tokens;
  a.rows = (uint32_t)rows;
  a.chunk = w.chunk;
  a.chunks = w.chunks;
  a.dim = dim;
  a.ldg = ldg;
  a.ldt = ldt;
  a.scale = scale;
  a.lr = lr;
  a.pieces = reinterpret_cast<float*>(ws + w.pieces);
  a.piece_ld = w.piece_ld;
  a.past = rows * dim * (int64_t)sizeof(T) > kCaches;
  a.g_past = tokens * dim * (int64_t)sizeof(T) > kCaches;
  const T* gp = static_cast<const T*>(g);
  T* tp = static_cast<T*>(table);
  const int bytes = dtf_access_bytes((uint64_t)g | (uint64_t)table | (uint64_t)(ldg * sizeof(T)) | (uint64_t)(ldt * sizeof(T)) |
                                     (uint64_t)(dim * sizeof(T)));
  int64_t fill = update ? 0 : rows;
  if (!few(tokens, dim / std::max<int>(bytes / (int)sizeof(T), 1), rows)) {
    Clear c{};
    if (!update && bytes == 16) c = Clear{static_cast<char*>(table), rows, (int64_t)(dim * sizeof(T)), (int64_t)(ldt * sizeof(T)), a.past};
    fill -= sort_tokens(ids, wide, tokens, (uint32_t)rows, w, ws, c, s);
  }
  auto go = [&](auto n) {
    constexpr int N = decltype(n)::value;
    if (update) launch_sums<T, N, true>(a, ids, wide, gp, tp, fill, s); else launch_sums<T, N, false>(a, ids, wide, gp, tp, fill, s);
  };
  if (bytes == 16) go(std::integral_constant<int, 16 / sizeof(T)>());
  else if (bytes == 8) go(std::integral_constant<int, 8 / sizeof(T)>());
  else if (bytes == 4 || sizeof(T) == 4) go(std::integral_constant<int, 4 / sizeof(T)>());
  else go(std::integral_constant<int, 1>());
  return hipGetLastError() == hipSuccess ? DTF_OK : DTF_ERR_LAUNCH;
}

template <typename T>
int launch_lookup(const void* table, int64_t ld, int64_t rows, const void* ids, int wide, int64_t tokens, int dim, float scale,
                  void* out, int64_t ldo, hipStream_t s) {
  const T* tp = static_cast<const T*>(table);
  T* op = static_cast<T*>(out);
  const int bytes = dtf_access_bytes((uint64_t)table | (uint64_t)out | (uint64_t)(ld * sizeof(T)) | (uint64_t)(ldo * sizeof(T)) |
                                     (uint64_t)(dim * sizeof(T)));
  auto go = [&](auto n) {
    constexpr int N = decltype(n)::value;
    const int packs = dim / N, l = log2_lanes(packs), groups = kThreads >> l;
    // four tokens at a time once that still leaves eight blocks for every CU
    const bool many = tokens / (4 * groups) >= 8 * 256;
    int64_t grid = (tokens + groups * (many ? 4 : 1) - 1) / (groups * (many ? 4 : 1));
    if (grid > (1 << 20)) grid = 1 << 20;       // (blocks x threads stays below 2^32)
    const bool past = tokens * dim * (int64_t)sizeof(T) > kCaches;
    if (many) lookup_kernel<T, N, 4><<<(unsigned)grid, kThreads, 0, s>>>(tp, ld, rows, ids, wide, tokens, packs, l, scale, op, ldo, past);
    else lookup_kernel<T, N, 1><<<(unsigned)grid, kThreads, 0, s>>>(tp, ld, rows, ids, wide, tokens, packs, l, scale, op, ldo, past);
  };
  if (bytes == 16) go(std::integral_constant<int, 16 / sizeof(T)>());
  else if (bytes == 8) go(std::integral_constant<int, 8 / sizeof(T)>());
  else if (bytes == 4 || sizeof(T) == 4) go(std::integral_constant<int, 4 / sizeof(T)>());
  else go(std::integral_constant<int, 1>());
  return hipGetLastError() == hipSuccess ? DTF_OK : DTF_ERR_LAUNCH;
}

// grids stay below 2^32 threads
constexpr int64_t kMaxTokens = (int64_t)1 << 26, kMaxRows = (int64_t)1 << 28;
constexpr int kMaxDim = 1 << 20;

bool bad_shape(int64_t tokens, int64_t rows, int dim, int dtype) {
  return tokens < 0 || tokens > kMaxTokens || rows < 1 || rows > kMaxRows || dim < 1 || dim > kMaxDim || dtype < 0 || dtype > 2;
}

}  // namespace

extern "C" int dtf_embed_lookup(const void* table, int dtype, int64_t rows, int dim, int64_t ld, const void* ids, int ids_wide,
                                int64_t tokens, float scale, void* out, int64_t ldo, void* stream) {
  if (bad_shape(tokens, rows, dim, dtype) || ld < dim || ldo < dim) return DTF_ERR_SHAPE;
  if (tokens == 0) return DTF_OK;
  if (!table || !ids || !out) return DTF_ERR_NULL;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DTF_F32) return launch_lookup<float>(table, ld, rows, ids, ids_wide, tokens, dim, scale, out, ldo, s);
  if (dtype == DTF_BF16) return launch_lookup<bf16_t>(table, ld, rows, ids, ids_wide, tokens, dim, scale, out, ldo, s);
  return launch_lookup<f16_t>(table, ld, rows, ids, ids_wide, tokens, dim, scale, out, ldo, s);
}

extern "C" int64_t dtf_embed_workspace(int64_t tokens, int dim) {
  if (tokens < 0 || tokens > kMaxTokens || dim < 1 || dim > kMaxDim) return -1;
  return plan(tokens, dim).total;
}

static int embed_scatter(bool update, const void* ids, int ids_wide, int64_t tokens, const void* g, int64_t ldg, void* table,
                         int dtype, int64_t rows, int dim, int64_t ldt, float scale, const float* lr, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  if (bad_shape(tokens, rows, dim, dtype) || ldt < dim || (tokens > 0 && ldg < dim)) return DTF_ERR_SHAPE;
  if (!table || !workspace || (tokens > 0 && (!ids || !g)) || (update && !lr)) return DTF_ERR_NULL;
  if (workspace_bytes < plan(tokens, dim).total || ((uintptr_t)workspace & 15u)) return DTF_ERR_SHAPE;
  if (update && tokens == 0) return DTF_OK;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DTF_F32)
    return scatter_sums<float>(update, ids, ids_wide, tokens, g, ldg, table, ldt, rows, dim, scale, lr, workspace, s);
  if (dtype == DTF_BF16)
    return scatter_sums<bf16_t>(update, ids, ids_wide, tokens, g, ldg, table, ldt, rows, dim, scale, lr, workspace, s);
  return scatter_sums<f16_t>(update, ids, ids_wide, tokens, g, ldg, table, ldt, rows, dim, scale, lr, workspace, s);
}

extern "C" int dtf_embed_grad(const void* ids, int ids_wide, int64_t tokens, const void* g, int64_t ldg, void* grad, int dtype,
                              int64_t rows, int dim, int64_t ldt, float scale, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  return embed_scatter(false, ids, ids_wide, tokens, g, ldg, grad, dtype, rows, dim, ldt, scale, nullptr, workspace,
                       workspace_bytes, stream);
}

extern "C" int dtf_embed_sgd(const void* ids, int ids_wide, int64_t tokens, const void* g, int64_t ldg, void* table, int dtype,
                             int64_t rows, int dim, int64_t ldt, float scale, const float* lr, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  return embed_scatter(true, ids, ids_wide, tokens, g, ldg, table, dtype, rows, dim, ldt, scale, lr, workspace, workspace_bytes,
                       stream);
}
