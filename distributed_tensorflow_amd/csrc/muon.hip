// Orthogonalised update of matrices (the Muon optimiser): five Newton-Schulz steps in place of a singular value
// decomposition.  For a gradient G [rows][cols] with a momentum buffer,
//
//   buf = mu * buf + G;   U = G + mu * buf  (Nesterov)  or  U = buf
//   X = U / (|U|_F + eps)                                          (on the transpose where rows > cols: m <= n below)
//   5 times:   A = X X^T,   B = b A + c A A,   X = a X + B X         (a, b, c) = (3.4445, -4.7750, 2.0315)
//   W -= lr * sqrt(max(1, cols / rows)) * X
//
// The singular values of X run through the odd quintic a s + b s^3 + c s^5, which lifts small ones by 3.4 a step and keeps
// those near one between 0.7 and 1.2: after five steps X is close to the orthogonal factor of U.
//
// Bound by the matrix cores: 5 (m^2 n + m^3 + 2 m^2 n) flops (A and B are symmetric: only the tiles on and above the
// diagonal are computed, and stored twice).  The small singular values are amplified by up to 3.4^5 = 485, and with them
// every rounding, so 16-bit products alone are not enough for an fp32 result, and fp32 MFMA has 1/16 of the fp16 rate.
// Every matrix is therefore kept as TWO fp16 planes, hi + lo = the value times a power of two: 22 significant bits, fewer only
// below 2^-16 of the largest possible entry (all entries are bounded: |X| <= 1.2, |A| <= 1.45, |B| <= 2.9 by the quintic).
// A product is three fp16 MFMAs, hi hi + hi lo + lo hi, summed in fp32; what is dropped, lo lo, is 2^-22 of the product, less
// than the rounding of an fp32 sum of a few terms.  Simulated and measured, the result is as far from the 64-bit iteration
// as that of fp32 matrix products (the fp32 sums dominate both).  (Iterating in the m x m space of the Gram matrix needs fewer
// flops for n > m but squares the condition: 5 to 16 times the error on gradients with a decaying spectrum; not used.)
//
// Layout.  Both operands of every product are read along k: A = X X^T takes rows of X twice, A A takes rows of the symmetric
// A, B X takes rows of B and rows of X^T.  So X is kept together with its transpose, each step's product writes both, and one
// GEMM form (row times row) serves all.  A row of a plane pair is groups of 32 columns: 32 hi halves then 32 lo halves, 128
// bytes, one cache line per row and k-step.  Dimensions are padded with zeros to whole tiles: the products need no bounds.
//
// GEMM.  A workgroup of four waves owns a square tile of 64, 128, 192 or 256 (or 32, see Narrow) and walks k in steps of 32 through a
// ring of 8, 4, 3 or 2 LDS images filled by direct buffer-to-LDS loads: 148, 132, 144 or 128 KB (ring_bytes()), one workgroup per CU, the
// loads of a step requested one to seven steps ahead of it (the matrices come from the other XCDs' writes: 0.8 us away, against 0.1 to 1.8 us of products per
// step).  A load instruction moves eight 128-byte rows; its LDS side is fixed (lane l at 16 l), so the 16-byte chunks of a row are
// permuted on the GLOBAL side: slot s of row r holds chunk s ^ ((r >> 1) & 7), and the sixteen rows that a quarter of a fragment
// read touches fill all 64 banks once (rows r and r + 1 lie in the two halves of the banks; measured: no conflict).
// A step's two halves of 16 k alternate between two sets of fragment registers: the LDS reads of one half and the loads are
// spread between the MFMAs of the half before, across the step's single barrier too.  Large tiles matter: per k-step of a
// tile of edge T the matrix cores are busy for 0.047 T^2 cycles and the LDS for 6 T (reads by four waves of T/2 x T/2, and the
// loads).  Tile edge and split of k are chosen per stage by a cost estimate (see choose()).  Few tiles and a long k: several
// workgroups take a range of k each and store their sums; a second launch adds them in order and does what the product's
// own end does otherwise.
//
// All matrices of a call go through each launch together: 2 + 15 launches per step of the optimiser (up to 15 more where k is
// split), whatever the number of layers (up to 8; more are taken in groups).
#include "dtf_api.h"
#include "dtf_types.h"

namespace {

typedef f16_t half8 __attribute__((ext_vector_type(8)));
typedef f16_t half4 __attribute__((ext_vector_type(4)));
typedef f16_t half2 __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kMax = DTF_MUON_MAX;
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScaleX = 32768.f, kScaleA = 16384.f, kScaleB = 8192.f;    // powers of two: entries stay below 65504
constexpr int kNormBlocks = 1024;     // at most: four partial sums a thread of split_kernel
constexpr int kWaves = 4;              // of a product workgroup

// One matrix of a call.  `rows` x `cols` as the caller has it; m <= n its shape (or its transpose's) padded to mp x np.
struct Item {
  const void* u;        // G, or the matrix to orthogonalise
  float* buf;           // momentum (null: orthogonalise u itself)
  void* out;            // W (updated) or the result
  int64_t ldu, ldo;
  int rows, cols, m, n, mp, np, flip;
  float shape_factor;   // sqrt(max(1, cols / rows))
  char *X, *XT[2], *A, *B;
  double* norm;         // partial sums of squares
};

struct Call {
  Item item[kMax];
  int count, dtype;
  float mu, eps;
  int nesterov;
  int norm_blocks;
  const float* lr;
};

// --- momentum and norm ----------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float direction(const Call& c, const Item& it, int64_t at_u, int64_t at_buf) {
  const float g = (float)static_cast<const T*>(it.u)[at_u];
  if (!it.buf) return g;
  const float b = it.buf[at_buf];
  return c.nesterov ? g + c.mu * b : b;
}

template <typename T>
__global__ __launch_bounds__(256) void norm_kernel(Call c) {
  const Item& it = c.item[blockIdx.y];
  const int64_t total = (int64_t)it.rows * it.cols, stride = (int64_t)gridDim.x * 256;
  const int64_t me = (int64_t)blockIdx.x * 256 + threadIdx.x;
  double sum = 0;
  // four elements at a time where the matrix has no gaps and is aligned; the rest, or all of a strided one, one by one
  const bool flat = it.ldu == it.cols && (reinterpret_cast<uintptr_t>(it.u) % (4 * sizeof(T))) == 0 &&
                    (reinterpret_cast<uintptr_t>(it.buf) & 15u) == 0;
  const int64_t quads = flat ? total / 4 : 0;
  for (int64_t q = me; q < quads; q += stride) {
    const Pack<T, 4> g = reinterpret_cast<const Pack<T, 4>*>(it.u)[q];
    f32x4 u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = (float)g.v[e];
    if (it.buf) {
      f32x4* at = reinterpret_cast<f32x4*>(it.buf) + q;
      const f32x4 b = c.mu * *at + u;
      *at = b;
      u = c.nesterov ? u + c.mu * b : b;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += (double)u[e] * (double)u[e];
  }
  for (int64_t i = 4 * quads + me; i < total; i += stride) {
    int64_t at = i;
    if (it.ldu != it.cols) {
      const int64_t r = i / it.cols;
      at = r * it.ldu + (i - r * it.cols);
    }
    if (it.buf) it.buf[i] = c.mu * it.buf[i] + (float)static_cast<const T*>(it.u)[at];
    const double u = direction<T>(c, it, at, i);
    sum += u * u;
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x);
  __shared__ double of_wave[4];
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) it.norm[blockIdx.x] = (of_wave[0] + of_wave[1]) + (of_wave[2] + of_wave[3]);
}

// --- plane pairs ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t split_pair(float scaled) {       // hi | lo << 16
  const f16_t hi = (f16_t)scaled;
  const f16_t lo = (f16_t)(scaled - (float)hi);
  return (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
}
// Byte offset of the hi half of (row, col) of a plane pair with `cols` padded columns; its lo half is 64 bytes on.
__device__ __forceinline__ int64_t plane_at(int64_t row, int col, int cols) {
  return row * cols * 4 + (col >> 5) * 128 + (col & 31) * 2;
}
// A 64 x 64 tile of pairs in LDS, its rows `line` and its columns `step` words apart, to row0, col0 of a plane pair: 256 bytes a
// row, sixteen bytes a thread and turn, consecutive threads one behind the other (64 bytes a thread: the kernel took 23 us
// for 1024 x 4096 instead of 17).
__device__ __forceinline__ void store_tile(char* plane, int row0, int col0, int cols, const uint32_t* pairs, int line, int step) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int row = k * 16 + (threadIdx.x >> 4), chunk = threadIdx.x & 15;      // chunk: group of 32 columns, hi or lo, 8 columns
    const int col = (chunk >> 3) * 32 + (chunk & 3) * 8, shift = (chunk >> 2 & 1) * 16;
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t* at = pairs + row * line + (col + 2 * e) * step;
      w[e] = (at[0] >> shift & 0xffffu) | (at[step] >> shift) << 16;
    }
    *reinterpret_cast<u32x4*>(plane + plane_at(row0 + row, col0, cols) + chunk * 16) = w;
  }
}

// X and X^T of U / (|U| + eps), 64 x 64 tiles of the padded shape.
template <typename T>
__global__ __launch_bounds__(256) void split_kernel(Call c) {
  __shared__ uint32_t tile[64][65];
  __shared__ double of_wave[4];
  const Item& it = c.item[blockIdx.y];
  const int pr = it.flip ? it.np : it.mp, pc = it.flip ? it.mp : it.np;       // padded rows and columns as the caller has them
  const int tiles_c = pc / 64, tiles = (pr / 64) * tiles_c;
  if ((int)blockIdx.x >= tiles) return;
  const int r0 = (blockIdx.x / tiles_c) * 64, c0 = (blockIdx.x % tiles_c) * 64;
  const int col = threadIdx.x & 63;
  // All requests at once and before the norm is added up, from clamped places: one by one they took 15 us.
  const T* gp = static_cast<const T*>(it.u) + min(c0 + col, it.cols - 1);
  const float* bp = it.buf + min(c0 + col, it.cols - 1);
  float u[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) u[k] = (float)gp[(int64_t)min(r0 + (int)(threadIdx.x >> 6) + 4 * k, it.rows - 1) * it.ldu];
  float b[16];
  if (it.buf) {
#pragma unroll
    for (int k = 0; k < 16; ++k) b[k] = bp[(int64_t)min(r0 + (int)(threadIdx.x >> 6) + 4 * k, it.rows - 1) * it.cols];
  }
  double total = 0;
#pragma unroll
  for (int i = 0; i < kNormBlocks; i += 256) {
    const double part = it.norm[min(i + (int)threadIdx.x, c.norm_blocks - 1)];
    total += i + (int)threadIdx.x < c.norm_blocks ? part : 0.0;
  }
  if (it.buf) {
#pragma unroll
    for (int k = 0; k < 16; ++k) u[k] = c.nesterov ? u[k] + c.mu * b[k] : b[k];
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) total += __shfl_xor(total, x);
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = total;
  __syncthreads();
  const double inv = (double)kScaleX / (sqrt((of_wave[0] + of_wave[1]) + (of_wave[2] + of_wave[3])) + (double)c.eps);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = (threadIdx.x >> 6) + 4 * k;
    tile[r][col] = r0 + r < it.rows && c0 + col < it.cols ? split_pair((float)((double)u[k] * inv)) : 0u;
  }
  __syncthreads();
  char* straight = it.flip ? it.XT[0] : it.X;          // [pr][pc]
  char* turned = it.flip ? it.X : it.XT[0];            // [pc][pr]
  store_tile(straight, r0, c0, pc, &tile[0][0], 65, 1);
  store_tile(turned, c0, r0, pr, &tile[0][0], 1, 65);
}

// --- products -----------------------------------------------------------------------------------------------------------
enum Stage { kGram = 0, kPoly = 1, kStep = 2, kLast = 3 };     // A = X X^T;  B = bA + cAA;  X = aX + BX;  the same, to the output

// What the launches of a stage read beside the planes themselves: 64 bytes a matrix, 512 for all of them, so that one load
// instruction brings them into a wave's registers, whichever its matrix is (see find()).
struct Job {
  const char *p, *q;          // the operands: rows of k
  const char* linear;         // of the linear term: A, or X through its transpose
  char *straight, *turned;    // the result, and its transpose
  int rows, cols, depth;      // of the product, padded
  int first, tiles;           // first tile and number of tiles
  int spare;
};
static_assert(sizeof(Job) == 64, "find() counts words");
struct Jobs {
  Job job[kMax];
  float* partial;             // split products: [tile][split][elements of a tile]
  int splits;                 // workgroups per tile, a range of k each
};
// Where the last product goes.
struct Final {
  void* out;
  int64_t ld;
  int m, n, flip;
  float shape_factor;
};
struct Finals {
  Final of[kMax];
  const float* lr;            // null: the factor itself, in `dtype`
  int dtype;
};
struct None {};
template <int STAGE>
struct EndOf {
  typedef None Args;
  struct Mine {};
  static __device__ __forceinline__ Mine take(const Args&, int) { return Mine{}; }
};
template <>
struct EndOf<kLast> {
  typedef Finals Args;
  struct Mine {
    Final f;
    const float* lr;
    int dtype;
  };
  static __device__ __forceinline__ Mine take(const Args& a, int which) { return Mine{a.of[which], a.lr, a.dtype}; }
};

// The matrix that workgroup (or wave) `id` works for, with `per` of them to a tile.  Looked up field by field the arguments were
// several trips to memory one behind the other: here every lane loads two words and the rest are reads of lanes (stack of three
// matrices 130 -> 127 us).
struct Task : Job {
  int which;
};
__device__ __forceinline__ Task find(const Jobs& jobs, int id, int per, int lane) {
  const uint2v mine = reinterpret_cast<const uint2v*>(&jobs)[lane];
  auto word = [&](int i, int k) { return (uint32_t)__builtin_amdgcn_readlane(k & 1 ? mine[1] : mine[0], 8 * i + (k >> 1)); };
  auto address = [&](int i, int k) {
    return (char*)(__attribute__((address_space(1))) char*)((uint64_t)word(i, k + 1) << 32 | word(i, k));
  };
  Task t;
  t.which = 0;
#pragma unroll
  for (int i = 1; i < kMax; ++i) t.which += id >= (int)word(i, 13) * per ? 1 : 0;
  t.p = address(t.which, 0), t.q = address(t.which, 2), t.linear = address(t.which, 4);
  t.straight = address(t.which, 6), t.turned = address(t.which, 8);
  t.rows = (int)word(t.which, 10), t.cols = (int)word(t.which, 11), t.depth = (int)word(t.which, 12);
  t.first = (int)word(t.which, 13), t.tiles = (int)word(t.which, 14);
  return t;
}

// At most `LEFT` of this wave's loads are still under way and its LDS reads are done, then the workgroup's.  (A barrier alone does
// not wait for loads that go to LDS, and __syncthreads() would wait for all of them.  The empty statements keep the compiler's
// own memory accesses on their side.)
template <int LEFT, bool BARRIER = true>
__device__ __forceinline__ void wait_and_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | (LEFT >> 4) << 14 | 7 << 4);     // vmcnt LEFT, lgkmcnt 0, expcnt untouched
  if (BARRIER) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ROWS rows of a plane pair from a tile's first row on; rows past the last one are read as the last one (their products are not
// stored).
template <int ROWS, int WAVES>
struct Fetcher {
  static constexpr int kLoads = ROWS / (8 * WAVES);
  const char* base;
  unsigned at[kLoads];
  __device__ __forceinline__ void init(const char* plane, int row0, int rows, int64_t row_bytes, int wave, int lane) {
    base = plane + row0 * row_bytes;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (i * WAVES + wave) * 8 + (lane >> 3);
      at[i] = (unsigned)(min(r, rows - 1 - row0) * row_bytes) + (unsigned)(((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
  }
  // The 128-byte group `k` of every row to an LDS image.
  __device__ __forceinline__ void go(char* __restrict lds, int wave, int k) const {
#ifdef __HIP_DEVICE_COMPILE__          // (the host pass of the compiler does not know the descriptor's type)
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, (int)0xffffffffu, 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(lds + (i * WAVES + wave) * 1024), 16, at[i], k * 128, 0, 0);
#endif
  }
};

// Operands of one half of a k-step (16 k): MI and NI tiles of 32 rows, hi and lo.
template <int MI, int NI>
struct Half {
  half8 a[MI][2], b[NI][2];
  // `p`, `q`: LDS images of the workgroup's rows of the two operands
  __device__ __forceinline__ void read(const char* __restrict p, const char* __restrict q, int row_p, int row_q, int lane, int ks) {
    const int r = lane & 31;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int slot = ((h * 4 + ks * 2 + (lane >> 5)) ^ ((r >> 1) & 7)) << 4;      // (every base row is a multiple of 32)
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i][h] = *reinterpret_cast<const half8*>(p + (row_p + 32 * i + r) * 128 + slot);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[j][h] = *reinterpret_cast<const half8*>(q + (row_q + 32 * j + r) * 128 + slot);
    }
  }
  // hi lo, lo hi, hi hi; the three MFMAs of a tile are MI * NI apart, or, with SUMS = 3, have a sum each (a chain of MFMAs on
  // one sum runs at half their rate)
  template <int SUMS>
  __device__ __forceinline__ void multiply(f32x16 (&acc)[SUMS][MI][NI]) const {
#pragma unroll
    for (int t = 0; t < 3; ++t)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          f32x16& sum = acc[SUMS == 3 ? t : 0][i][j];
          sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][t == 1], b[j][t == 0], sum, 0, 0, 0);
        }
  }
};

// Instruction order of a half step: the LDS reads of the next half (and, with LOADS, the loads) spread over the first three
// quarters of its MFMAs.  A wave issues in order: reads in one block left the matrix pipe idle while they queued for the LDS
// (52 % busy against 69 % at 4096 x 4096).
template <int R, int READS, int MFMAS, int LOADS>
__device__ __forceinline__ void interleave() {
  constexpr int kOver = MFMAS - MFMAS / 4;
  if constexpr (R < READS) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                                // an LDS read
    if constexpr ((R + 1) * LOADS / READS > R * LOADS / READS)
      __builtin_amdgcn_sched_group_barrier(0x010, (R + 1) * LOADS / READS - R * LOADS / READS, 0);    // a load
    if constexpr ((R + 1) * kOver / READS > R * kOver / READS)
      __builtin_amdgcn_sched_group_barrier(0x008, (R + 1) * kOver / READS - R * kOver / READS, 0);    // MFMAs
    interleave<R + 1, READS, MFMAS, LOADS>();
  } else {
    __builtin_amdgcn_sched_group_barrier(0x008, MFMAS - kOver, 0);
  }
}

// A wave's 32 x 32 tile of a stage's product, rows from i0 and columns from j0 on.  Element e of a lane: row 8 (e / 4) +
// 4 (lane / 32) + e % 4 and column lane % 32.  In memory it is 32 lines of 128 bytes, and every access below moves whole lines (lane
// l has the 16-byte chunk l % 8 of line l / 8 + 8 n): accesses of 8 or 16 bytes to 32 lines at a time cost 5000 cycles a tile.
// The way between the two layouts is through LDS.
constexpr int kTurnRow = 36;                      // words of a line: its 16-byte chunks spread over the banks
constexpr int kTurnWords = 2 * 32 * kTurnRow;     // two turning areas of a wave
// Order of a wave's own LDS accesses (nobody else touches its areas).
__device__ __forceinline__ void own_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

struct Linear {
  u32x4 chunk[4];
  __device__ __forceinline__ void read(const Task& t, int i0, int j0, int lane) {
    const char* s = t.linear + plane_at(j0 + (lane >> 3), i0, t.rows) + 16 * (lane & 7);
#pragma unroll
    for (int n = 0; n < 4; ++n) chunk[n] = *reinterpret_cast<const u32x4*>(s + (int64_t)n * 8 * t.rows * 4);
  }
};

// What becomes of the tile.  `area`: the wave's turning areas.  `mirror`: also store the transposed tile of a symmetric result.
template <int STAGE>
__device__ __forceinline__ void store_tile(const Task& t, const typename EndOf<STAGE>::Mine& end, int i0, int j0, bool mirror,
                                           const f32x16& sum, const Linear& linear, uint32_t* area, int lane) {
  const int half = lane >> 5, jc = lane & 31;
  uint32_t* turn = area;
  uint32_t* lines = area + 32 * kTurnRow;
  float v[16];
  if (STAGE == kGram) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = sum[e] * (kScaleA / (kScaleX * kScaleX));
  } else {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      *reinterpret_cast<u32x4*>(lines + ((lane >> 3) + 8 * n) * kTurnRow + 4 * (lane & 7)) = linear.chunk[n];
    own_lds();
    const float lin = STAGE == kPoly ? kB * (kScaleB / kScaleA) : STAGE == kStep ? kA : kA / kScaleX;
    const float quad = STAGE == kPoly ? kC * kScaleB / (kScaleA * kScaleA)
                       : STAGE == kStep ? 1.f / kScaleB : 1.f / (kScaleB * kScaleX);
    const char* line = reinterpret_cast<const char*>(lines + jc * kTurnRow) + 8 * half;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const half4 hi = *reinterpret_cast<const half4*>(line + 16 * g), lo = *reinterpret_cast<const half4*>(line + 64 + 16 * g);
#pragma unroll
      for (int x = 0; x < 4; ++x)      // (two mixed-precision multiply-adds: the planes are not converted)
        v[4 * g + x] = fmaf((float)hi[x], lin, fmaf((float)lo[x], lin, quad * sum[4 * g + x]));
    }
  }
  if constexpr (STAGE == kLast) {
    const Final& it = end.f;
    // (places past the matrix are read as its last ones and not stored)
    const int64_t step_row = it.flip ? 1 : it.ld, step_col = it.flip ? it.ld : 1;
    const int row0 = i0 + 4 * half, col = j0 + jc;
    const int64_t at_col = min(col, it.n - 1) * step_col;
    auto place = [&](int e) { return min(row0 + 8 * (e / 4) + e % 4, it.m - 1) * step_row + at_col; };
    auto inside = [&](int e) { return row0 + 8 * (e / 4) + e % 4 < it.m && col < it.n; };
    if (end.lr || end.dtype == DTF_F32) {
      float* out = static_cast<float*>(it.out);
      if (end.lr) {                       // the weights: all of them requested before the first store
        const float step_size = end.lr[0] * it.shape_factor;
        float old[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) old[e] = out[place(e)];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = old[e] - step_size * v[e];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (inside(e)) out[place(e)] = v[e];
    } else {
      uint16_t* out = static_cast<uint16_t*>(it.out);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint16_t bits = end.dtype == DTF_BF16 ? __builtin_bit_cast(uint16_t, (bf16_t)v[e]) : __builtin_bit_cast(uint16_t, (f16_t)v[e]);
        if (inside(e)) out[place(e)] = bits;
      }
    }
    return;
  }
  // hi and lo of two rows at a time
  half2 hi[8], lo[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const float2v x = {v[2 * p], v[2 * p + 1]};
    hi[p] = __builtin_convertvector(x, half2);
    lo[p] = __builtin_convertvector(x - __builtin_convertvector(hi[p], float2v), half2);
  }
  f16_t* at = reinterpret_cast<f16_t*>(turn + 4 * half * kTurnRow) + jc;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    at[(8 * (e / 4) + e % 4) * 2 * kTurnRow] = hi[e / 2][e % 2];
    at[(8 * (e / 4) + e % 4) * 2 * kTurnRow + 32] = lo[e / 2][e % 2];
  }
  if (mirror) {
    // Line j of the transposed tile: this lane has rows 4 half .. 4 half + 3 of every eight, the lane 32 away the other four.
    // Exchanged between two groups of eight, each lane holds whole chunks.
    own_lds();                            // (the linear term has been read)
    uint32_t* line = lines + jc * kTurnRow + 4 * half;
#pragma unroll
    for (int g = 0; g < 4; g += 2)
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const half2* of = part ? lo : hi;
        const auto s0 = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, of[2 * g]), __builtin_bit_cast(uint32_t, of[2 * g + 2]), false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, of[2 * g + 1]), __builtin_bit_cast(uint32_t, of[2 * g + 3]), false, false);
        *reinterpret_cast<u32x4*>(line + 4 * g + 16 * part) = u32x4{s0[0], s1[0], s0[1], s1[1]};
      }
  }
  own_lds();
  const int l8 = lane >> 3, chunk = lane & 7;
  if (mirror) {
    char* to = t.turned + plane_at(j0 + l8, i0, t.rows) + 16 * chunk;
#pragma unroll
    for (int n = 0; n < 4; ++n)
      *reinterpret_cast<u32x4*>(to + (int64_t)n * 8 * t.rows * 4) = *reinterpret_cast<const u32x4*>(lines + (l8 + 8 * n) * kTurnRow + 4 * chunk);
  }
  const int cols = t.cols;
  char* to = t.straight + plane_at(i0 + l8, j0, cols) + 16 * chunk;
#pragma unroll
  for (int n = 0; n < 4; ++n)
    *reinterpret_cast<u32x4*>(to + (int64_t)n * 8 * cols * 4) = *reinterpret_cast<const u32x4*>(turn + (l8 + 8 * n) * kTurnRow + 4 * chunk);
  own_lds();
}

// Tile `t` of a stage: rows and columns in tiles.  Symmetric results: t = tj (tj + 1) / 2 + ti, ti <= tj.
template <int STAGE>
__device__ __forceinline__ void tile_place(const Task& task, int edge, int t, int& ti, int& tj) {
  if (STAGE <= kPoly) {
    tj = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (tj * (tj + 1) / 2 > t) --tj;
    while ((tj + 1) * (tj + 2) / 2 <= t) ++tj;
    ti = t - tj * (tj + 1) / 2;
  } else {
    // groups of eight tile rows, column by column inside: neighbours share rows of both operands
    const int tiles_m = (task.rows + edge - 1) / edge, tiles_n = (task.cols + edge - 1) / edge;
    const int group = t / (8 * tiles_n), high = min(8, tiles_m - 8 * group), in = t - group * 8 * tiles_n;
    tj = in / high;
    ti = 8 * group + in - tj * high;
  }
}

constexpr int ring_of(int tile) { return tile == 256 ? 2 : tile == 192 ? 3 : tile == 128 ? 4 : 8; }
constexpr int kTurn = kWaves * kTurnWords * 4;      // all waves' turning areas, in bytes

constexpr int ring_bytes(int tile) {                // (image 0 becomes the turning areas, and is as large as those)
  return (2 * tile * 128 < kTurn ? kTurn : 2 * tile * 128) + (ring_of(tile) - 1) * 2 * tile * 128;
}
static_assert(ring_bytes(64) == 148 << 10 && ring_bytes(128) == 132 << 10 && ring_bytes(192) == 144 << 10 && ring_bytes(256) == 128 << 10,
              "a CU has 160 KB");

// LDS image I of the ring: the rows of one operand, then the other's.  (One variable each: the compiler must see that a load to
// one image does not concern the reads of another.)
template <int TILE, int I>
__device__ __forceinline__ char* image() {
  __shared__ __attribute__((aligned(1024))) char bytes[I == 0 && 2 * TILE * 128 < kTurn ? kTurn : 2 * TILE * 128];
  return bytes;
}

template <int TILE>
struct Product {
  static constexpr int kRing = ring_of(TILE), MI = TILE / 64, NI = TILE / 64;
  static constexpr int kLoads = 2 * Fetcher<TILE, kWaves>::kLoads;       // of a wave and step
  static constexpr int kReads = 2 * (MI + NI), kMfmas = 3 * MI * NI, kSums = MI * NI == 1 ? 3 : 1;
  typedef f32x16 Sums[kSums][MI][NI];
  // Small tiles have registers for all fragments of two steps: the reads of step k are covered by the whole of step k - 1, and the
  // wait in front of the barrier finds them done (128: 931 -> 890 cycles a step; 64 stays at 417, of which
  // its LDS accesses take 384).
  static constexpr bool kWhole = TILE <= 128;
  Fetcher<TILE, kWaves> p, q;
  Half<MI, NI> first, second;               // halves of a step, in turn
  Half<MI, NI> whole[2][2];                 // kWhole: [step parity][half]
  int wave, lane, row_p, row_q;

  template <int I>
  __device__ __forceinline__ void load(int k) const {
    p.go(image<TILE, I>(), wave, k);
    q.go(image<TILE, I>() + TILE * 128, wave, k);
  }
  template <int I>
  __device__ __forceinline__ void preload(int k, int last) const {
    if constexpr (I < kRing - 1) {
      load<I>(min(k + I, last));
      preload<I + 1>(k, last);
    }
  }
  // Step k, in image I; `last`: the last step of the range (loaded again by the steps at the end, which nobody reads).
  template <int I>
  __device__ __forceinline__ void step(Sums& acc, int k, int last) {
    wait_and_barrier<(kRing - 2) * kLoads>();          // step k has landed, every wave is done with step k - 1
    load<(I + kRing - 1) % kRing>(min(k + kRing - 1, last));
    if constexpr (kWhole) {
#pragma unroll
      for (int h = 0; h < 2; ++h) whole[I & 1][h].read(image<TILE, I>(), image<TILE, I>() + TILE * 128, row_p, row_q, lane, h);
#pragma unroll
      for (int h = 0; h < 2; ++h) whole[~I & 1][h].template multiply<kSums>(acc);      // step k - 1
      interleave<0, 2 * kReads, 2 * kMfmas, kLoads>();
      __builtin_amdgcn_sched_barrier(0);
      return;
    }
    first.read(image<TILE, I>(), image<TILE, I>() + TILE * 128, row_p, row_q, lane, 0);
    second.template multiply<kSums>(acc);                              // the second half of step k - 1
    interleave<0, kReads, kMfmas, kLoads>();
    __builtin_amdgcn_sched_barrier(0);
    second.read(image<TILE, I>(), image<TILE, I>() + TILE * 128, row_p, row_q, lane, 1);
    first.template multiply<kSums>(acc);
    interleave<0, kReads, kMfmas, 0>();
    __builtin_amdgcn_sched_barrier(0);
  }
  // Steps k, k + 1, ... of two rounds of the ring; whether the range goes on behind them.
  static constexpr int kSteps = 2 * kRing;
  template <int I>
  __device__ __forceinline__ bool turn(Sums& acc, int k, int last) {
    step<I % kRing>(acc, k + I, last);
    if (I % 2 == 1 && k + I == last) return false;      // (ranges are whole pairs of steps)
    if constexpr (I + 1 < kSteps) return turn<I + 1>(acc, k, last);
    return true;
  }
  __device__ __forceinline__ void run(Sums& acc, int first_step, int last) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {                      // (the first step multiplies these)
#pragma unroll
      for (int i = 0; i < MI; ++i) second.a[i][h] = half8{};
#pragma unroll
      for (int j = 0; j < NI; ++j) second.b[j][h] = half8{};
    }
    whole[1][0] = whole[1][1] = second;
    preload<0>(first_step, last);
    int k = first_step;
    if constexpr (kRing == 2) {                        // (one way out, which the accumulators of the largest tile need to stay
#pragma clang loop unroll(disable)
      for (; k < last; k += 2) {                       //  where they are)
        step<0>(acc, k, last);
        step<1>(acc, k + 1, last);
      }
    } else {
      // (the first turn stands by itself: at the head of a loop the compiler waits for every load once)
      if (turn<0>(acc, k, last)) {
        k += kSteps;
#pragma clang loop unroll(disable)
        while (turn<0>(acc, k, last)) k += kSteps;
      }
    }
    if constexpr (kWhole) {
#pragma unroll
      for (int h = 0; h < 2; ++h) whole[1][h].template multiply<kSums>(acc);
    } else {
      second.template multiply<kSums>(acc);
    }
    wait_and_barrier<0>();                             // nothing is on its way to the images any more, and nobody reads them
  }
};

// Where a product workgroup works: matrix, part of k, tile.  Workgroups go round the eight XCDs; numbered so that those of one XCD
// follow each other, and with the tiles of one range of k next to each other, the workgroups that share an L2 read the same rows.
struct Place {
  Task task;
  int part, tile;
};
__device__ __forceinline__ Place place_of(const Jobs& jobs, int lane) {
  const int per = gridDim.x >> 3, extra = gridDim.x & 7, xcd = blockIdx.x & 7;
  const int id = xcd * per + min(xcd, extra) + (int)(blockIdx.x >> 3);
  Place at;
  at.task = find(jobs, id, jobs.splits, lane);
  const int local = id - at.task.first * jobs.splits;
  at.part = local / at.task.tiles, at.tile = local - at.part * at.task.tiles;
  return at;
}

// Tiles of 32, for launches that leave most CUs without a larger one: their time is the way from memory, so the four waves share
// the tile's steps, each with a ring of its own (sixteen steps under way instead of eight) and nothing to wait for but its own loads.
struct Narrow {
  static constexpr int kRing = 4;
  Fetcher<32, 1> p, q;
  int wave, lane;
  static constexpr int kLoads = 2 * Fetcher<32, 1>::kLoads;
  template <int I>
  __device__ __forceinline__ char* mine() const { return image<128, I>() + wave * 8192; }
  template <int I>
  __device__ __forceinline__ void load(int k) const {
    p.go(mine<I>(), 0, k);
    q.go(mine<I>() + 4096, 0, k);
  }
  template <int I>
  __device__ __forceinline__ void preload(int k, int last) const {
    if constexpr (I < kRing - 1) {
      load<I>(min(k + I * kWaves, last));
      preload<I + 1>(k, last);
    }
  }
  // Steps k, k + kWaves, ... up to `last`, a round of the ring; whether the range goes on behind them.
  template <int I>
  __device__ __forceinline__ bool turn(f32x16 (&acc)[3][1][1], int k, int last) const {
    wait_and_barrier<(kRing - 2) * kLoads, false>();        // this step has landed, the fragments of the one before are in registers
    load<(I + kRing - 1) % kRing>(min(k + (I + kRing - 1) * kWaves, last));
    Half<1, 1> half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) half[h].read(mine<I>(), mine<I>() + 4096, 0, 0, lane, h);
#pragma unroll
    for (int h = 0; h < 2; ++h) half[h].template multiply<3>(acc);
    if (k + (I + 1) * kWaves > last) return false;
    if constexpr (I + 1 < kRing) return turn<I + 1>(acc, k, last);
    return true;
  }
  __device__ __forceinline__ void run(f32x16 (&acc)[3][1][1], int k, int last) const {
    preload<0>(k, last);
    if (turn<0>(acc, k, last)) {
      k += kRing * kWaves;
#pragma clang loop unroll(disable)
      while (turn<0>(acc, k, last)) k += kRing * kWaves;
    }
  }
};

template <int STAGE>
__global__ __launch_bounds__(kWaves * 64, 1) void narrow_kernel(Jobs jobs, typename EndOf<STAGE>::Args ends) {
  Narrow g;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of(jobs, lane);
  const Task& task = at.task;
  const auto end = EndOf<STAGE>::take(ends, task.which);
  int ti, tj;
  tile_place<STAGE>(task, 32, at.tile, ti, tj);
  const int64_t row_bytes = (int64_t)task.depth * 4;
  g.p.init(task.p, ti * 32, task.rows, row_bytes, 0, lane);
  g.q.init(task.q, tj * 32, task.cols, row_bytes, 0, lane);
  g.wave = wave, g.lane = lane;
  Linear linear{};
  if (STAGE != kGram && wave == 0) linear.read(task, ti * 32, tj * 32, lane);
  f32x16 sums[3][1][1];
#pragma unroll
  for (int t = 0; t < 3; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[t][0][0][e] = 0.f;
  if (wave < task.depth / 32) g.run(sums, wave, task.depth / 32 - 1);
  f32x16& sum = sums[0][0][0];
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] += sums[1][0][0][e] + sums[2][0][0][e];
  wait_and_barrier<0>();                  // nothing is on its way to the images any more, and nobody reads them
  f32x4* line = reinterpret_cast<f32x4*>(image<128, 1>()) + lane;
  if (wave > 0) {
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      line[(wave * 4 + g4) * 64] = f32x4{sum[4 * g4], sum[4 * g4 + 1], sum[4 * g4 + 2], sum[4 * g4 + 3]};
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const f32x4 v = line[(w * 4 + g4) * 64];
#pragma unroll
      for (int x = 0; x < 4; ++x) sum[4 * g4 + x] += v[x];
    }
  store_tile<STAGE>(task, end, ti * 32, tj * 32, STAGE > kPoly || ti != tj, sum, linear, reinterpret_cast<uint32_t*>(image<128, 0>()), lane);
}

template <int TILE, int STAGE>
__global__ __launch_bounds__(kWaves * 64, 1) void product_kernel(Jobs jobs, typename EndOf<STAGE>::Args all_ends) {
  constexpr int MI = Product<TILE>::MI, NI = Product<TILE>::NI;
  Product<TILE> g;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of(jobs, lane);
  const Task& task = at.task;
  const auto end = EndOf<STAGE>::take(all_ends, task.which);
  const int part = at.part, tile = at.tile, splits = jobs.splits;
  int ti, tj;
  tile_place<STAGE>(task, TILE, tile, ti, tj);
  const int64_t row_bytes = (int64_t)task.depth * 4;            // (an even number of steps of 32)
  g.p.init(task.p, ti * TILE, task.rows, row_bytes, wave, lane);
  g.q.init(task.q, tj * TILE, task.cols, row_bytes, wave, lane);
  g.wave = wave, g.lane = lane;
  const int row_p = g.row_p = (wave >> 1) * (TILE / 2), row_q = g.row_q = (wave & 1) * (TILE / 2);
  const int pairs = task.depth / 64;
  const int k_first = 2 * (int)((int64_t)pairs * part / splits), k_last = 2 * (int)((int64_t)pairs * (part + 1) / splits);
  // 32 x 32 tiles past the matrix are neither read nor stored (dimensions are whole multiples of 64: a wave has none, or full rows)
  auto there = [&](int i, int j) { return ti * TILE + row_p + 32 * i < task.rows && tj * TILE + row_q + 32 * j < task.cols; };
  Linear early{};                         // (of the smallest tile: under way during the product)
  if (MI * NI == 1 && STAGE != kGram && splits == 1 && there(0, 0)) early.read(task, ti * TILE + row_p, tj * TILE + row_q, lane);
  constexpr int kSums = Product<TILE>::kSums;
  typename Product<TILE>::Sums sums;
  f32x16 (&acc)[MI][NI] = sums[0];
#pragma unroll
  for (int t = 0; t < kSums; ++t)
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[t][i][j][e] = 0.f;
  if (k_first < k_last) g.run(sums, k_first, k_last - 1);         // (a matrix with fewer steps than parts: this part's sums are zeros)

  if constexpr (kSums == 3) {
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][0][e] += sums[1][0][0][e] + sums[2][0][0][e];
  }

  if (splits > 1) {
    float* to = jobs.partial + ((int64_t)(task.first + tile) * splits + part) * (TILE * TILE) + wave * (TILE * TILE / 4) + lane * 4;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<f32x4*>(to + ((i * NI + j) * 4 + e / 4) * 256) =
              f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
    return;
  }
  // Nobody reads the images any more: image 0 becomes the waves' turning areas.  The linear terms of a row of tiles are under way
  // while the row before is stored; straight-line code, so that waiting for them does not mean waiting for the stores behind them
  // (a loop over the tiles took 1.7 us for each: its head waited for everything).
  uint32_t* turn = reinterpret_cast<uint32_t*>(image<TILE, 0>()) + wave * kTurnWords;
  constexpr int kRows = TILE == 256 ? 1 : 2;          // (the largest tile has no registers left for a second row)
  f32x4* line = reinterpret_cast<f32x4*>(image<TILE, 1>() + wave * (2 * TILE * 128 / kWaves)) + lane;
  Linear linear[kRows][NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    linear[0][j] = early;
    if (MI * NI > 1 && STAGE != kGram && there(0, j)) linear[0][j].read(task, ti * TILE + row_p, tj * TILE + row_q + 32 * j, lane);
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    if (kRows == 1) {         // (its sums go through image 1, a row of tiles at a time: straight from the accumulators they spilled)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 4) line[(j * 4 + e / 4) * 64] = f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
      own_lds();
    }
#pragma unroll
    for (int j = 0; j < NI; ++j)
      if (kRows == 2 && i + 1 < MI && STAGE != kGram && there(i + 1, j))
        linear[(i + 1) % kRows][j].read(task, ti * TILE + row_p + 32 * (i + 1), tj * TILE + row_q + 32 * j, lane);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      f32x16 sum;
      if (kRows == 1) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 v = line[(j * 4 + g) * 64];
#pragma unroll
          for (int x = 0; x < 4; ++x) sum[4 * g + x] = v[x];
        }
      } else {
        sum = acc[i][j];
      }
      if (there(i, j))
        store_tile<STAGE>(task, end, ti * TILE + row_p + 32 * i, tj * TILE + row_q + 32 * j, STAGE > kPoly || ti != tj, sum,
                          linear[i % kRows][j], turn, lane);
      if (kRows == 1 && i + 1 < MI && STAGE != kGram && there(i + 1, j))
        linear[0][j].read(task, ti * TILE + row_p + 32 * (i + 1), tj * TILE + row_q + 32 * j, lane);
    }
  }
}

// Split products: the sums of a 32 x 32 tile's parts in order, one wave each.  `edge`: of the product's tiles.
template <int STAGE>
__global__ __launch_bounds__(256) void finish_kernel(Jobs jobs, typename EndOf<STAGE>::Args ends, int edge, int waves) {
  __shared__ __attribute__((aligned(16))) uint32_t turns[4][kTurnWords];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = blockIdx.x * 4 + wave;
  if (id >= waves) return;
  const int side = edge / 64, per_wave = side * side, per_tile = 4 * per_wave;      // (of a product wave: side x side tiles)
  const Task task = find(jobs, id, per_tile, lane);
  const auto end = EndOf<STAGE>::take(ends, task.which);
  const int local = id - task.first * per_tile, tile = local / per_tile, sub = local - tile * per_tile;
  const int of_wave = sub / per_wave, ij = sub - of_wave * per_wave, splits = jobs.splits;
  int ti, tj;
  tile_place<STAGE>(task, edge, tile, ti, tj);
  const int i0 = ti * edge + (of_wave >> 1) * (edge / 2) + 32 * (ij / side), j0 = tj * edge + (of_wave & 1) * (edge / 2) + 32 * (ij % side);
  if (i0 >= task.rows || j0 >= task.cols) return;
  const int64_t elems = (int64_t)edge * edge;
  const float* from = jobs.partial + (int64_t)(task.first + tile) * splits * elems + of_wave * (elems / 4) + ij * 1024 + lane * 4;
  Linear linear{};
  if (STAGE != kGram) linear.read(task, i0, j0, lane);
  f32x16 sum;
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.f;
  for (int s0 = 0; s0 < splits; s0 += 4) {
    f32x4 v[4][4];                         // (four parts requested together; past the end the last one again)
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int g = 0; g < 4; ++g) v[k][g] = *reinterpret_cast<const f32x4*>(from + min(s0 + k, splits - 1) * elems + g * 256);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[e] += s0 + k < splits ? v[k][e / 4][e % 4] : 0.f;
  }
  store_tile<STAGE>(task, end, i0, j0, STAGE > kPoly || ti != tj, sum, linear, turns[wave], lane);
}

// --- host ---------------------------------------------------------------------------------------------------------------
inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

constexpr int kMaxDim = 1 << 16;

bool bad_shapes(int count, const int32_t* rows, const int32_t* cols) {
  if (count < 1 || count > kMax || !rows || !cols) return true;
  for (int i = 0; i < count; ++i)
    if (rows[i] < 1 || cols[i] < 1 || rows[i] > kMaxDim || cols[i] > kMaxDim) return true;
  return false;
}

// How a stage's product is cut: tile edge and workgroups per tile (a range of k each).
struct Cut {
  int edge, splits;
};
struct StagePlan {
  Cut cut;
  int first[kMax + 1];      // first tile of every matrix
  int64_t partial_floats;
};

int64_t tiles_of(const Call& c, int i, int stage, int edge) {
  const int64_t tm = (c.item[i].mp + edge - 1) / edge, tn = (c.item[i].np + edge - 1) / edge;
  return stage <= kPoly ? tm * (tm + 1) / 2 : tm * tn;
}

thread_local int g_force_edge = 0, g_force_splits = 0;      // tuning (dtf_debug_set_muon_cut): of the calling thread's calls

// The cheapest cut by an estimate in microseconds.  By tile edge: a k-step with few and with all CUs at work (a full chip runs
// into its power limit: 1.3 PFLOP/s of fp16 products at 1.4 to 1.6 GHz, where a lone workgroup does a step at 96 % of the matrix
// rate at 2.4 GHz) and what a workgroup spends outside its steps, both measured.  One workgroup per CU at a time.  Long launches
// stay near the power limit even when some CUs have no work.  A split product pays a second launch and its sums' traffic.
// Against the choice, in us: 4096^2 x 4096 symmetric 192/1 178 (256/1 242, 128/1 233, 128/2 224); 4096^3 256/1 313 (192/1 345,
// 128/1 359, 64/1 472); 1024 x 4096 x 1024 128/1 33 (256/1 72, 64/1 44); 1024^2 x 1024 symmetric 64/1 11 (32/1 19,
// 128/4 19, 256/1 70); 512^2 x 832 symmetric 32/1 7.3 (64/1 9.9, 64/2 12, 128/2 16).
Cut choose(const Call& c, int stage) {
  static const struct { int edge; double step, loaded, rest; } kinds[] = {
      {256, 1.34, 2.3, 18.0}, {192, 0.755, 1.3, 11.5}, {128, 0.39, 0.65, 6.0}, {64, 0.175, 0.24, 2.0}, {32, 0.085, 0.12, 1.5}};
  Cut best{64, 1};
  double least = 1e300;
  int depth = 0;
  for (int i = 0; i < c.count; ++i) {
    const int d = stage == kGram ? c.item[i].np : c.item[i].mp;
    depth = d > depth ? d : depth;
  }
  for (const auto& kind : kinds) {
    if (g_force_edge && kind.edge != g_force_edge) continue;
    int64_t tiles = 0;
    for (int i = 0; i < c.count; ++i) tiles += tiles_of(c, i, stage, kind.edge);
    for (int s = 1; s <= 16; ++s) {
      if (g_force_splits && s != g_force_splits && s != 1) continue;
      if (s > 1 && (depth / 64 < 2 * s || kind.edge == 32)) break;
      const int64_t groups = tiles * s, full = groups / 256;
      const double steps = 2.0 * ((depth / 64 + s - 1) / s), share = (groups - full * 256) / 256.0;
      double us = 3.5 + full * (steps * kind.loaded + kind.rest);
      if (share > 0) {
        const bool lasting = us + steps * kind.loaded > 100;
        const double busy = kind.loaded * (lasting ? 0.45 + 0.55 * share : share);
        us += steps * (busy > kind.step ? busy : kind.step) + kind.rest;
      }
      if (s > 1) us += 3 + (double)groups * kind.edge * kind.edge * 8 / 8e6;
      if (g_force_splits && s == g_force_splits) us = 0;
      if (us < least) {
        least = us;
        best = Cut{kind.edge, s};
      }
    }
  }
  return best;
}

StagePlan plan_stage(const Call& c, int stage) {
  StagePlan r{};
  r.cut = choose(c, stage);
  int64_t at = 0;
  for (int i = 0; i < kMax; ++i) {
    r.first[i] = (int)at;
    if (i < c.count) at += tiles_of(c, i, stage, r.cut.edge);
  }
  r.first[kMax] = (int)at;
  r.partial_floats = r.cut.splits > 1 ? at * r.cut.splits * r.cut.edge * r.cut.edge : 0;
  return r;
}

struct Layout {
  int64_t total;
  StagePlan stage[3];
  float* partial;
};
// Fills the workspace part of `c` (from `base`, which may be null when only the size is asked for) and cuts the products.
Layout lay_out(Call& c, const int32_t* rows, const int32_t* cols, int count, char* base) {
  Layout l;
  c.count = count;
  int64_t at = 0, most = 0;
  auto take = [&](int64_t bytes) {
    char* p = base + at;
    at += up(bytes, 1024);
    return p;
  };
  for (int i = 0; i < count; ++i) {
    Item& it = c.item[i];
    it.rows = rows[i], it.cols = cols[i];
    it.flip = rows[i] > cols[i];
    it.m = it.flip ? cols[i] : rows[i];
    it.n = it.flip ? rows[i] : cols[i];
    it.mp = (int)up(it.m, 64), it.np = (int)up(it.n, 64);
    it.norm = reinterpret_cast<double*>(take(kNormBlocks * 8));
    const int64_t wide = (int64_t)it.mp * it.np * 4, square = (int64_t)it.mp * it.mp * 4;
    it.X = take(wide), it.XT[0] = take(wide), it.XT[1] = take(wide);
    it.A = take(square), it.B = take(square);
    const int64_t elements = (int64_t)rows[i] * cols[i];
    most = elements > most ? elements : most;
  }
  const int64_t blocks = (most + 2047) / 2048;           // eight elements a thread
  c.norm_blocks = (int)(blocks > kNormBlocks ? kNormBlocks : blocks);
  int64_t partial = 0;
  for (int stage = kGram; stage <= kStep; ++stage) {
    l.stage[stage] = plan_stage(c, stage);
    partial = l.stage[stage].partial_floats > partial ? l.stage[stage].partial_floats : partial;
  }
  l.partial = reinterpret_cast<float*>(take(partial * 4));
  l.total = at;
  return l;
}

template <int STAGE>
void launch_stage(const Call& c, const Layout& l, int parity, const typename EndOf<STAGE>::Args& ends, hipStream_t s) {
  const StagePlan& p = l.stage[STAGE == kLast ? kStep : STAGE];
  Jobs jobs{};
  jobs.partial = l.partial;
  jobs.splits = p.cut.splits;
  for (int i = 0; i < kMax; ++i) {
    Job& j = jobs.job[i];
    j.first = p.first[i], j.tiles = p.first[i + 1] - p.first[i];
    if (i >= c.count) continue;              // (behind every workgroup)
    const Item& it = c.item[i];
    j.p = STAGE == kGram ? it.X : STAGE == kPoly ? it.A : it.B;
    j.q = STAGE == kGram ? it.X : STAGE == kPoly ? it.A : it.XT[parity];
    j.linear = STAGE == kPoly ? it.A : it.XT[parity];
    j.straight = STAGE == kGram ? it.A : STAGE == kPoly ? it.B : it.X;
    j.turned = STAGE == kGram ? it.A : STAGE == kPoly ? it.B : it.XT[parity ^ 1];
    j.rows = it.mp;
    j.cols = STAGE <= kPoly ? it.mp : it.np;
    j.depth = STAGE == kGram ? it.np : it.mp;
  }
  const int edge = p.cut.edge, blocks = p.first[kMax] * p.cut.splits;
  switch (edge) {
    case 32: narrow_kernel<STAGE><<<blocks, 256, 0, s>>>(jobs, ends); break;
    case 64: product_kernel<64, STAGE><<<blocks, 256, 0, s>>>(jobs, ends); break;
    case 128: product_kernel<128, STAGE><<<blocks, 256, 0, s>>>(jobs, ends); break;
    case 192: product_kernel<192, STAGE><<<blocks, 256, 0, s>>>(jobs, ends); break;
    default: product_kernel<256, STAGE><<<blocks, 256, 0, s>>>(jobs, ends);
  }
  if (p.cut.splits > 1) {
    const int waves = p.first[kMax] * (edge / 32) * (edge / 32);
    finish_kernel<STAGE><<<(waves + 3) / 4, 256, 0, s>>>(jobs, ends, edge, waves);
  }
}

template <typename T>
int run(Call& c, const Layout& l, hipStream_t s) {
  norm_kernel<T><<<dim3(c.norm_blocks, c.count), 256, 0, s>>>(c);
  int64_t most = 0;
  for (int i = 0; i < c.count; ++i) {
    const int64_t t = (int64_t)(c.item[i].mp / 64) * (c.item[i].np / 64);
    most = t > most ? t : most;
  }
  split_kernel<T><<<dim3((unsigned)most, c.count), 256, 0, s>>>(c);
  Finals finals{};
  for (int i = 0; i < c.count; ++i) {
    const Item& it = c.item[i];
    finals.of[i] = Final{it.out, it.ldo, it.m, it.n, it.flip, it.shape_factor};
  }
  finals.lr = c.lr, finals.dtype = c.dtype;
  for (int k = 0; k < 5; ++k) {
    launch_stage<kGram>(c, l, k & 1, None{}, s);
    launch_stage<kPoly>(c, l, k & 1, None{}, s);
    if (k < 4) launch_stage<kStep>(c, l, k & 1, None{}, s);
    else launch_stage<kLast>(c, l, k & 1, finals, s);
  }
  return hipGetLastError() == hipSuccess ? DTF_OK : DTF_ERR_LAUNCH;
}

}  // namespace

extern "C" int64_t dtf_muon_workspace(int count, const int32_t* rows, const int32_t* cols) {
  if (bad_shapes(count, rows, cols)) return -1;
  Call c{};
  return lay_out(c, rows, cols, count, nullptr).total;
}

extern "C" int dtf_orthogonalize(const void* x, int dtype, int rows, int cols, int64_t ldx, void* out, int64_t ldo, float eps,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  const int32_t r = rows, k = cols;
  if (bad_shapes(1, &r, &k) || dtype < 0 || dtype > 2 || ldx < cols || ldo < cols || !(eps >= 0)) return DTF_ERR_SHAPE;
  if (!x || !out || !workspace) return DTF_ERR_NULL;
  Call c{};
  const Layout l = lay_out(c, &r, &k, 1, static_cast<char*>(workspace));
  if (workspace_bytes < l.total || ((uintptr_t)workspace & 255u)) return DTF_ERR_SHAPE;
  c.item[0].u = x, c.item[0].ldu = ldx, c.item[0].out = out, c.item[0].ldo = ldo;
  c.dtype = dtype, c.eps = eps;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DTF_F32) return run<float>(c, l, s);
  if (dtype == DTF_BF16) return run<bf16_t>(c, l, s);
  return run<f16_t>(c, l, s);
}

extern "C" int dtf_muon_step(int count, const int32_t* rows, const int32_t* cols, const uint64_t* w, const uint64_t* g,
                             const uint64_t* buf, const float* lr, float momentum, int nesterov, float eps, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (bad_shapes(count, rows, cols) || !(eps >= 0)) return DTF_ERR_SHAPE;
  if (!w || !g || !buf || !lr || !workspace) return DTF_ERR_NULL;
  Call c{};
  const Layout l = lay_out(c, rows, cols, count, static_cast<char*>(workspace));
  if (workspace_bytes < l.total || ((uintptr_t)workspace & 255u)) return DTF_ERR_SHAPE;
  for (int i = 0; i < count; ++i) {
    if (!w[i] || !g[i] || !buf[i]) return DTF_ERR_NULL;
    Item& it = c.item[i];
    it.u = reinterpret_cast<const void*>(g[i]), it.ldu = cols[i];
    it.buf = reinterpret_cast<float*>(buf[i]);
    it.out = reinterpret_cast<void*>(w[i]), it.ldo = cols[i];
    it.shape_factor = cols[i] > rows[i] ? sqrtf((float)cols[i] / (float)rows[i]) : 1.f;
  }
  c.mu = momentum, c.nesterov = nesterov, c.eps = eps, c.lr = lr;
  return run<float>(c, l, (hipStream_t)stream);
}

// Tuning and tests: products of this thread's next calls in tiles of this edge (32, 64, 128, 192, 256) with this many parts of k where k is long
// enough; 0: chosen from the shapes.  (The workspace of a plan has to be made under the same setting.)
extern "C" void dtf_debug_set_muon_cut(int edge, int splits) {
  g_force_edge = edge == 32 || edge == 64 || edge == 128 || edge == 192 || edge == 256 ? edge : 0;
  g_force_splits = splits > 0 && splits <= 16 ? splits : 0;
}
