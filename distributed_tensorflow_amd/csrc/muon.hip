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
// Every matrix is therefore kept as TWO fp16 planes, hi + lo = the value times a power of two of its row: 22 significant bits, fewer
// only below 2^-16 of the largest entry that the row may have (see Scales).  A product is three fp16 MFMAs, hi hi + hi lo + lo hi,
// summed in fp32; what is dropped, lo lo, is 2^-22 of the product, less than the rounding of an fp32 sum of a few terms.
// Simulated and measured, the result is as far from the 64-bit iteration as that of fp32 matrix products, as a whole and in rows and
// columns of 10^-14 of the others (the fp32 sums dominate both; 256 x 512 with half the rows at 10^-9: 1.9e-7 of those rows,
// 3.5e-7 in fp32).  (Iterating in the m x m space of the Gram matrix needs fewer flops for n > m but squares the condition: 5 to 16
// times the error on gradients with a decaying spectrum; not used.)
//
// Layout.  Both operands of every product are read along k: A = X X^T takes rows of X twice, A A takes rows of the symmetric
// A, B X takes rows of B and rows of X^T.  So X is kept together with its transpose, each step's product writes both, and one
// GEMM form (row times row) serves all.  The linear terms a X and b A are read as fp32 (see Linear).  A row of a plane pair is
// groups of 32 columns: 32 hi halves then 32 lo halves, 128 bytes, one cache line per row and k-step.  Dimensions are padded with
// zeros to whole tiles: the products need no bounds.
//
// GEMM.  A workgroup of four waves owns a square tile of 64, 128, 192 or 256 (or 32, see Narrow) and walks k in steps of 32 through a
// ring of 8, 4, 3 or 2 LDS images filled by direct buffer-to-LDS loads: 148, 132, 144 or 128 KB (ring_bytes()), one workgroup per
// CU, the loads of a step requested one to seven steps ahead of it (the matrices come from the other XCDs' writes: 0.8 us away,
// against 0.1 to 1.8 us of products per step).  A load instruction moves eight 128-byte rows; its LDS side is fixed (lane l at
// 16 l), so the 16-byte chunks of a row are permuted on the GLOBAL side: slot s of row r holds chunk s ^ ((r >> 1) & 7), and the
// sixteen rows that a quarter of a fragment read touches fill all 64 banks once (rows r and r + 1 lie in the two halves of the
// banks; measured: no conflict).
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

#include <algorithm>

namespace {

typedef f16_t half8 __attribute__((ext_vector_type(8)));
typedef f16_t half2 __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kMax = DTF_MUON_MAX;
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScaleX = 32768.f, kScaleA = 16384.f, kScaleB = 8192.f;    // powers of two: entries stay below 65504
constexpr int kParts = 16;            // of the rows, and of the columns, for the norm and the maxima (see lay_out())
constexpr int kBlocks = kParts * kParts;
constexpr int kMaxDim = 1 << 16;
constexpr int kNormThreads = 1024;
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
  float *d, *e;         // scales of the m rows and the n columns (see Scales)
  float *linear_a, *linear_x;     // A without its scales and X, fp32 (see Linear)
  int edge_r, edge_c, parts_r, parts_c;      // parts of the matrix for the norm and the maxima
  double* norm;         // [parts_r][parts_c]: sums of squares
  float *row_max, *col_max;       // [parts_c][padded rows], [parts_r][padded columns]: largest magnitudes
};

struct Call {
  Item item[kMax];
  int count, dtype;
  float mu, eps;
  int nesterov;
  const float* lr;
};

// --- momentum, norm and scales ------------------------------------------------------------------------------------------
// The largest of a row of sixteen lanes, in each of them.
template <int ROTATE>
__device__ __forceinline__ float most_of_rotated(float v) {
  const int other = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + ROTATE, 15, 15, false);      // row_ror
  return fmaxf(v, __builtin_bit_cast(float, other));
}
__device__ __forceinline__ float most_of_16(float v) {
  return most_of_rotated<1>(most_of_rotated<2>(most_of_rotated<4>(most_of_rotated<8>(v))));
}

// A part of the matrix per block, 64 rows of 256 columns at a time, four quads a thread: the momentum, the sum of squares, and the
// largest magnitude of every row and column (exact, so that their order does not matter).  (4096 x 4096: 41 us, 4.9 TB/s; the maxima
// cost 8 of them.)
template <typename T>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(Call c) {
  const Item& it = c.item[blockIdx.y];
  if ((int)blockIdx.x >= it.parts_r * it.parts_c) return;
  __shared__ uint32_t row_max[kMaxDim / kParts], col_max[kMaxDim / kParts];
  __shared__ double of_wave[kNormThreads / 64];
  const int part_r = blockIdx.x / it.parts_c, part_c = blockIdx.x - part_r * it.parts_c;
  const int r0 = part_r * it.edge_r, c0 = part_c * it.edge_c;
  const int r1 = min(r0 + it.edge_r, it.rows), c1 = min(c0 + it.edge_c, it.cols);
  for (int i = threadIdx.x; i < it.edge_r; i += kNormThreads) row_max[i] = 0;
  for (int i = threadIdx.x; i < it.edge_c; i += kNormThreads) col_max[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63, row = threadIdx.x >> 4;
  // whole quads where every row is aligned
  const bool aligned = it.ldu % 4 == 0 && (reinterpret_cast<uintptr_t>(it.u) % (4 * sizeof(T))) == 0 &&
                       (!it.buf || (it.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(it.buf) & 15u) == 0));
  double sum = 0;
  constexpr int U = 4;                         // quads of a row under way
  for (int c_first = c0; c_first < c1; c_first += 64 * U) {
    const int cs = c_first + 4 * (threadIdx.x & 15);
    f32x4 top[U];
#pragma unroll
    for (int k = 0; k < U; ++k) top[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int r = r0 + row; r - row < r1; r += 64) {
      const T* u = static_cast<const T*>(it.u) + r * it.ldu;
      float* m = it.buf + (int64_t)r * it.cols;
      f32x4 g[U], b[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        g[k] = b[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int col = cs + 64 * k;
        if (r >= r1) continue;
        if (aligned && col + 4 <= c1) {
          const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4>*>(u + col);
#pragma unroll
          for (int e = 0; e < 4; ++e) g[k][e] = (float)p.v[e];
          if (it.buf) b[k] = *reinterpret_cast<const f32x4*>(m + col);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < c1) {
              g[k][e] = (float)u[col + e];
              if (it.buf) b[k][e] = m[col + e];
            }
        }
      }
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int col = cs + 64 * k;
        f32x4 v = g[k];
        if (it.buf && r < r1) {
          const f32x4 now = c.mu * b[k] + g[k];
          if (aligned && col + 4 <= c1) {
            *reinterpret_cast<f32x4*>(m + col) = now;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < c1) m[col + e] = now[e];
          }
          v = c.nesterov ? g[k] + c.mu * now : now;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum += (double)v[e] * (double)v[e];
          top[k][e] = fmaxf(top[k][e], fabsf(v[e]));
          most = fmaxf(most, fabsf(v[e]));
        }
      }
      most = most_of_16(most);
      if ((lane & 15) == 0 && r < r1) atomicMax(&row_max[r - r0], __builtin_bit_cast(uint32_t, most));
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (c_first + 64 * k >= c1) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = cs + 64 * k + e;
        const float most = top[k][e];      // (a bit cast of a vector's element is one of its first element)
        if (col < c1) atomicMax(&col_max[col - c0], __builtin_bit_cast(uint32_t, most));
      }
    }
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x);
  if (lane == 0) of_wave[threadIdx.x >> 6] = sum;
  __syncthreads();
  const int pr = it.flip ? it.np : it.mp, pc = it.flip ? it.mp : it.np;       // padded rows and columns as the caller has them
  for (int i = threadIdx.x; i < min(it.edge_r, pr - r0); i += kNormThreads)
    it.row_max[(int64_t)part_c * pr + r0 + i] = __builtin_bit_cast(float, row_max[i]);
  for (int i = threadIdx.x; i < min(it.edge_c, pc - c0); i += kNormThreads)
    it.col_max[(int64_t)part_r * pc + c0 + i] = __builtin_bit_cast(float, col_max[i]);
  if (threadIdx.x == 0) {
    double total = 0;
    for (int w = 0; w < kNormThreads / 64; ++w) total += of_wave[w];
    it.norm[blockIdx.x] = total;
  }
}

// Smallest power of two that is not below v, from 2^-100 to 1.
__device__ __forceinline__ float scale_above(float v) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, fminf(fmaxf(v, 0x1p-100f), 1.f));
  return __builtin_bit_cast(float, (bits + 0x7fffffu) & 0xff800000u);
}
// 1 / v of such a power of two.
__device__ __forceinline__ float reciprocal(float v) { return __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(uint32_t, v)); }

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
// A 64 x 64 tile of values in LDS, its rows `line` and its columns `step` words apart and each row times its `scale`, to row0, col0
// of a plane pair: 256 bytes a row, sixteen bytes a thread and turn, consecutive threads one behind the other (64 bytes a thread:
// the kernel took 23 us for 1024 x 4096 instead of 17).
__device__ __forceinline__ void store_tile(char* plane, int row0, int col0, int cols, const float* values, int line, int step,
                                           const float* scale) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int row = k * 16 + (threadIdx.x >> 4), chunk = threadIdx.x & 15;      // chunk: group of 32 columns, hi or lo, 8 columns
    const int col = (chunk >> 3) * 32 + (chunk & 3) * 8, shift = (chunk >> 2 & 1) * 16;
    const float f = scale[row];
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* at = values + row * line + (col + 2 * e) * step;
      w[e] = (split_pair(at[0] * f) >> shift & 0xffffu) | (split_pair(at[step] * f) >> shift) << 16;
    }
    *reinterpret_cast<u32x4*>(plane + plane_at(row0 + row, col0, cols) + chunk * 16) = w;
  }
}

// X of U / (|U| + eps) as planes, turned and straight, and in fp32, and the scales: 64 x 64 tiles of the padded shape.
template <typename T>
__global__ __launch_bounds__(256) void split_kernel(Call c) {
  __shared__ float tile[64][65];
  __shared__ double of_wave[4];
  __shared__ float most[2][4][64], to[2][64];         // of the rows, of the columns
  const Item& it = c.item[blockIdx.y];
  const int pr = it.flip ? it.np : it.mp, pc = it.flip ? it.mp : it.np;       // padded rows and columns as the caller has them
  const int tiles_c = pc / 64, tiles = (pr / 64) * tiles_c;
  if ((int)blockIdx.x >= tiles) return;
  const int r0 = (blockIdx.x / tiles_c) * 64, c0 = (blockIdx.x % tiles_c) * 64;
  const int col = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // All requests at once and before the norm is added up, from clamped places: one by one they took 15 us.
  const T* gp = static_cast<const T*>(it.u) + min(c0 + col, it.cols - 1);
  const float* bp = it.buf + min(c0 + col, it.cols - 1);
  float u[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) u[k] = (float)gp[(int64_t)min(r0 + wave + 4 * k, it.rows - 1) * it.ldu];
  float b[16];
  if (it.buf) {
#pragma unroll
    for (int k = 0; k < 16; ++k) b[k] = bp[(int64_t)min(r0 + wave + 4 * k, it.rows - 1) * it.cols];
  }
  const int parts = it.parts_r * it.parts_c;
  double total = it.norm[min((int)threadIdx.x, parts - 1)];
  float row_top = 0.f, col_top = 0.f;                 // (the last part again past the end)
  for (int p = wave; p < max(it.parts_r, it.parts_c); p += 16)
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      row_top = fmaxf(row_top, it.row_max[(int64_t)min(p + k, it.parts_c - 1) * pr + r0 + col]);
      col_top = fmaxf(col_top, it.col_max[(int64_t)min(p + k, it.parts_r - 1) * pc + c0 + col]);
    }
  if ((int)threadIdx.x >= parts) total = 0.0;
  if (it.buf) {
#pragma unroll
    for (int k = 0; k < 16; ++k) u[k] = c.nesterov ? u[k] + c.mu * b[k] : b[k];
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) total += __shfl_xor(total, x);
  if (col == 0) of_wave[wave] = total;
  most[0][wave][col] = row_top;
  most[1][wave][col] = col_top;
  __syncthreads();
  const double length = sqrt((of_wave[0] + of_wave[1]) + (of_wave[2] + of_wave[3])) + (double)c.eps;
  const double inv = length == 0.0 ? 0.0 : 1.0 / length;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = wave + 4 * k;
    tile[r][col] = r0 + r < it.rows && c0 + col < it.cols ? (float)((double)u[k] * inv) : 0.f;
  }
  if (wave < 2) {                        // the scales of the tile's rows (wave 0) and columns
    const float top = fmaxf(fmaxf(most[wave][0][col], most[wave][1][col]), fmaxf(most[wave][2][col], most[wave][3][col]));
    const float s = scale_above((float)((double)top * inv * (double)sqrtf((float)(wave ? it.rows : it.cols))));
    to[wave][col] = kScaleX * reciprocal(s);
    float* const scales = (wave == 1) != (it.flip != 0) ? it.e : it.d;
    if ((wave ? r0 : c0) == 0) scales[(wave ? c0 : r0) + col] = s;
  }
  __syncthreads();
  char* straight = it.flip ? it.XT[0] : it.X;          // [pr][pc]
  char* turned = it.flip ? it.X : it.XT[0];            // [pc][pr]
  store_tile(straight, r0, c0, pc, &tile[0][0], 65, 1, to[0]);
  store_tile(turned, c0, r0, pr, &tile[0][0], 1, 65, to[1]);
  // (block by block as Linear reads them)
  const int i0 = it.flip ? c0 : r0, j0 = it.flip ? r0 : c0, lane = threadIdx.x & 63, g = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f32x4 v;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = 32 * (k >> 1) + 8 * g + 4 * (lane >> 5) + x, j = 32 * (k & 1) + (lane & 31);
      v[x] = it.flip ? tile[j][i] : tile[i][j];
    }
    *reinterpret_cast<f32x4*>(it.linear_x + ((int64_t)(i0 / 32 + (k >> 1)) * (it.np / 32) + j0 / 32 + (k & 1)) * 1024 + g * 256 + lane * 4) = v;
  }
}

// --- products -----------------------------------------------------------------------------------------------------------
enum Stage { kGram = 0, kPoly = 1, kStep = 2, kLast = 3 };     // A = X X^T;  B = bA + cAA;  X = aX + BX;  the same, to the output

// What the launches of a stage read beside the planes themselves: 64 bytes a matrix, 512 for all of them, so that one load
// instruction brings them into a wave's registers, whichever its matrix is (see find()).
struct Job {
  const char *p, *q;          // the operands: rows of k
  char* linear;               // of the linear term: A (written by kGram), or X (kStep writes the next one in its place)
  char *straight, *turned;    // the result, and its transpose
  int rows, cols, depth;      // of the product, padded
  int first, tiles;           // first tile and number of tiles
  int spare;
  // The scales lie in front of the linear terms: those of the columns, those of the rows, A, X.
  __host__ __device__ static int64_t scale_bytes(int count) { return ((int64_t)count * 4 + 1023) / 1024 * 1024; }
  __device__ __forceinline__ const float* row_scales(bool symmetric) const {
    return reinterpret_cast<const float*>(linear - (symmetric ? 0 : (int64_t)rows * rows * 4) - scale_bytes(rows));
  }
  __device__ __forceinline__ const float* col_scales(bool symmetric) const {
    const float* d = row_scales(symmetric);
    return symmetric ? d : reinterpret_cast<const float*>(reinterpret_cast<const char*>(d) - scale_bytes(cols));
  }
};
static_assert(sizeof(Job) == 64, "find() counts words");
struct Jobs {
  Job job[kMax];
  float* partial;             // split products: [tile][split][elements of a tile]
  int splits;                 // workgroups per tile, a range of k each
  float growth;               // of the scales up to this iteration (see Scales)
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

// The linear term of a tile in fp32, as the sums lie in the registers: 4 KB a tile, whole lines in either direction.
struct Linear {
  f32x4 v[4];
  static __device__ __forceinline__ f32x4* at(const Task& t, int i0, int j0, int lane) {
    return reinterpret_cast<f32x4*>(t.linear) + ((int64_t)(i0 >> 5) * (t.cols >> 5) + (j0 >> 5)) * 256 + lane;
  }
  __device__ __forceinline__ void read(const Task& t, int i0, int j0, int lane) {
    const f32x4* from = at(t, i0, j0, lane);
#pragma unroll
    for (int g = 0; g < 4; ++g) v[g] = from[64 * g];
  }
};

// Scales.  Row i of X is kept divided by d_i and column j (a row of X^T) by e_j, powers of two that are not below their norms (the
// largest magnitude times the root of the length, rounded up); rows of A and B are divided by d_i too.  So an entry has its 22 bits
// relative to its own row, however little that is next to the others.  (One scale for the whole matrix: rows of 10^-6 of the
// others were 400 times as far off as in fp32, nothing was left of rows of 10^-10.  It took 128 us for the stack of three matrices
// instead of 132, 365 for 1024 x 4096 instead of 385, 3.52 ms for a step of 4096 x 4096 instead of 3.64: X in fp32 is 4 bytes an
// element more to write in each step.)  No product needs more than that: with P = D^-1 X, R = D^-1 A, S = D^-1 B and T = E^-1 X^T,
//   A = D (P P^T) D,   A A = D (R R^T) D,   B X = D (S T^T) E,
// so the scales meet the sums at a product's end alone.  The linear terms carry no scale of one side: A is kept as D^-1 A D^-1
// and X as it is, in fp32.  A step multiplies no singular value by more than 3.4445, and so no row's or column's norm: the scales
// grow by 4 with each step, up to 1.  |P|, |T| <= 1.2, |R| <= 1.45, |S| <= 1.2 * 2.83 by the quintic.
struct Scales {               // of a tile's rows and columns, in LDS
  const float *row, *row_to;  // the scale, and kScaleX over the next step's
  const float *col, *col_to;
};
__device__ __forceinline__ float scale_now(float first, float growth) { return fminf(first * growth, 1.f); }
__device__ __forceinline__ float scale_to(float first, float growth) { return kScaleX * reciprocal(fminf(first * (4.f * growth), 1.f)); }

// Value times scale as hi and lo, two rows at a time.
__device__ __forceinline__ void split_rows(const f32x4 (&v)[4], half2 (&hi)[8], half2 (&lo)[8]) {
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const float2v x = {v[p / 2][2 * (p & 1)], v[p / 2][2 * (p & 1) + 1]};
    hi[p] = __builtin_convertvector(x, half2);
    lo[p] = __builtin_convertvector(x - __builtin_convertvector(hi[p], float2v), half2);
  }
}

// What becomes of the tile.  `area`: the wave's turning areas.  `mirror`: also store the transposed tile of a symmetric result.
template <int STAGE>
__device__ __forceinline__ void store_tile(const Task& t, const typename EndOf<STAGE>::Mine& end, int i0, int j0, bool mirror,
                                           const f32x16& sum, const Linear& linear, const Scales& scales, uint32_t* area, int lane) {
  const int half = lane >> 5, jc = lane & 31;
  uint32_t* turn = area;
  uint32_t* lines = area + 32 * kTurnRow;
  f32x4 v[4], row[4];
  const float col = scales.col[jc];
#pragma unroll
  for (int g = 0; g < 4; ++g) row[g] = *reinterpret_cast<const f32x4*>(scales.row + 8 * g + 4 * half);
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float s = sum[4 * g + x];
      v[g][x] = STAGE == kGram   ? s * (1.f / (kScaleX * kScaleX))
                : STAGE == kPoly ? fmaf(kB, linear.v[g][x], s * (kC / (kScaleA * kScaleA)))
                                 : fmaf(kA, linear.v[g][x], s * (row[g][x] * (1.f / (kScaleB * kScaleX))) * col);
    }
  if constexpr (STAGE == kLast) {
    const Final& it = end.f;
    // (places past the matrix are read as its last ones and not stored)
    const int64_t step_row = it.flip ? 1 : it.ld, step_col = it.flip ? it.ld : 1;
    const int row0 = i0 + 4 * half, at_j = j0 + jc;
    const int64_t at_col = min(at_j, it.n - 1) * step_col;
    auto place = [&](int e) { return min(row0 + 8 * (e / 4) + e % 4, it.m - 1) * step_row + at_col; };
    auto inside = [&](int e) { return row0 + 8 * (e / 4) + e % 4 < it.m && at_j < it.n; };
    if (end.lr || end.dtype == DTF_F32) {
      float* out = static_cast<float*>(it.out);
      if (end.lr) {                       // the weights: all of them requested before the first store
        const float step_size = end.lr[0] * it.shape_factor;
        float old[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) old[e] = out[place(e)];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e / 4][e % 4] = old[e] - step_size * v[e / 4][e % 4];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (inside(e)) out[place(e)] = v[e / 4][e % 4];
    } else {
      uint16_t* out = static_cast<uint16_t*>(it.out);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = v[e / 4][e % 4];
        const uint16_t bits = end.dtype == DTF_BF16 ? __builtin_bit_cast(uint16_t, (bf16_t)x) : __builtin_bit_cast(uint16_t, (f16_t)x);
        if (inside(e)) out[place(e)] = bits;
      }
    }
    return;
  }
  if (STAGE != kPoly) {
    f32x4* to = Linear::at(t, i0, j0, lane);
#pragma unroll
    for (int g = 0; g < 4; ++g) to[64 * g] = v[g];
  }
  half2 hi[8], lo[8];
  f32x4 w[4];
  constexpr float kSquare = STAGE == kGram ? kScaleA : kScaleB;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    w[g] = STAGE <= kPoly ? v[g] * (col * kSquare) : v[g] * *reinterpret_cast<const f32x4*>(scales.row_to + 8 * g + 4 * half);
  split_rows(w, hi, lo);
  f16_t* at = reinterpret_cast<f16_t*>(turn + 4 * half * kTurnRow) + jc;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    at[(8 * (e / 4) + e % 4) * 2 * kTurnRow] = hi[e / 2][e % 2];
    at[(8 * (e / 4) + e % 4) * 2 * kTurnRow + 32] = lo[e / 2][e % 2];
  }
  if (mirror) {
    // Line j of the transposed tile: this lane has rows 4 half .. 4 half + 3 of every eight, the lane 32 away the other four.
    // Exchanged between two groups of eight, each lane holds whole chunks.
    const float col_to = STAGE <= kPoly ? 0.f : scales.col_to[jc];
#pragma unroll
    for (int g = 0; g < 4; ++g) w[g] = STAGE <= kPoly ? v[g] * (row[g] * kSquare) : v[g] * col_to;
    split_rows(w, hi, lo);
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

// A wave's tile of 32: its scales to LDS (`at`, 128 words of the wave's own).  Lanes 0 .. 31 have read a row's, the others a
// column's (see read_scale).
template <int STAGE>
__device__ __forceinline__ float read_scale(const Task& t, int i0, int j0, int lane) {
  return lane < 32 ? t.row_scales(STAGE <= kPoly)[i0 + lane] : t.col_scales(STAGE <= kPoly)[j0 + lane - 32];
}
__device__ __forceinline__ Scales lay_scales(float first, float growth, float* at, int lane) {
  at[lane] = scale_now(first, growth);
  at[64 + lane] = scale_to(first, growth);
  own_lds();
  return Scales{at, at + 64, at + 32, at + 96};
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
              "a CU has 160 KB, and up to 4 KB are for the scales of a tile");

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
  float scale = 0.f;
  if (wave == 0) scale = read_scale<STAGE>(task, ti * 32, tj * 32, lane);
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
  const Scales scales = lay_scales(scale, jobs.growth, reinterpret_cast<float*>(image<128, 2>()), lane);
  store_tile<STAGE>(task, end, ti * 32, tj * 32, STAGE > kPoly || ti != tj, sum, linear, scales, reinterpret_cast<uint32_t*>(image<128, 0>()), lane);
}

template <int TILE, int STAGE>
__global__ __launch_bounds__(kWaves * 64, 1) void product_kernel(Jobs jobs, typename EndOf<STAGE>::Args all_ends) {
  __shared__ __attribute__((aligned(16))) float scale_of[4][TILE];      // rows and columns: the scales, kScaleX over the next ones
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
  // 32 x 32 tiles past the matrix are neither read nor stored (dimensions are whole multiples of 64: a wave has none, or full rows),
  // nor those below the diagonal of a symmetric result, which are stored with their mirror images
  auto there = [&](int i, int j) {
    const int i0 = ti * TILE + row_p + 32 * i, j0 = tj * TILE + row_q + 32 * j;
    return i0 < task.rows && j0 < task.cols && (STAGE > kPoly || i0 <= j0);
  };
  float row_scale = 0.f, col_scale = 0.f;
  if (threadIdx.x < TILE && splits == 1) {
    row_scale = task.row_scales(STAGE <= kPoly)[min(ti * TILE + (int)threadIdx.x, task.rows - 1)];
    col_scale = task.col_scales(STAGE <= kPoly)[min(tj * TILE + (int)threadIdx.x, task.cols - 1)];
  }
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
  if (threadIdx.x < TILE) {
    scale_of[0][threadIdx.x] = scale_now(row_scale, jobs.growth);
    scale_of[1][threadIdx.x] = scale_to(row_scale, jobs.growth);
    scale_of[2][threadIdx.x] = scale_now(col_scale, jobs.growth);
    scale_of[3][threadIdx.x] = scale_to(col_scale, jobs.growth);
  }
  __syncthreads();
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
      if (there(i, j)) {
        const int i0 = ti * TILE + row_p + 32 * i, j0 = tj * TILE + row_q + 32 * j, in_p = row_p + 32 * i, in_q = row_q + 32 * j;
        store_tile<STAGE>(task, end, i0, j0, STAGE > kPoly || i0 != j0, sum, linear[i % kRows][j],
                          Scales{scale_of[0] + in_p, scale_of[1] + in_p, scale_of[2] + in_q, scale_of[3] + in_q}, turn, lane);
      }
      if (kRows == 1 && i + 1 < MI && STAGE != kGram && there(i + 1, j))
        linear[0][j].read(task, ti * TILE + row_p + 32 * (i + 1), tj * TILE + row_q + 32 * j, lane);
    }
  }
}

// Split products: the sums of a 32 x 32 tile's parts in order, one wave each.  `edge`: of the product's tiles.
template <int STAGE>
__global__ __launch_bounds__(256) void finish_kernel(Jobs jobs, typename EndOf<STAGE>::Args ends, int edge, int waves) {
  __shared__ __attribute__((aligned(16))) uint32_t turns[4][kTurnWords];
  __shared__ __attribute__((aligned(16))) float scale_of[4][128];
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
  if (i0 >= task.rows || j0 >= task.cols || (STAGE <= kPoly && i0 > j0)) return;
  const int64_t elems = (int64_t)edge * edge;
  const float* from = jobs.partial + (int64_t)(task.first + tile) * splits * elems + of_wave * (elems / 4) + ij * 1024 + lane * 4;
  Linear linear{};
  const float scale = read_scale<STAGE>(task, i0, j0, lane);
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
  store_tile<STAGE>(task, end, i0, j0, STAGE > kPoly || i0 != j0, sum, linear, lay_scales(scale, jobs.growth, scale_of[wave], lane),
                    turns[wave], lane);
}

// --- host ---------------------------------------------------------------------------------------------------------------
inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

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
  int64_t at = 0;
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
    // Parts of whole tiles of 64: kBlocks at most, up to 64 of the rows of a narrow matrix or the columns of a flat one.  (Every
    // tile of split_kernel reads the maxima of all parts of its rows and columns.)
    const int tiles_r = (rows[i] + 63) / 64, tiles_c = (cols[i] + 63) / 64;
    const int most_r = std::max(kParts, std::min(64, kBlocks / tiles_c)), most_c = std::max(kParts, std::min(64, kBlocks / tiles_r));
    it.edge_r = (int)up((rows[i] + most_r - 1) / most_r, 64), it.edge_c = (int)up((cols[i] + most_c - 1) / most_c, 64);
    it.parts_r = (rows[i] + it.edge_r - 1) / it.edge_r, it.parts_c = (cols[i] + it.edge_c - 1) / it.edge_c;
    it.norm = reinterpret_cast<double*>(take(kBlocks * 8));
    it.row_max = reinterpret_cast<float*>(take((int64_t)it.parts_c * up(rows[i], 64) * 4));
    it.col_max = reinterpret_cast<float*>(take((int64_t)it.parts_r * up(cols[i], 64) * 4));
    const int64_t wide = (int64_t)it.mp * it.np * 4, square = (int64_t)it.mp * it.mp * 4;
    it.X = take(wide), it.XT[0] = take(wide), it.XT[1] = take(wide);
    it.A = take(square), it.B = take(square);
    it.e = reinterpret_cast<float*>(take(Job::scale_bytes(it.np)));        // (in this order: see Job)
    it.d = reinterpret_cast<float*>(take(Job::scale_bytes(it.mp)));
    it.linear_a = reinterpret_cast<float*>(take(square)), it.linear_x = reinterpret_cast<float*>(take(wide));
  }
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
void launch_stage(const Call& c, const Layout& l, int iteration, const typename EndOf<STAGE>::Args& ends, hipStream_t s) {
  const int parity = iteration & 1;
  const StagePlan& p = l.stage[STAGE == kLast ? kStep : STAGE];
  Jobs jobs{};
  jobs.partial = l.partial;
  jobs.splits = p.cut.splits;
  jobs.growth = (float)(1 << 2 * iteration);
  for (int i = 0; i < kMax; ++i) {
    Job& j = jobs.job[i];
    j.first = p.first[i], j.tiles = p.first[i + 1] - p.first[i];
    if (i >= c.count) continue;              // (behind every workgroup)
    const Item& it = c.item[i];
    j.p = STAGE == kGram ? it.X : STAGE == kPoly ? it.A : it.B;
    j.q = STAGE == kGram ? it.X : STAGE == kPoly ? it.A : it.XT[parity];
    j.linear = reinterpret_cast<char*>(STAGE <= kPoly ? it.linear_a : it.linear_x);
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
  int64_t most = 0;
  int parts = 0;
  for (int i = 0; i < c.count; ++i) {
    const int64_t t = (int64_t)(c.item[i].mp / 64) * (c.item[i].np / 64);
    most = t > most ? t : most;
    parts = std::max(parts, c.item[i].parts_r * c.item[i].parts_c);
  }
  norm_kernel<T><<<dim3(parts, c.count), kNormThreads, 0, s>>>(c);
  split_kernel<T><<<dim3((unsigned)most, c.count), 256, 0, s>>>(c);
  Finals finals{};
  for (int i = 0; i < c.count; ++i) {
    const Item& it = c.item[i];
    finals.of[i] = Final{it.out, it.ldo, it.m, it.n, it.flip, it.shape_factor};
  }
  finals.lr = c.lr, finals.dtype = c.dtype;
  for (int k = 0; k < 5; ++k) {
    launch_stage<kGram>(c, l, k, None{}, s);
    launch_stage<kPoly>(c, l, k, None{}, s);
    if (k < 4) launch_stage<kStep>(c, l, k, None{}, s);
    else launch_stage<kLast>(c, l, k, finals, s);
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
