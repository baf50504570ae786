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
// GEMM.  A workgroup owns a tile and walks k in steps of 32 through two LDS images filled by direct global-to-LDS loads (the
// load of step k + 1 is in flight while step k is multiplied; one barrier per step).  A load instruction moves eight 128-byte rows;
// its LDS side is fixed (lane l at 16 l), so the 16-byte chunks of a row are permuted on the GLOBAL side: slot s of row r holds
// chunk s ^ (r & 7), and the 32 rows a fragment read touches spread over all banks.  Few tiles and a long k: several
// workgroups split the k range of a tile and the last to arrive adds the partial sums in their order.
//
// All matrices of a call go through each launch together: 2 + 15 launches per step of the optimiser, whatever the number of
// layers (up to 8; more are taken in groups).
#include "dtf_api.h"
#include "dtf_types.h"

namespace {

typedef f16_t half8 __attribute__((ext_vector_type(8)));
typedef f16_t half4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kMax = DTF_MUON_MAX;
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScaleX = 32768.f, kScaleA = 16384.f, kScaleB = 8192.f;    // powers of two: entries stay below 65504
constexpr int kNormBlocks = 128;
constexpr int kMaxTickets = 4096;

// One matrix of a call.  `rows` x `cols` as the caller has it; m <= n its shape (or its transpose's) padded to mp x np.
struct Item {
  const void* u;        // G, or the matrix to orthogonalise
  float* buf;           // momentum (null: orthogonalise u itself)
  void* out;            // W (updated) or the result
  int64_t ldu, ldo;
  int rows, cols, m, n, mp, np, flip;
  float shape_factor;   // sqrt(max(1, cols / rows))
  char *X, *XT[2], *A, *B;
  double* norm;         // [kNormBlocks] partial sums of squares
};

struct Call {
  Item item[kMax];
  int count, dtype;
  float mu, eps;
  int nesterov;
  const float* lr;
  uint32_t* tickets;
  float* partial;       // split products: [tile][split][elements of a tile]
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
  if (blockIdx.y == 0)
    for (int i = blockIdx.x * 256 + threadIdx.x; i < kMaxTickets; i += kNormBlocks * 256) c.tickets[i] = 0;
  const int64_t total = (int64_t)it.rows * it.cols;
  double sum = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += kNormBlocks * 256) {
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
// 32 pairs, `step` words apart in LDS, to the hi (part 0) or lo (part 1) half of a 128-byte group.
__device__ __forceinline__ void store_group(char* group, const uint32_t* pairs, int step, int part) {
  const int shift = part * 16;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = ((pairs[(8 * q + 2 * e) * step] >> shift) & 0xffffu) | ((pairs[(8 * q + 2 * e + 1) * step] >> shift) << 16);
    *reinterpret_cast<uint4*>(group + part * 64 + q * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// X and X^T of U / (|U| + eps), 64 x 64 tiles of the padded shape.
template <typename T>
__global__ __launch_bounds__(256) void split_kernel(Call c) {
  __shared__ uint32_t tile[64][65];
  __shared__ double inv_s;
  const Item& it = c.item[blockIdx.y];
  const int pr = it.flip ? it.np : it.mp, pc = it.flip ? it.mp : it.np;       // padded rows and columns as the caller has them
  const int tiles_c = pc / 64, tiles = (pr / 64) * tiles_c;
  if ((int)blockIdx.x >= tiles) return;
  const int r0 = (blockIdx.x / tiles_c) * 64, c0 = (blockIdx.x % tiles_c) * 64;
  if (threadIdx.x < 64) {
    double s = it.norm[threadIdx.x] + it.norm[threadIdx.x + 64];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) s += __shfl_xor(s, x);
    if (threadIdx.x == 0) inv_s = (double)kScaleX / (sqrt(s) + (double)c.eps);
  }
  __syncthreads();
  const double inv = inv_s;
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int r = (threadIdx.x >> 6) + 4 * k, col = threadIdx.x & 63;
    float x = 0.f;
    if (r0 + r < it.rows && c0 + col < it.cols)
      x = (float)((double)direction<T>(c, it, (int64_t)(r0 + r) * it.ldu + c0 + col, (int64_t)(r0 + r) * it.cols + c0 + col) * inv);
    tile[r][col] = split_pair(x);
  }
  __syncthreads();
  char* straight = it.flip ? it.XT[0] : it.X;          // [pr][pc]
  char* turned = it.flip ? it.X : it.XT[0];            // [pc][pr]
  const int line = threadIdx.x >> 2, group = (threadIdx.x >> 1) & 1, part = threadIdx.x & 1;
  store_group(straight + plane_at(r0 + line, c0 + 32 * group, pc), &tile[line][32 * group], 1, part);
  store_group(turned + plane_at(c0 + line, r0 + 32 * group, pr), &tile[32 * group][line], 65, part);
}

// --- products -----------------------------------------------------------------------------------------------------------
enum Stage { kGram = 0, kPoly = 1, kStep = 2, kLast = 3 };     // A = X X^T;  B = bA + cAA;  X = aX + BX;  the same, to the output

struct Tiles {
  int first[kMax + 1];     // first workgroup of every matrix
  int splits[kMax];
  int ticket0[kMax];       // first ticket, and first tile of the partial sums
};

// This wave's loads have landed and its LDS reads are done, then the workgroup's.  (0x0070: vmcnt 0, lgkmcnt 0.  A barrier alone
// does not wait for loads that go to LDS.)
__device__ __forceinline__ void wait_and_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);
  __syncthreads();
}

// ROWS rows of a plane pair, the 128-byte group `k` of each, to an LDS image; W waves.
template <int ROWS, int W>
__device__ __forceinline__ void fetch(const char* src, int64_t row_bytes, char* __restrict lds, int wave, int lane, int k) {
  const char* at = src + (int64_t)(wave * 8 + (lane >> 3)) * row_bytes + (int64_t)k * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
#pragma unroll
  for (int i = 0; i < ROWS / (8 * W); ++i)
    __builtin_amdgcn_global_load_lds((global_void*)(at + (int64_t)i * 8 * W * row_bytes), (lds_void*)(lds + (i * W + wave) * 1024), 16, 0, 0);
}

// One k-step of 32: a wave's MI x NI tiles of 32 x 32.  `p` and `q`: LDS images of the workgroup's rows of the two operands.
template <int MI, int NI>
__device__ __forceinline__ void multiply(const char* __restrict p, const char* __restrict q, f32x16 (&acc)[MI][NI], int row_p,
                                         int row_q, int lane) {
  const int r = lane & 31;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    half8 a[MI][2], b[NI][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int slot = ((h * 4 + ks * 2 + (lane >> 5)) ^ (r & 7)) << 4;      // (every base row is a multiple of 32)
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i][h] = *reinterpret_cast<const half8*>(p + (row_p + 32 * i + r) * 128 + slot);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[j][h] = *reinterpret_cast<const half8*>(q + (row_q + 32 * j + r) * 128 + slot);
    }
    // the small products first; a tile's three MFMAs are MI * NI apart
#pragma unroll
    for (int t = 0; t < 3; ++t)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][t == 1], b[j][t == 0], acc[i][j], 0, 0, 0);
  }
}

template <int TILE, int WM, int WN, typename T>
__global__ __launch_bounds__(WM * WN * 64) void product_kernel(Call c, Tiles tl, int stage, int parity) {
  constexpr int W = WM * WN, MI = TILE / WM / 32, NI = TILE / WN / 32;
  constexpr int kImage = TILE * 128;
  constexpr int kStage = W * 32 * 33 * 4;                        // a 32 x 33 word tile per wave
  __shared__ __attribute__((aligned(1024))) char image0[2 * kImage > kStage ? 2 * kImage : kStage];
  __shared__ __attribute__((aligned(1024))) char image1[2 * kImage];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int which = 0;
  while ((int)blockIdx.x >= tl.first[which + 1]) ++which;
  const Item& it = c.item[which];
  const int splits = tl.splits[which], local = blockIdx.x - tl.first[which];
  const int tile = local / splits, part = local - tile * splits;
  const bool symmetric = stage <= kPoly;
  int ti, tj;
  if (symmetric) {                      // tile t = tj (tj + 1) / 2 + ti, ti <= tj
    tj = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while (tj * (tj + 1) / 2 > tile) --tj;
    while ((tj + 1) * (tj + 2) / 2 <= tile) ++tj;
    ti = tile - tj * (tj + 1) / 2;
  } else {
    const int tiles_m = it.mp / TILE;
    tj = tile / tiles_m;
    ti = tile - tj * tiles_m;
  }
  const char* P = stage == kGram ? it.X : stage == kPoly ? it.A : it.B;
  const char* Q = stage == kGram ? it.X : stage == kPoly ? it.A : it.XT[parity];
  const int depth = stage == kGram ? it.np : it.mp;              // k, padded: an even number of steps of 32
  const int64_t row_bytes = (int64_t)depth * 4;
  const char* p = P + (int64_t)ti * TILE * row_bytes;
  const char* q = Q + (int64_t)tj * TILE * row_bytes;
  const int pairs = depth / 64;
  const int k_first = 2 * (int)((int64_t)pairs * part / splits), k_last = 2 * (int)((int64_t)pairs * (part + 1) / splits);
  const int row_p = (wave / WN) * (TILE / WM), row_q = (wave % WN) * (TILE / WN);

  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  fetch<TILE, W>(p, row_bytes, image0, wave, lane, k_first);
  fetch<TILE, W>(q, row_bytes, image0 + kImage, wave, lane, k_first);
  for (int k = k_first; k < k_last; k += 2) {
    // every load of image 0 has landed, and every wave is done with image 1
    wait_and_barrier();
    fetch<TILE, W>(p, row_bytes, image1, wave, lane, k + 1);
    fetch<TILE, W>(q, row_bytes, image1 + kImage, wave, lane, k + 1);
    __builtin_amdgcn_sched_barrier(0);       // (the loads go out before the step's LDS reads, not after them)
    multiply<MI, NI>(image0, image0 + kImage, acc, row_p, row_q, lane);
    wait_and_barrier();
    if (k + 2 < k_last) {
      fetch<TILE, W>(p, row_bytes, image0, wave, lane, k + 2);
      fetch<TILE, W>(q, row_bytes, image0 + kImage, wave, lane, k + 2);
    }
    __builtin_amdgcn_sched_barrier(0);
    multiply<MI, NI>(image1, image1 + kImage, acc, row_p, row_q, lane);
  }

  if (splits > 1) {
    constexpr int kElems = TILE * TILE;
    float* mine = c.partial + ((int64_t)tl.ticket0[which] + (int64_t)tile * splits) * kElems;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<f32x4*>(mine + (int64_t)part * kElems + (((i * NI + j) * 4 + e / 4) * W * 64 + tid) * 4) =
              f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
    __threadfence();
    __syncthreads();
    __shared__ uint32_t arrived;
    uint32_t* ticket = c.tickets + tl.ticket0[which] + tile;
    if (tid == 0) arrived = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if ((int)arrived != splits - 1) return;
    __threadfence();
    if (tid == 0) *ticket = 0;           // for the next launch
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
          for (int s = 0; s < splits; ++s)
            sum += *reinterpret_cast<const f32x4*>(mine + (int64_t)s * kElems + (((i * NI + j) * 4 + e / 4) * W * 64 + tid) * 4);
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i][j][e + x] = sum[x];
        }
  }
  wait_and_barrier();                    // image 0 becomes the waves' turning tiles

  // Element e of acc[i][j]: row 8 (e / 4) + 4 (lane / 32) + e % 4 and column lane % 32 of the 32 x 32 tile.
  uint32_t* turn = reinterpret_cast<uint32_t*>(image0) + wave * 32 * 33;
  const int half = lane >> 5, jc = lane & 31;
  const float step_size = stage == kLast && it.buf ? c.lr[0] * it.shape_factor : 0.f;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int i0 = ti * TILE + row_p + 32 * i, j0 = tj * TILE + row_q + 32 * j;
      float v[16];
      if (stage == kGram) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[i][j][e] * (kScaleA / (kScaleX * kScaleX));
      } else {
        // the matrix in the linear term, through its transpose: 4 consecutive rows of one column are 8 + 8 bytes
        const char* s = (stage == kPoly ? it.A : it.XT[parity]) + plane_at(j0 + jc, i0, it.mp) + 8 * half;
        const float lin = stage == kPoly ? kB * (kScaleB / kScaleA) : stage == kStep ? kA : kA / kScaleX;
        const float quad = stage == kPoly ? kC * kScaleB / (kScaleA * kScaleA)
                           : stage == kStep ? 1.f / kScaleB : 1.f / (kScaleB * kScaleX);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const half4 hi = *reinterpret_cast<const half4*>(s + 16 * g), lo = *reinterpret_cast<const half4*>(s + 64 + 16 * g);
#pragma unroll
          for (int x = 0; x < 4; ++x) v[4 * g + x] = lin * ((float)hi[x] + (float)lo[x]) + quad * acc[i][j][4 * g + x];
        }
      }
      if (stage == kLast) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int row = i0 + 8 * (e / 4) + 4 * half + e % 4, col = j0 + jc;
          if (row < it.m && col < it.n) {
            const int64_t at = it.flip ? (int64_t)col * it.ldo + row : (int64_t)row * it.ldo + col;
            if (it.buf) {
              float* w = static_cast<float*>(it.out) + at;
              *w -= step_size * v[e];
            } else {
              static_cast<T*>(it.out)[at] = (T)v[e];
            }
          }
        }
        continue;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) turn[(8 * (e / 4) + 4 * half + e % 4) * 33 + jc] = split_pair(v[e]);
      // (a wave's own tile: no barrier, only the order of its own LDS accesses)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const int line = lane >> 1, part_of = lane & 1;
      char* straight = stage == kGram ? it.A : stage == kPoly ? it.B : it.X;
      char* turned = stage == kGram ? it.A : stage == kPoly ? it.B : it.XT[parity ^ 1];
      const int straight_cols = stage <= kPoly ? it.mp : it.np;
      store_group(straight + plane_at(i0 + line, j0, straight_cols), turn + line * 33, 1, part_of);
      if (!symmetric || ti != tj) store_group(turned + plane_at(j0 + line, i0, it.mp), turn + line, 33, part_of);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// --- host ---------------------------------------------------------------------------------------------------------------
inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Shape {
  int m, n, mp, np, flip;
};
Shape shape_of(int rows, int cols, int tile) {
  Shape s;
  s.flip = rows > cols;
  s.m = s.flip ? cols : rows;
  s.n = s.flip ? rows : cols;
  s.mp = (int)up(s.m, tile);
  s.np = (int)up(s.n, tile);
  return s;
}

// 64 x 64 tiles while the largest product of the call has fewer than 128 tiles of 128 x 128.
int tile_of(int count, const int32_t* rows, const int32_t* cols) {
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) tiles += up(rows[i], 128) / 128 * (up(cols[i], 128) / 128);
  return tiles < 128 ? 64 : 128;
}

constexpr int kMaxDim = 1 << 16;

bool bad_shapes(int count, const int32_t* rows, const int32_t* cols) {
  if (count < 1 || count > kMax || !rows || !cols) return true;
  for (int i = 0; i < count; ++i)
    if (rows[i] < 1 || cols[i] < 1 || rows[i] > kMaxDim || cols[i] > kMaxDim) return true;
  return false;
}

// Workgroups that split the k range of a tile: enough for two per CU, each with at least 8 steps of 32.
int splits_for(int64_t tiles, int depth) {
  int64_t s = 512 / (tiles > 0 ? tiles : 1);
  const int64_t most = depth / 64 / 4;
  if (s > most) s = most;
  if (s > 16) s = 16;
  return s < 1 ? 1 : (int)s;
}

struct StageTiles {
  Tiles t;
  int64_t partial_tiles;
  int blocks;
};
StageTiles stage_tiles(const Call& c, int stage, int tile) {
  StageTiles r{};
  int64_t total = 0;
  int tiles[kMax];
  for (int i = 0; i < c.count; ++i) {
    const int tm = c.item[i].mp / tile, tn = c.item[i].np / tile;
    tiles[i] = stage <= kPoly ? tm * (tm + 1) / 2 : tm * tn;
    total += tiles[i];
  }
  int64_t at = 0, tickets = 0;
  for (int i = 0; i < c.count; ++i) {
    const int depth = stage == kGram ? c.item[i].np : c.item[i].mp;
    int s = splits_for(total, depth);
    if (tickets + (int64_t)tiles[i] * s > kMaxTickets) s = 1;
    r.t.first[i] = (int)at;
    r.t.splits[i] = s;
    r.t.ticket0[i] = (int)tickets;
    at += (int64_t)tiles[i] * s;
    if (s > 1) tickets += (int64_t)tiles[i] * s;
  }
  for (int i = c.count; i <= kMax; ++i) r.t.first[i] = (int)at;
  r.blocks = (int)at;
  r.partial_tiles = tickets;
  return r;
}

struct Layout {
  int64_t total;
  int tile;
};
// Fills the workspace part of `c.item` (offsets from `base`, which may be null when only the size is asked for).
Layout lay_out(Call& c, const int32_t* rows, const int32_t* cols, int count, char* base) {
  Layout l;
  l.tile = tile_of(count, rows, cols);
  c.count = count;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = base + at;
    at += up(bytes, 1024);
    return p;
  };
  c.tickets = reinterpret_cast<uint32_t*>(take(kMaxTickets * 4));
  for (int i = 0; i < count; ++i) {
    Item& it = c.item[i];
    const Shape s = shape_of(rows[i], cols[i], l.tile);
    it.rows = rows[i], it.cols = cols[i];
    it.m = s.m, it.n = s.n, it.mp = s.mp, it.np = s.np, it.flip = s.flip;
    it.norm = reinterpret_cast<double*>(take(kNormBlocks * 8));
    it.X = take((int64_t)s.mp * s.np * 4);
    it.XT[0] = take((int64_t)s.mp * s.np * 4);
    it.XT[1] = take((int64_t)s.mp * s.np * 4);
    it.A = take((int64_t)s.mp * s.mp * 4);
    it.B = take((int64_t)s.mp * s.mp * 4);
  }
  int64_t partial = 0;
  for (int stage = kGram; stage <= kStep; ++stage) {
    const int64_t p = stage_tiles(c, stage, l.tile).partial_tiles;
    partial = p > partial ? p : partial;
  }
  c.partial = reinterpret_cast<float*>(take(partial * l.tile * l.tile * 4));
  l.total = at;
  return l;
}

template <typename T>
int run(Call& c, int tile, hipStream_t s) {
  norm_kernel<T><<<dim3(kNormBlocks, c.count), 256, 0, s>>>(c);
  int64_t most = 0;
  for (int i = 0; i < c.count; ++i) {
    const int64_t t = (int64_t)(c.item[i].mp / 64) * (c.item[i].np / 64);
    most = t > most ? t : most;
  }
  split_kernel<T><<<dim3((unsigned)most, c.count), 256, 0, s>>>(c);
  StageTiles st[3];
  for (int stage = kGram; stage <= kStep; ++stage) st[stage] = stage_tiles(c, stage, tile);
  for (int k = 0; k < 5; ++k)
    for (int stage = kGram; stage <= kStep; ++stage) {
      const int what = stage == kStep && k == 4 ? kLast : stage;
      if (tile == 64)
        product_kernel<64, 2, 2, T><<<st[stage].blocks, 256, 0, s>>>(c, st[stage].t, what, k & 1);
      else
        product_kernel<128, 2, 2, T><<<st[stage].blocks, 256, 0, s>>>(c, st[stage].t, what, k & 1);
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
  if (dtype == DTF_F32) return run<float>(c, l.tile, s);
  if (dtype == DTF_BF16) return run<bf16_t>(c, l.tile, s);
  return run<f16_t>(c, l.tile, s);
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
  return run<float>(c, l.tile, (hipStream_t)stream);
}
