// Softmax cross-entropy over a vocabulary against INTEGER labels, loss and gradient: the output end of a model over tokens,
// where a one-hot label matrix would be as large as the logits.
//
//   loss[t]  = log(sum_c exp z[t][c]) - z[t][l_t]
//   dz[t][c] = w_t * (exp(z[t][c]) / sum_c' exp z[t][c'] - [c = l_t])        w_t = grad_scale, or the row's upstream gradient
//
// l_t < 0 is padding: loss 0, a gradient row of zeros, the logits are not looked at.  l_t >= classes: NaN loss and gradient
// row (as the reference framework's op on a GPU).  A row with a NaN, a +inf or nothing but -inf has the loss and gradient NaN,
// single -inf logits (masked classes) have probability zero.  Logits and dz in fp32, bf16 or fp16 (one rounding at the store),
// everything in between in fp32.
//
// Bound by memory: one read of the logits and one write of the gradient.  A group of threads owns a row and keeps it in
// REGISTERS between the sums and the gradient (64 bytes to 256 KB a row: up to 16 packs of 16 bytes for each of up to 1024 threads),
// so the second use of a row costs no traffic.  Every thread finds the maximum of its own elements first and sums
// exponentials relative to it; the pairs (maximum, sum) meet in one exchange: one barrier per row and not two.  Rows that do
// not fit are streamed twice, or, where they are few, cut into slices for a block each.  Rows may start at any element: packs are aligned to 16 bytes of memory, and the first and last
// pack of a row are taken element by element.
#include "dtf_api.h"
#include "dtf_types.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The difference to the maximum is formed before it is scaled: the largest term is exactly 1, a row with one class left has
// the loss 0 and no gradient.  (One multiply-add from the scaled maximum would save an instruction and both properties.)
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

struct XentArgs {
  int64_t tokens, classes;
  int64_t ld, ldz;
  const void* labels;
  int wide;
  float grad_scale;
  const float* g;          // backward pass: upstream gradient of the rows
  int64_t g_stride;
  float* row_loss;         // may be null
  float* stats;            // [tokens][2]: maximum and sum of exponentials relative to it (may be null)
};

// (maximum, sum of exponentials relative to it) of two disjoint sets.  A set of nothing but -inf (a thread past the end of
// the row, masked classes) has the sum 0; so has a whole row of them, whose loss is NaN through m - z.
__device__ __forceinline__ void merge(float& m, float& s, float om, float os) {
  const float top = fmaxf(m, om), at = top == -INFINITY ? 0.f : top;
  s = s * exp_of(m - at) + os * exp_of(om - at);
  m = top;
}

// Over the G threads of a row (G = 64: a wave; otherwise the whole block).  The order of additions is fixed.
template <int G>
__device__ __forceinline__ void merge_row(float& m, float& s) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const float om = __shfl_xor(m, x), os = __shfl_xor(s, x);
    merge(m, s, om, os);
  }
  // (two lanes that merge each other's pair may differ in the last bit of the sum: all take the first lane's)
  s = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, s)));
  if (G > 64) {
    __shared__ float2 of_wave[G / 64];
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = make_float2(m, s);
    __syncthreads();
    m = of_wave[0].x;
    s = of_wave[0].y;
#pragma unroll
    for (int w = 1; w < G / 64; ++w) merge(m, s, of_wave[w].x, of_wave[w].y);
  }
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Makes the compiler forget that it has seen the values: of a row of 16-bit logits it would otherwise keep the converted
// floats of one pass for the next, twice the registers, and spill (1024 threads x 16 packs: 4.7 ms instead of 1.7).
template <typename P, int V>
__device__ __forceinline__ void forget(P (&z)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    u32x4 w = __builtin_bit_cast(u32x4, z[k]);
    asm volatile("" : "+v"(w));
    z[k] = __builtin_bit_cast(P, w);
  }
}

// One row as packs of 16 bytes aligned in memory; element e of pack i is class i * N + e - lead.
template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  typedef Pack<T, N> P;
  T* first;
  int lead;
  int classes;      // (a row has fewer than 2^31 elements)
  int packs;
  __device__ __forceinline__ Row(T* row, int64_t c) {
    first = row;
    lead = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    classes = (int)c;
    packs = (lead + classes + N - 1) / N;
  }
  __device__ __forceinline__ bool whole(int i) const { return i * N >= lead && i * N - lead + N <= classes; }
  __device__ __forceinline__ bool inside(int c) const { return c >= 0 && c < classes; }
  // V packs, `step` apart from pack i; outside the row: -inf.  The whole packs are requested first and together; the at most
  // two partial ones of the row cost their threads a second round.
  template <int V>
  __device__ __forceinline__ void load(int i, int step, P (&p)[V]) const {
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll
      for (int e = 0; e < N; ++e) p[k].v[e] = (T)(-INFINITY);
      if (whole(i + k * step)) p[k] = *reinterpret_cast<const P*>(first + ((i + k * step) * N - lead));
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (i + k * step < packs && !whole(i + k * step)) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int c = (i + k * step) * N + e - lead;
          if (inside(c)) p[k].v[e] = first[c];
        }
      }
    }
  }
};

// Stores pack i of the row's gradient; `dst` has the logits' alignment modulo 16 bytes if SAME.
template <typename T, bool SAME>
__device__ __forceinline__ void store_pack(const Row<T>& row, T* dst, int i, const typename Row<T>::P& p) {
  constexpr int N = Row<T>::N;
  if (SAME && row.whole(i)) {
    // (past the caches: nobody reads the gradient soon, and the logits keep their room; 5.4 -> 5.7 TB/s)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, p), reinterpret_cast<u32x4*>(dst + (i * N - row.lead)));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int c = i * N + e - row.lead;
      if (row.inside(c)) dst[c] = p.v[e];
    }
  }
}

template <typename T>
__device__ __forceinline__ typename Row<T>::P gradient_pack(const Row<T>& row, int i, const typename Row<T>::P& z, float m,
                                                            float factor, float weight, int label) {
  typename Row<T>::P p;
  const int at = label + row.lead - i * Row<T>::N;      // the label's element of this pack, if it has it
  if ((unsigned)at < (unsigned)Row<T>::N) {
#pragma unroll
    for (int e = 0; e < Row<T>::N; ++e) p.v[e] = (T)(factor * exp_of((float)z.v[e] - m) - (e == at ? weight : 0.f));
  } else {
#pragma unroll
    for (int e = 0; e < Row<T>::N; ++e) p.v[e] = (T)(factor * exp_of((float)z.v[e] - m));
  }
  return p;
}

__device__ __forceinline__ int64_t label_of(const XentArgs& a, int64_t t) {
  return a.wide ? static_cast<const int64_t*>(a.labels)[t] : (int64_t) static_cast<const int32_t*>(a.labels)[t];
}

// G threads per row (64: several rows per block), V packs per thread: the row fits G * V packs.
template <typename T, int G, int V, bool SAME>
__global__ __launch_bounds__(G < 256 ? 256 : G) void xent_kernel(XentArgs a, T* logits, T* dz) {
  constexpr int kRows = G < 256 ? 256 / G : 1;
  typedef typename Row<T>::P P;
  const int tid = threadIdx.x % G;
  const int64_t t = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  if (t >= a.tokens) return;          // (a whole wave, or the whole block)
  const Row<T> row(logits + t * a.ld, a.classes);
  const int64_t label = label_of(a, t);
  T* dst = dz + t * a.ldz;
  if (label < 0 || label >= a.classes) {
    const float fill = label < 0 ? 0.f : NAN;
    if (dz) {
      P p;
#pragma unroll
      for (int e = 0; e < Row<T>::N; ++e) p.v[e] = (T)fill;
      for (int i = tid; i < row.packs; i += G) store_pack<T, SAME>(row, dst, i, p);
    }
    if (tid == 0) {
      if (a.row_loss) a.row_loss[t] = fill;
      if (a.stats) a.stats[2 * t] = 0.f, a.stats[2 * t + 1] = 1.f;
    }
    return;
  }
  P z[V];
  row.load(tid, G, z);
  const float z_label = tid == 0 ? (float)row.first[label] : 0.f;     // (read before any thread of the row may store dz)
  float m = -INFINITY, s = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k)
#pragma unroll
    for (int e = 0; e < Row<T>::N; ++e) m = fmaxf(m, (float)z[k].v[e]);
  const float own = m == -INFINITY ? 0.f : m;
  constexpr bool kForget = sizeof(T) == 2 && G == 1024;
  if (kForget) forget(z);
#pragma unroll
  for (int k = 0; k < V; ++k)
#pragma unroll
    for (int e = 0; e < Row<T>::N; ++e) s += exp_of((float)z[k].v[e] - own);
  merge_row<G>(m, s);
  if (tid == 0) {
    if (a.row_loss) a.row_loss[t] = (m - z_label) + logf(s);
    if (a.stats) a.stats[2 * t] = m, a.stats[2 * t + 1] = s;
  }
  if (!dz) return;
  if (kForget) forget(z);
  const float factor = a.grad_scale / s;
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (k * G + tid < row.packs)
      store_pack<T, SAME>(row, dst, k * G + tid, gradient_pack<T>(row, k * G + tid, z[k], m, factor, a.grad_scale, (int)label));
}

// Rows of any length: two passes over memory (the first alone without dz).
constexpr int kStream = 1024;
template <typename T, bool SAME>
__global__ __launch_bounds__(kStream) void xent_stream_kernel(XentArgs a, T* logits, T* dz) {
  typedef typename Row<T>::P P;
  const int tid = threadIdx.x;
  const int64_t t = blockIdx.x;
  const Row<T> row(logits + t * a.ld, a.classes);
  const int64_t label = label_of(a, t);
  const bool use = label >= 0 && label < a.classes;
  T* dst = dz + t * a.ldz;
  if (!use) {
    const float fill = label < 0 ? 0.f : NAN;
    if (dz) {
      P p;
#pragma unroll
      for (int e = 0; e < Row<T>::N; ++e) p.v[e] = (T)fill;
      for (int i = tid; i < row.packs; i += kStream) store_pack<T, SAME>(row, dst, i, p);
    }
    if (tid == 0) {
      if (a.row_loss) a.row_loss[t] = fill;
      if (a.stats) a.stats[2 * t] = 0.f, a.stats[2 * t + 1] = 1.f;
    }
    return;
  }
  const float z_label = tid == 0 ? (float)row.first[label] : 0.f;
  float m = -INFINITY, s = 0.f;
  constexpr int U = 4;
  for (int i0 = tid; i0 < row.packs; i0 += U * kStream) {
    P z[U];
    row.load(i0, kStream, z);
    float top = m;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < Row<T>::N; ++e) top = fmaxf(top, (float)z[k].v[e]);
    const float own = top == -INFINITY ? 0.f : top;
    s *= exp_of(m - own);             // (m = -inf: s is 0 and stays 0)
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < Row<T>::N; ++e) s += exp_of((float)z[k].v[e] - own);
    m = top;
  }
  merge_row<kStream>(m, s);
  if (tid == 0) {
    if (a.row_loss) a.row_loss[t] = (m - z_label) + logf(s);
    if (a.stats) a.stats[2 * t] = m, a.stats[2 * t + 1] = s;
  }
  if (!dz) return;
  const float factor = a.grad_scale / s;
  for (int i0 = tid; i0 < row.packs; i0 += 2 * kStream) {
    P z[2];
    row.load(i0, kStream, z);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (i0 + k * kStream < row.packs)
        store_pack<T, SAME>(row, dst, i0 + k * kStream,
                            gradient_pack<T>(row, i0 + k * kStream, z[k], m, factor, a.grad_scale, (int)label));
  }
}

// Few long rows: one block per row would leave most CUs without work, so a block takes kSlice packs of a row.  First the maximum and
// the sum of every slice and the label's logit (before a gradient can lie on top of it), then, in a second launch, every block joins
// its row's pairs in the same order and writes its slice of the gradient.
constexpr int kGradPacks = 4, kGradThreads = 256, kSlice = kGradPacks * kGradThreads;
struct Parts {
  float2* pair;       // [tokens][slices]
  float* z_label;     // [tokens]
  int slices;
};
template <typename T>
__global__ __launch_bounds__(kGradThreads) void xent_part_kernel(XentArgs a, T* logits, Parts parts) {
  typedef typename Row<T>::P P;
  const int64_t t = blockIdx.x;
  const Row<T> row(logits + t * a.ld, a.classes);
  const int64_t label = label_of(a, t);
  if (label < 0 || label >= a.classes) return;
  P z[kGradPacks];
  row.load(blockIdx.y * kSlice + threadIdx.x, kGradThreads, z);
  float m = -INFINITY, s = 0.f;
#pragma unroll
  for (int k = 0; k < kGradPacks; ++k)
#pragma unroll
    for (int e = 0; e < Row<T>::N; ++e) m = fmaxf(m, (float)z[k].v[e]);
  const float own = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int k = 0; k < kGradPacks; ++k)
#pragma unroll
    for (int e = 0; e < Row<T>::N; ++e) s += exp_of((float)z[k].v[e] - own);
  merge_row<kGradThreads>(m, s);
  if (threadIdx.x == 0) {
    parts.pair[t * parts.slices + blockIdx.y] = make_float2(m, s);
    if (((int)label + row.lead) / Row<T>::N / kSlice == (int)blockIdx.y) parts.z_label[t] = (float)row.first[label];
  }
}

// The backward pass: from the statistics of the forward pass, or (JOIN) as the second launch of few rows.
template <typename T, bool SAME, bool JOIN>
__global__ __launch_bounds__(kGradThreads) void xent_grad_kernel(XentArgs a, T* logits, T* dz, Parts parts) {
  typedef typename Row<T>::P P;
  const int64_t t = blockIdx.x;
  const Row<T> row(logits + t * a.ld, a.classes);
  const int64_t label = label_of(a, t);
  T* dst = dz + t * a.ldz;
  const int i0 = blockIdx.y * kSlice + threadIdx.x;
  const bool use = label >= 0 && label < a.classes;
  P z[kGradPacks];
  if (use && dz) row.load(i0, kGradThreads, z);
  float weight, m, total;
  if (JOIN) {
    weight = a.grad_scale, m = -INFINITY, total = 0.f;
    if (use) {
      for (int i = threadIdx.x; i < parts.slices; i += kGradThreads) {
        const float2 pair = parts.pair[t * parts.slices + i];
        merge(m, total, pair.x, pair.y);
      }
      merge_row<kGradThreads>(m, total);
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) {
      if (a.row_loss) a.row_loss[t] = use ? (m - parts.z_label[t]) + logf(total) : label < 0 ? 0.f : NAN;
      if (a.stats) a.stats[2 * t] = use ? m : 0.f, a.stats[2 * t + 1] = use ? total : 1.f;
    }
    if (!dz) return;
  } else {
    weight = a.g[t * a.g_stride], m = a.stats[2 * t], total = a.stats[2 * t + 1];
  }
  const float factor = weight / total;
#pragma unroll
  for (int k = 0; k < kGradPacks; ++k) {
    const int i = i0 + k * kGradThreads;
    if (i >= row.packs) break;
    P p;
    if (use) {
      p = gradient_pack<T>(row, i, z[k], m, factor, weight, (int)label);
    } else {
#pragma unroll
      for (int e = 0; e < Row<T>::N; ++e) p.v[e] = (T)(label < 0 ? 0.f : NAN);
    }
    store_pack<T, SAME>(row, dst, i, p);
  }
}

template <typename T, bool SAME>
int launch_xent(const XentArgs& a, T* logits, T* dz, hipStream_t s) {
  constexpr int N = 16 / sizeof(T);
  // packs of a row: rows that are whole packs apart all start at the first one's place in a pack, others at the worst
  const int64_t lead = a.ld * (int64_t)sizeof(T) % 16 == 0 ? (int64_t)((uintptr_t)logits & 15u) / (int64_t)sizeof(T) : N - 1;
  const int64_t packs = (lead + a.classes + N - 1) / N;
  const unsigned rows = (unsigned)a.tokens;
#define DTF_XENT(G, V)                                                                                           \
  if (packs <= G * V) {                                                                                          \
    xent_kernel<T, G, V, SAME><<<(rows + (G < 256 ? 256 / G : 1) - 1) / (G < 256 ? 256 / G : 1), G < 256 ? 256 : G, 0, s>>>(a, logits, dz); \
    return hipGetLastError() == hipSuccess ? DTF_OK : DTF_ERR_LAUNCH;                                            \
  }
  // Many threads with few packs each: measured at 8192 rows of 64 KB, 1024 x 4 takes 193 us, 512 x 8 217 and 256 x 16 214; at
  // 16384 rows of 16 KB 256 x 4 takes 84 us, 64 x 16 105, 512 x 2 108; at 4096 rows of 128 KB 1024 x 8 187, 512 x 16 206.
  DTF_XENT(64, 1)
  DTF_XENT(64, 4)
  DTF_XENT(256, 4)
  DTF_XENT(512, 4)
  DTF_XENT(1024, 4)
  DTF_XENT(1024, 8)
  DTF_XENT(1024, 16)
#undef DTF_XENT
  xent_stream_kernel<T, SAME><<<rows, kStream, 0, s>>>(a, logits, dz);
  return hipGetLastError() == hipSuccess ? DTF_OK : DTF_ERR_LAUNCH;
}

// Slices of a row that starts anywhere in a pack.
inline int64_t slices_of(int64_t classes, int per_pack) { return ((classes + 2 * per_pack - 2) / per_pack + kSlice - 1) / kSlice; }

// Rows are cut where one block a row takes longer than a second launch (cut: 13.5 us a call up to 64 x 131072 bf16).  One block a
// row, fp32: 1 x 50001 10 us, 1 x 131072 20, 1 x 1000000 133, 64 x 262144 44 (cut 33), 128 x 131072 32 (cut 34).
bool cut_rows(int64_t tokens, int64_t slices) { return tokens <= 64 && slices > 16; }

template <typename T>
int run_xent(const XentArgs& a, const void* logits, void* dz, bool backward, const Parts& parts, hipStream_t s) {
  T* z = static_cast<T*>(const_cast<void*>(logits));
  T* d = static_cast<T*>(dz);
  const bool same = !d || ((((uintptr_t)z ^ (uintptr_t)d) & 15u) == 0 && ((a.ld - a.ldz) * (int64_t)sizeof(T)) % 16 == 0);
  if (backward) {
    constexpr int N = 16 / sizeof(T);
    const dim3 grid((unsigned)a.tokens, (unsigned)slices_of(a.classes, N));
    if (same) xent_grad_kernel<T, true, false><<<grid, kGradThreads, 0, s>>>(a, z, d, Parts{});
    else xent_grad_kernel<T, false, false><<<grid, kGradThreads, 0, s>>>(a, z, d, Parts{});
    return hipGetLastError() == hipSuccess ? DTF_OK : DTF_ERR_LAUNCH;
  }
  if (parts.slices) {
    const dim3 grid((unsigned)a.tokens, (unsigned)parts.slices);
    xent_part_kernel<T><<<grid, kGradThreads, 0, s>>>(a, z, parts);
    const dim3 second((unsigned)a.tokens, d ? (unsigned)parts.slices : 1u);
    if (same) xent_grad_kernel<T, true, true><<<second, kGradThreads, 0, s>>>(a, z, d, parts);
    else xent_grad_kernel<T, false, true><<<second, kGradThreads, 0, s>>>(a, z, d, parts);
    return hipGetLastError() == hipSuccess ? DTF_OK : DTF_ERR_LAUNCH;
  }
  return same ? launch_xent<T, true>(a, z, d, s) : launch_xent<T, false>(a, z, d, s);
}

int checked(const XentArgs& a, const void* logits, int dtype, void* dz, bool backward, void* stream, void* workspace = nullptr,
            int64_t workspace_bytes = 0) {
  // (grids stay below 2^32 threads, the class index of a row below 2^31)
  if (a.tokens < 0 || a.tokens > (1 << 21) || a.classes < 1 || a.classes > (1 << 26) || dtype < 0 || dtype > 2 ||
      a.ld < a.classes || (dz && a.ldz < a.classes))
    return DTF_ERR_SHAPE;
  if (a.tokens == 0) return DTF_OK;
  if (!logits || !a.labels || (backward && (!dz || !a.stats || !a.g))) return DTF_ERR_NULL;
  hipStream_t s = (hipStream_t)stream;
  Parts parts{};
  const int64_t slices = slices_of(a.classes, 16 / dtf_type_size(dtype));
  if (workspace && cut_rows(a.tokens, slices)) {
    if (workspace_bytes < a.tokens * (slices * 8 + 4) || ((uintptr_t)workspace & 7u)) return DTF_ERR_SHAPE;
    parts = Parts{static_cast<float2*>(workspace), reinterpret_cast<float*>(static_cast<float2*>(workspace) + a.tokens * slices), (int)slices};
  }
  if (dtype == DTF_F32) return run_xent<float>(a, logits, dz, backward, parts, s);
  if (dtype == DTF_BF16) return run_xent<bf16_t>(a, logits, dz, backward, parts, s);
  return run_xent<f16_t>(a, logits, dz, backward, parts, s);
}

}  // namespace

extern "C" int64_t dtf_sparse_xent_workspace(int dtype, int64_t tokens, int64_t classes) {
  if (tokens < 0 || classes < 1 || classes > (1 << 26) || dtype < 0 || dtype > 2) return -1;
  const int64_t slices = slices_of(classes, 16 / dtf_type_size(dtype));
  return cut_rows(tokens, slices) ? tokens * (slices * 8 + 4) : 0;
}

extern "C" int dtf_sparse_xent(const void* logits, int dtype, int64_t tokens, int64_t classes, int64_t ld, const void* labels,
                               int labels_wide, void* dz, int64_t ldz, float grad_scale, float* row_loss, float* stats,
                               void* stream) {
  return dtf_sparse_xent_cut(logits, dtype, tokens, classes, ld, labels, labels_wide, dz, ldz, grad_scale, row_loss, stats, nullptr, 0, stream);
}

extern "C" int dtf_sparse_xent_cut(const void* logits, int dtype, int64_t tokens, int64_t classes, int64_t ld, const void* labels,
                                   int labels_wide, void* dz, int64_t ldz, float grad_scale, float* row_loss, float* stats,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  XentArgs a{};
  a.tokens = tokens, a.classes = classes, a.ld = ld, a.ldz = dz ? ldz : ld;
  a.labels = labels, a.wide = labels_wide, a.grad_scale = grad_scale, a.row_loss = row_loss, a.stats = stats;
  return checked(a, logits, dtype, dz, false, stream, workspace, workspace_bytes);
}

extern "C" int dtf_sparse_xent_grad(const void* logits, int dtype, int64_t tokens, int64_t classes, int64_t ld, const void* labels,
                                    int labels_wide, const float* stats, const float* g, int64_t g_stride, void* dz, int64_t ldz,
                                    void* stream) {
  XentArgs a{};
  a.tokens = tokens, a.classes = classes, a.ld = ld, a.ldz = ldz;
  a.labels = labels, a.wide = labels_wide, a.g = g, a.g_stride = g_stride, a.stats = const_cast<float*>(stats);
  return checked(a, logits, dtype, dz, true, stream);
}
