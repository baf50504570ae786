// Element types of the token-model kernels (embed.hip, xent.hip, muon.hip): storage in fp32, bf16 or fp16, arithmetic in
// fp32, one rounding (to nearest even) where a value is stored.
#pragma once
#include "dtf_common.h"

#define DTF_F32 0
#define DTF_BF16 1
#define DTF_F16 2

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// N consecutive elements as one aligned memory access of N * sizeof(T) bytes.
template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};

static inline int dtf_type_size(int dtype) { return dtype == DTF_F32 ? 4 : 2; }

// Largest access in bytes (16, 8, 4 or 2) that divides every address and byte stride or'ed into `bits`.
static inline int dtf_access_bytes(uint64_t bits) {
  if ((bits & 15u) == 0) return 16;
  if ((bits & 7u) == 0) return 8;
  if ((bits & 3u) == 0) return 4;
  return 2;
}
