// Element types of the operators around the flow (embedding, group norm, gradient norm): float32, bfloat16 and
// float16 values, widened to float32 where they are loaded and rounded once (to nearest even) where they are stored.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nessai_amd.h"

int nsa_fail(int code, const char* fmt, ...);  // nsa_api.hip: sets nsa_last_error, returns `code`

typedef __bf16 nsa_bf16;
typedef _Float16 nsa_f16;

// V neighbouring elements, moved as one access of V * sizeof(T) bytes (the caller checks the alignment)
template <typename T, int V>
struct alignas(V * sizeof(T)) NsaPack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void nsa_load(const T* p, float (&out)[V]) {
  const NsaPack<T, V> a = *reinterpret_cast<const NsaPack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = (float)a.v[i];
}

template <typename T, int V>
__device__ __forceinline__ void nsa_store(T* p, const float (&in)[V]) {
  NsaPack<T, V> a;
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] = (T)in[i];
  *reinterpret_cast<NsaPack<T, V>*>(p) = a;
}

static inline int nsa_elem_bytes(int dtype) { return dtype == NSA_DT_F32 ? 4 : 2; }
static inline bool nsa_elem_known(int dtype) { return dtype == NSA_DT_F32 || dtype == NSA_DT_BF16 || dtype == NSA_DT_F16; }
