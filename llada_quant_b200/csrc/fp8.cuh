// What the e4m3 product's kernels share.
#pragma once

#include <algorithm>

#include "llq_common.cuh"

namespace llq {

// e4m3 rows [M][K] (pitch ldx) with scales [M][G], e4m3 weight [N][K] (pitch ldw) with scales [ceil(N / 128)][G]
struct Fp8Operands {
  const uint8_t* x;
  const float* xs;
  int64_t ldx;
  const uint8_t* w;
  const float* ws;
  int64_t ldw;
  const void* bias;
  void* out;
  int out_type;
  int64_t M;
  int N, K, G;
};

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

int fp8_gemm_tc(const Fp8Operands& p, cudaStream_t st);

}  // namespace llq
