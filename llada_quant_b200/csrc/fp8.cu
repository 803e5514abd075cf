// 8-bit floating point (e4m3) with one fp32 scale per 128 values of a row, or per 128 x 128 block:
// the quantizer and the product of e4m3 rows with an e4m3 weight.
#include <type_traits>

#include <cuda_fp8.h>

#include "fp8.cuh"
#include "llq_internal.cuh"

namespace llq {

namespace {

constexpr int BLK = 128;
// up to this many rows the product runs on fp8_few_rows_kernel, above on fp8_tc_kernel
constexpr int64_t kFewRows = 16;
// groups whose largest magnitude lies below 448 * 2^-60 are scaled as if it were this, so that the
// product of two scales stays a normal fp32 number
constexpr float kAmaxFloor = 448.f * 0x1p-60f;

__device__ __forceinline__ float group_amax(uint32_t bits) {
  // bits: the largest magnitude's bit pattern; patterns order as magnitudes, NaN above all
  const float m = __uint_as_float(bits);
  return m < kAmaxFloor ? kAmaxFloor : m;
}

__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float group_scale(float amax) { return __fdiv_rn(amax, 448.f); }

// v * 448 / amax, correctly rounded in fp32; 448 = 0.4375 * 2^10, so that no product overflows
__device__ __forceinline__ float ratio(float v, float amax) {
  return __fdiv_rn(__fmul_rn(v, 0.4375f), __fmul_rn(amax, 0x1p-10f));
}

// v * 448 / amax by the reciprocal and one correction with the exact remainder (Markstein, 1990): within a rounding of
// the quotient, and the quotient itself where it fits in fp32.  Of bf16 or fp16 values it is either a border between two
// codes exactly or at least 2^-22 of itself away from one (the numerator has 14 bits at most, a border times the
// denominator 16, both in units that differ by powers of two), so the code is that of ratio().  fp32 values may come
// closer: quantize_values looks.
struct Divider {
  float a, r;
  __device__ __forceinline__ explicit Divider(float amax) {
    a = __fmul_rn(amax, 0x1p-10f);
    r = __fdiv_rn(1.f, a);
    a = fminf(a, 3e38f);  // amax infinite: r = 0, and every finite value gives 0
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float n = __fmul_rn(v, 0.4375f), q = __fmul_rn(n, r);
    return copysignf(__fmaf_rn(__fmaf_rn(-q, a, n), r, q), v);  // (the correction makes +0 of -0)
  }
};

// two values to e4m3 (nearest even; NaN stays NaN), lo in the low byte
__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The codes of N values of type T of a group: e4m3 of ratio(v).  (A division for each value took 42 us at 8192 x 4096
// bf16, and a test for borders with the division behind it 50: a quarter of all groups of bf16 values has some on one.)
template <typename T, int N>
__device__ __forceinline__ void quantize_values(const float (&v)[N], float amax, const Divider& div, uint16_t (&q)[N / 2]) {
  uint32_t differ = 0;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float x = div(v[2 * i]), y = div(v[2 * i + 1]);
    q[i] = to_e4m3x2(x, y);
    if (sizeof(T) == 4) {  // next to a border?
      const float lo = 1.f - 0x1p-22f, hi = 1.f + 0x1p-22f;
      differ |= to_e4m3x2(x * lo, y * lo) ^ to_e4m3x2(x * hi, y * hi);
    }
  }
  if (sizeof(T) == 4 && differ) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) q[i] = to_e4m3x2(ratio(v[2 * i], amax), ratio(v[2 * i + 1], amax));
  }
}

// two e4m3 codes as an fp16 pair, exactly
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

// 8 consecutive values as fp32
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void load8<__half>(const __half* p, float (&v)[8]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// values c .. c + 7 of a row of K, zero beyond; `vec`: the row may be read in 16-byte pieces
template <typename T>
__device__ __forceinline__ void load_part(const T* row, int64_t c, int64_t K, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= K) {
    load8(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_f32(row[c + i]) : 0.f;
  }
}

// the codes of values c .. c + 7 into a row whose pitch is a multiple of 16 bytes; nothing beyond K is written
__device__ __forceinline__ void store_part(uint8_t* row, int64_t c, int64_t K, const uint16_t (&q)[4]) {
  if (c + 8 <= K) {
    *reinterpret_cast<uint2*>(row + c) = make_uint2(q[0] | (static_cast<uint32_t>(q[1]) << 16),
                                                    q[2] | (static_cast<uint32_t>(q[3]) << 16));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < K) row[c + i] = static_cast<uint8_t>(q[i >> 1] >> (8 * (i & 1)));
  }
}

// 16 values c .. c + 15 of a row of K (zero beyond), and the largest magnitude's bits among them as fp32
template <typename T>
__device__ __forceinline__ void load16(const T* row, int64_t c, int64_t K, bool vec, float (&v)[16], uint32_t& m) {
  if (vec && c + 16 <= K) {
    if (sizeof(T) == 2) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c)), b = __ldg(reinterpret_cast<const uint4*>(row + c) + 1);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      uint32_t top = 0;  // of both halves: their patterns order as magnitudes
#pragma unroll
      for (int i = 0; i < 8; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
      const uint16_t t16 = static_cast<uint16_t>(max(top >> 16, top & 0xffffu));
      m = std::is_same<T, __half>::value ? __float_as_uint(__half2float(__ushort_as_half(t16)))
                                         : static_cast<uint32_t>(t16) << 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        } else {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(row + c) + i);
      v[4 * i] = a.x;
      v[4 * i + 1] = a.y;
      v[4 * i + 2] = a.z;
      v[4 * i + 3] = a.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < K ? to_f32(row[c + i]) : 0.f;
  }
  m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, mag(v[i]));
}

// One scale per 128 values of a row: 8 lanes hold a group, 16 values each.  I: 32-bit indices of groups where they fit
// (a 64-bit division per group took as long as all the rest).
template <typename T, typename I>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const T* __restrict__ x, I n, I G, int64_t K, int64_t ldx, int vec,
                                                       uint8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scale) {
  pdl_wait();
  const int l = threadIdx.x & 7;
  const I stride = static_cast<I>(gridDim.x) * (blockDim.x >> 3);
#pragma unroll 1
  for (I i = static_cast<I>(blockIdx.x) * (blockDim.x >> 3) + (threadIdx.x >> 3); i - (threadIdx.x >> 3 & 3) < n; i += stride) {
    const bool in = i < n;  // a warp's four groups leave the loop together
    const I m = in ? i / G : 0;
    const int64_t c = in ? static_cast<int64_t>(i - m * G) * BLK + 16 * l : K;
    float v[16];
    uint32_t b;
    load16(x + static_cast<int64_t>(m) * ldx, c, K, vec != 0, v, b);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    const float amax = group_amax(b);
    uint16_t q[8];
    quantize_values<T>(v, amax, Divider(amax), q);
    uint8_t* to = codes + static_cast<int64_t>(m) * ldc;
    if (c + 16 <= K) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = q[2 * j] | (static_cast<uint32_t>(q[2 * j + 1]) << 16);
      *reinterpret_cast<uint4*>(to + c) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c + j < K) to[c + j] = static_cast<uint8_t>(q[j >> 1] >> (8 * (j & 1)));
    }
    if (l == 0 && in) scale[i] = group_scale(amax);
  }
}

// one scale per 128 x 128 block: a CTA per block, 16 lanes a row, 8 rows of 16 passes
template <typename T>
__global__ void __launch_bounds__(256) fp8_blocks_kernel(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx, int vec,
                                                         uint8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scale) {
  pdl_wait();
  __shared__ uint32_t red[8];
  const int64_t G = (K + BLK - 1) / BLK;
  const int64_t mb = blockIdx.x / G, g = blockIdx.x - mb * G;
  const int64_t c = g * BLK + 8 * (threadIdx.x & 15);
  float v[8][8];
  uint32_t b = 0;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int64_t m = mb * BLK + p * 16 + (threadIdx.x >> 4);
    load_part(x + (m < M ? m : 0) * ldx, m < M ? c : K, K, vec != 0, v[p]);
#pragma unroll
    for (int j = 0; j < 8; ++j) b = max(b, mag(v[p][j]));
  }
  b = __reduce_max_sync(0xffffffffu, b);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = b;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) b = max(b, red[j]);
  const float amax = group_amax(b);
  const Divider div(amax);
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int64_t m = mb * BLK + p * 16 + (threadIdx.x >> 4);
    uint16_t q[4];
    quantize_values<T>(v[p], amax, div, q);
    if (m < M) store_part(codes + m * ldc, c, K, q);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = group_scale(amax);
}

// ---------------------------------------------------------------------------
// product for few rows
// ---------------------------------------------------------------------------

struct LinArgs {
  const void* x;          // e4m3 codes, or values of type T that are quantized on the way
  const float* xs;        // scales of the codes, [M][G]
  int64_t ldx;
  int vec;
  const uint8_t* w;       // e4m3 [N][K], pitch ldw
  const float* ws;        // [ceil(N / 128)][G]
  int64_t ldw;
  const void* bias;       // of the output's type, or null
  void* out;              // [M][N]
  int out_type;
  int64_t M;
  int N, K, G;
};

__device__ __forceinline__ float load_as_f32(const void* p, int type, int64_t i) {
  return type == LLQ_F32    ? static_cast<const float*>(p)[i]
         : type == LLQ_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                            : __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_from_f32(void* p, int type, int64_t i, float v) {
  if (type == LLQ_F32) static_cast<float*>(p)[i] = v;
  else if (type == LLQ_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_once(const uint8_t* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}

__device__ __forceinline__ void codes_to_f16(uint32_t c, uint32_t& lo, uint32_t& hi) {
  lo = e4m3x2_to_f16x2(static_cast<uint16_t>(c));
  hi = e4m3x2_to_f16x2(static_cast<uint16_t>(c >> 16));
}

struct Raw {};  // tag: x holds e4m3 codes

// this lane's 32 values 128 s + 32 t .. of a row of x, as 16 code pairs, and the group's scale
template <typename T>
__device__ __forceinline__ void row_codes(const LinArgs& a, int64_t m, bool in, int s, int t, uint32_t (&q)[8], float& scale) {
  const int64_t c = static_cast<int64_t>(s) * BLK + 32 * t;
  float v[4][8];
  uint32_t b = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    load_part(static_cast<const T*>(a.x) + m * a.ldx, in ? c + 8 * i : a.K, a.K, a.vec != 0, v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) b = max(b, mag(v[i][j]));
  }
  b = max(b, __shfl_xor_sync(0xffffffffu, b, 1));
  b = max(b, __shfl_xor_sync(0xffffffffu, b, 2));
  const float amax = group_amax(b);
  scale = group_scale(amax);
  const Divider div(amax);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t c[4];
    quantize_values<T>(v[i], amax, div, c);
#pragma unroll
    for (int j = 0; j < 2; ++j) q[2 * i + j] = c[2 * j] | (static_cast<uint32_t>(c[2 * j + 1]) << 16);
  }
}
template <>
__device__ __forceinline__ void row_codes<Raw>(const LinArgs& a, int64_t m, bool in, int s, int t, uint32_t (&q)[8], float& scale) {
  const int64_t c = static_cast<int64_t>(s) * BLK + 32 * t;
  const uint8_t* p = static_cast<const uint8_t*>(a.x) + m * a.ldx + c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (in && c + 16 * i < a.K) v = __ldg(reinterpret_cast<const uint4*>(p) + i);  // K is a multiple of 16
    q[4 * i] = v.x;
    q[4 * i + 1] = v.y;
    q[4 * i + 2] = v.z;
    q[4 * i + 3] = v.w;
  }
  scale = in ? a.xs[m * a.G + s] : 0.f;
}

// 16 weight rows per CTA as the rows of mma.sync m16n8k16, 8 rows of x as its columns; 16 warps split K by
// 128-groups and hold the next group's codes while they work on one.  e4m3 is exact in fp16, so the products are exact
// and sums are fp32.  Rows of x that come as values are quantized by every CTA for itself: 4 KB of them against the 32
// KB of weights that the CTA reads, and one launch less.
constexpr int FEW_WARPS = 16;

template <typename T>
__global__ void __launch_bounds__(FEW_WARPS * 32) fp8_few_rows_kernel(const LinArgs a) {
  __shared__ float red[FEW_WARPS][16][9];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 8;
  const int ra = min(n0 + g, a.N - 1), rb = min(n0 + g + 8, a.N - 1);
  const uint8_t* pa = a.w + ra * a.ldw + 32 * t;
  const uint8_t* pb = a.w + rb * a.ldw + 32 * t;
  const float* ws = a.ws + static_cast<int64_t>(n0 / BLK) * a.G;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  uint4 wa[2], wb[2];
  float wsc = 0.f;
  auto load = [&](int s) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool in = s * BLK + 32 * t + 16 * i < a.K;
      wa[i] = in ? load_once(pa + s * BLK + 16 * i) : make_uint4(0, 0, 0, 0);
      wb[i] = in ? load_once(pb + s * BLK + 16 * i) : make_uint4(0, 0, 0, 0);
    }
    wsc = s < a.G ? __ldg(ws + s) : 0.f;
  };
  load(warp);
#pragma unroll 1
  for (int s = warp; s < a.G; s += FEW_WARPS) {
    uint32_t q[8];
    float sc;
    row_codes<T>(a, m0 + g < a.M ? m0 + g : 0, m0 + g < a.M, s, t, q, sc);
    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t ua[4] = {wa[i].x, wa[i].y, wa[i].z, wa[i].w}, ub[4] = {wb[i].x, wb[i].y, wb[i].z, wb[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a0, a1, a2, a3, b0, b1;
        codes_to_f16(ua[j], a0, a2);
        codes_to_f16(ub[j], a1, a3);
        codes_to_f16(q[4 * i + j], b0, b1);
        mma_f16(d, a0, a1, a2, a3, b0, b1);
      }
    }
    // columns 2t and 2t + 1: rows of x whose scales lanes 8t and 8t + 4 hold
    const float s0 = __fmul_rn(__shfl_sync(0xffffffffu, sc, 8 * t), wsc);
    const float s1 = __fmul_rn(__shfl_sync(0xffffffffu, sc, 8 * t + 4), wsc);
    load(s + FEW_WARPS);
    acc[0] = __fmaf_rn(s0, d[0], acc[0]);
    acc[1] = __fmaf_rn(s1, d[1], acc[1]);
    acc[2] = __fmaf_rn(s0, d[2], acc[2]);
    acc[3] = __fmaf_rn(s1, d[3], acc[3]);
  }
  red[warp][g][2 * t] = acc[0];
  red[warp][g][2 * t + 1] = acc[1];
  red[warp][g + 8][2 * t] = acc[2];
  red[warp][g + 8][2 * t + 1] = acc[3];
  __syncthreads();
  if (threadIdx.x < 128) {
    const int r = threadIdx.x & 15, col = threadIdx.x >> 4;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < FEW_WARPS; ++w) v = __fadd_rn(v, red[w][r][col]);
    const int n = n0 + r;
    const int64_t m = m0 + col;
    if (n < a.N && m < a.M) {
      if (a.bias != nullptr) v = __fadd_rn(v, load_as_f32(a.bias, a.out_type, n));
      store_from_f32(a.out, a.out_type, m * a.N + n, v);
    }
  }
}

template <typename T>
int launch_rows(const void* x, int64_t M, int64_t K, int64_t ldx, int block_rows, uint8_t* codes, int64_t ldc, float* scale,
                cudaStream_t st) {
  const int vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * sizeof(T)) % 16 == 0;
  const int64_t G = (K + BLK - 1) / BLK;
  if (block_rows == 1) {
    const int64_t n = M * G;
    int64_t blocks = (n + 31) / 32;
    const int64_t most = static_cast<int64_t>(num_sms()) * 8;
    if (blocks > most) blocks = most;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (n < (1 << 30))
      launch_pdl(fp8_rows_kernel<T, uint32_t>, grid, dim3(256), 0, st, static_cast<const T*>(x), static_cast<uint32_t>(n),
                 static_cast<uint32_t>(G), K, ldx, vec, codes, ldc, scale);
    else
      launch_pdl(fp8_rows_kernel<T, int64_t>, grid, dim3(256), 0, st, static_cast<const T*>(x), n, G, K, ldx, vec, codes, ldc,
                 scale);
    return check_launch("fp8_rows_kernel");
  }
  launch_pdl(fp8_blocks_kernel<T>, dim3(static_cast<unsigned>((M + BLK - 1) / BLK * G)), dim3(256), 0, st,
             static_cast<const T*>(x), M, K, ldx, vec, codes, ldc, scale);
  return check_launch("fp8_blocks_kernel");
}

}  // namespace

int fp8_quantize(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int block_rows, uint8_t* codes, int64_t ldc,
                 float* scale, cudaStream_t st) {
  if (M < 0 || K < 1 || ldx < K || ldc < K) return fail(LLQ_EINVAL, "bad shape M=%lld K=%lld ldx=%lld ldc=%lld",
                                                        (long long)M, (long long)K, (long long)ldx, (long long)ldc);
  if (block_rows != 1 && block_rows != BLK)
    return fail(LLQ_EUNSUPPORTED, "one scale per 1 x 128 or per 128 x 128, got %d rows", block_rows);
  if (ldc % 16 != 0 || (reinterpret_cast<uintptr_t>(codes) & 15) != 0)
    return fail(LLQ_EINVAL, "the codes need a 16-byte aligned base and row pitch");
  if (block_rows == BLK && (M + BLK - 1) / BLK * ((K + BLK - 1) / BLK) > 0x7fffffff)
    return fail(LLQ_EINVAL, "too many blocks");
  if (M == 0) return LLQ_OK;
  if (x == nullptr || codes == nullptr || scale == nullptr) return fail(LLQ_EINVAL, "null pointer");
  switch (x_dtype) {
    case LLQ_F32: return launch_rows<float>(x, M, K, ldx, block_rows, codes, ldc, scale, st);
    case LLQ_F16: return launch_rows<__half>(x, M, K, ldx, block_rows, codes, ldc, scale, st);
    case LLQ_BF16: return launch_rows<__nv_bfloat16>(x, M, K, ldx, block_rows, codes, ldc, scale, st);
  }
  return fail(LLQ_EUNSUPPORTED, "unknown dtype %d", x_dtype);
}

int fp8_linear(const void* x, int x_dtype, const float* x_scale, int64_t M, int K, int64_t ldx, const uint8_t* w,
               const float* w_scale, int N, int64_t ldw, const void* bias, void* out, int out_dtype, void* workspace,
               size_t bytes, cudaStream_t st) {
  if (M < 0 || K < 1 || N < 1 || ldx < K || ldw < K)
    return fail(LLQ_EINVAL, "bad shape M=%lld K=%d N=%d ldx=%lld ldw=%lld", (long long)M, K, N, (long long)ldx, (long long)ldw);
  if (out_dtype != LLQ_F32 && out_dtype != LLQ_F16 && out_dtype != LLQ_BF16)
    return fail(LLQ_EUNSUPPORTED, "unknown output dtype %d", out_dtype);
  if (K % 16 != 0) return fail(LLQ_EUNSUPPORTED, "the e4m3 product needs K in multiples of 16, got %d", K);
  if (ldw % 16 != 0 || (reinterpret_cast<uintptr_t>(w) & 15) != 0)
    return fail(LLQ_EINVAL, "the weight codes need a 16-byte aligned base and row pitch");
  if (M > 0x7fffffff - 256) return fail(LLQ_EINVAL, "too many rows");
  if (M == 0) return LLQ_OK;
  if (x == nullptr || w == nullptr || w_scale == nullptr || out == nullptr) return fail(LLQ_EINVAL, "null pointer");
  const int size = x_dtype == LLQ_E4M3 ? 1 : x_dtype == LLQ_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * size) % 16 == 0;
  if (x_dtype == LLQ_E4M3) {
    if (x_scale == nullptr) return fail(LLQ_EINVAL, "e4m3 rows need their scales");
    if (!vec) return fail(LLQ_EINVAL, "the row codes need a 16-byte aligned base and row pitch");
  } else if (x_dtype != LLQ_F32 && x_dtype != LLQ_F16 && x_dtype != LLQ_BF16) {
    return fail(LLQ_EUNSUPPORTED, "unknown dtype %d", x_dtype);
  }
  const int G = (K + BLK - 1) / BLK;
  if (M > kFewRows) {
    Fp8Operands p{};
    p.x = static_cast<const uint8_t*>(x);
    p.xs = x_scale;
    p.ldx = ldx;
    if (x_dtype != LLQ_E4M3) {  // quantized once into the workspace
      const size_t need = fp8_linear_workspace(M, K, N, x_dtype);
      if (workspace == nullptr || bytes < need) return fail(LLQ_ENOSPACE, "workspace needs %zu bytes, got %zu", need, bytes);
      if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(LLQ_EINVAL, "the workspace needs 16-byte alignment");
      uint8_t* codes = static_cast<uint8_t*>(workspace);
      float* scale = reinterpret_cast<float*>(codes + static_cast<size_t>(M) * K);
      const int rc = fp8_quantize(x, x_dtype, M, K, ldx, 1, codes, K, scale, st);
      if (rc) return rc;
      p.x = codes;
      p.xs = scale;
      p.ldx = K;
    }
    p.w = w;
    p.ws = w_scale;
    p.ldw = ldw;
    p.bias = bias;
    p.out = out;
    p.out_type = out_dtype;
    p.M = M;
    p.N = N;
    p.K = K;
    p.G = G;
    return fp8_gemm_tc(p, st);
  }
  LinArgs a{};
  a.x = x;
  a.xs = x_scale;
  a.ldx = ldx;
  a.vec = vec;
  a.w = w;
  a.ws = w_scale;
  a.ldw = ldw;
  a.bias = bias;
  a.out = out;
  a.out_type = out_dtype;
  a.M = M;
  a.N = N;
  a.K = K;
  a.G = G;
  const dim3 grid((N + 15) / 16, static_cast<unsigned>((M + 7) / 8));
  switch (x_dtype) {
    case LLQ_E4M3: launch_pdl(fp8_few_rows_kernel<Raw>, grid, dim3(FEW_WARPS * 32), 0, st, a); break;
    case LLQ_F32: launch_pdl(fp8_few_rows_kernel<float>, grid, dim3(FEW_WARPS * 32), 0, st, a); break;
    case LLQ_F16: launch_pdl(fp8_few_rows_kernel<__half>, grid, dim3(FEW_WARPS * 32), 0, st, a); break;
    default: launch_pdl(fp8_few_rows_kernel<__nv_bfloat16>, grid, dim3(FEW_WARPS * 32), 0, st, a); break;
  }
  return check_launch("fp8_few_rows_kernel");
}

// codes [M][K] (K is a multiple of 16) and scales [M][G] of rows that are quantized before the tensor-core product
size_t fp8_linear_workspace(int64_t M, int K, int N, int x_dtype) {
  if (M <= kFewRows || K < 1 || x_dtype == LLQ_E4M3) return 0;
  return static_cast<size_t>(M) * K + static_cast<size_t>(M) * ((K + BLK - 1) / BLK) * 4;
}

}  // namespace llq
