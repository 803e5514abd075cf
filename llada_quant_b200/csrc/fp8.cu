// 8-bit floating point (e4m3) with one fp32 scale per 128 values of a row, or per 128 x 128 block:
// the quantizer and the product of e4m3 rows with an e4m3 weight.
#include <type_traits>

#include <cuda_fp8.h>

#include "fp8.cuh"
#include "llq_internal.cuh"

namespace llq {

namespace {

constexpr int BLK = 128;
constexpr int64_t kOwnK = 16384;  // longest rows that fp8_few_rows_kernel quantizes (it holds 8 in shared memory)
// groups whose largest magnitude lies below 448 * 2^-60 are scaled as if it were this, so that the
// product of two scales stays a normal fp32 number
constexpr float kAmaxFloor = 448.f * 0x1p-60f;

__device__ __forceinline__ float group_amax(uint32_t bits) {
  // bits: the largest magnitude's bit pattern; patterns order as magnitudes, NaN above all
  const float m = __uint_as_float(bits);
  return m < kAmaxFloor ? kAmaxFloor : m;
}

__device__ __forceinline__ float group_scale(float amax) { return __fdiv_rn(amax, 448.f); }

// v * 448 / amax in fp32; 448 = 0.4375 * 2^10, so that no product overflows.  For bf16 and fp16 values the product is exact
// and the quotient correctly rounded; for fp32 values both are rounded, so it is within 2^-23 of itself.
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
    return __fmaf_rn(-__fmaf_rn(q, a, -n), r, q);  // (so written it keeps the sign of a zero)
  }
};

// two values to e4m3 (nearest even; NaN stays NaN), lo in the low byte
__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The codes of N values of type T of a group: e4m3 of ratio(v).  (With a division for each value 8192 x 4096 bf16
// takes 27.4 us, with this 18.4; fp32 28.8 both.  A test for borders with the division behind it is slower than either for
// bf16: a quarter of all groups has some on one.)
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

// the codes of values c .. c + 15 into a row whose pitch is a multiple of 16 bytes; nothing beyond K is written
__device__ __forceinline__ void store16(uint8_t* row, int64_t c, int64_t K, const uint32_t (&w)[4]) {
  if (c + 16 <= K) {
    *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c + j < K) row[c + j] = static_cast<uint8_t>(w[j >> 2] >> (8 * (j & 3)));
  }
}

// 16 values of a row as they lie in memory: they stay so until their codes are made, which halves the registers
template <typename T>
struct Raw16 {
  uint32_t w[4 * sizeof(T)];

  // values c .. c + 15 of a row of K, zero beyond
  __device__ __forceinline__ void load(const T* row, int64_t c, int64_t K, bool vec) {
    constexpr int N = sizeof(T);  // 16-byte pieces
    if (vec && c + 16 <= K) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c) + i);
        w[4 * i] = a.x;
        w[4 * i + 1] = a.y;
        w[4 * i + 2] = a.z;
        w[4 * i + 3] = a.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4 * N; ++i) {
        if (sizeof(T) == 4) {
          w[i] = c + i < K ? reinterpret_cast<const uint32_t*>(row)[c + i] : 0u;
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
          w[i] = (c + 2 * i < K ? h[c + 2 * i] : 0u) | (c + 2 * i + 1 < K ? static_cast<uint32_t>(h[c + 2 * i + 1]) << 16 : 0u);
        }
      }
    }
  }

  // the largest magnitude's bits as fp32
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const T2 v = __hmax2_nan(__habs2(*reinterpret_cast<const T2*>(&w[i])), *reinterpret_cast<const T2*>(&m));
        m = *reinterpret_cast<const uint32_t*>(&v);
      }
      const uint32_t t = max(m >> 16, m & 0xffffu);  // (patterns order as magnitudes, NaN above all)
      return std::is_same<T, __half>::value ? __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(t)))) : t << 16;
    }
  }

  // the codes under a group's largest magnitude
  __device__ __forceinline__ void codes(float amax, const Divider& div, uint32_t (&c)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v[4];
      uint16_t q[2];
      four(j, v);
      quantize_values<T>(v, amax, div, q);
      c[j] = q[0] | (static_cast<uint32_t>(q[1]) << 16);
    }
  }

  // values 4 j .. 4 j + 3
  __device__ __forceinline__ void four(int j, float (&v)[4]) const {
    if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[(4 * j + i) % (4 * sizeof(T))]);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t u = w[2 * j + i];
        if (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        } else {
          v[2 * i] = __uint_as_float(u << 16);
          v[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
        }
      }
    }
  }
};

// One scale per 128 values of a row: 8 lanes hold a group, 16 values each.  I: 32-bit indices of groups where they fit.
// It has to read 2 (4) bytes a value and write 1; what holds it below the memory's rate is that a warp computes while it
// has no load under way, about 6 instructions a value, so many warps and few instructions are wanted: 8192 x 4096 bf16
// takes 18.4 us at 6 CTAs per SM (5.5 TB/s), 19.1 at 5 and 19.7 at 7; with a division per group for its row 19.6, and asking for the
// next group ahead costs a fifth, in registers.  fp32: 28.8 us at 5 CTAs (5.8 TB/s), 30.0 at 4, 31.6 at 6.
template <typename T>
constexpr int kRowsBlocks = sizeof(T) == 4 ? 5 : 6;
// the same for blocks of 128 rows: 4096 x 8192 bf16 18.7 us at 4 CTAs per SM (5.4 TB/s), 19.7 at 3, 22.9 at 5, 25.7 at 6;
// fp32 35.7 at 2 (4.7 TB/s), 35.4 at 1, 41.6 at 3, 49.3 at 4, and 1000 x 2048 4.5 at 2 and 1, 5.2 at 3
template <typename T>
constexpr int kBlocksBlocks = sizeof(T) == 4 ? 2 : 4;

template <typename T, typename I>
__global__ void __launch_bounds__(256, kRowsBlocks<T>) fp8_rows_kernel(const T* __restrict__ x, I n, I G, int64_t K, int64_t ldx,
                                                                    int vec, uint8_t* __restrict__ codes, int64_t ldc,
                                                                    float* __restrict__ scale) {
  pdl_wait();
  const int l = threadIdx.x & 7;
  const I stride = static_cast<I>(gridDim.x) * (blockDim.x >> 3);
  const I i0 = static_cast<I>(blockIdx.x) * (blockDim.x >> 3) + (threadIdx.x >> 3);
  const I rows = stride / G, rest = stride - rows * G;
  I m = i0 / G, g = i0 - m * G;  // group g of row m
#pragma unroll 1
  for (I i = i0; i - (threadIdx.x >> 3 & 3) < n; i += stride) {  // a warp's four groups leave the loop together
    const int64_t c = i < n ? static_cast<int64_t>(g) * BLK + 16 * l : K;
    Raw16<T> raw;
    raw.load(x + (i < n ? static_cast<int64_t>(m) * ldx : 0), c, K, vec != 0);
    uint32_t b = raw.top();
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    const float amax = group_amax(b);
    uint32_t w[4];
    raw.codes(amax, Divider(amax), w);
    store16(codes + static_cast<int64_t>(m) * ldc, c, K, w);
    if (l == 0 && i < n) scale[i] = group_scale(amax);
    m += rows;
    g += rest;
    if (g >= G) {
      g -= G;
      ++m;
    }
  }
}

// One scale per 128 x 128 block: a CTA per block, 8 lanes a row, 32 rows of 4 passes; the values wait in registers for
// the block's maximum.
template <typename T>
__global__ void __launch_bounds__(256, kBlocksBlocks<T>) fp8_blocks_kernel(const T* __restrict__ x, int64_t M, int64_t K,
                                                                          int64_t ldx, int vec, uint32_t G,
                                                                          uint8_t* __restrict__ codes, int64_t ldc,
                                                                          float* __restrict__ scale) {
  pdl_wait();
  __shared__ uint32_t red[8];
  const uint32_t mb = blockIdx.x / G, g = blockIdx.x - mb * G;
  const int64_t c = static_cast<int64_t>(g) * BLK + 16 * (threadIdx.x & 7);
  const int64_t m0 = static_cast<int64_t>(mb) * BLK + (threadIdx.x >> 3);
  Raw16<T> raw[4];
  uint32_t b = 0;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t m = m0 + p * 32;
    raw[p].load(x + (m < M ? m : 0) * ldx, m < M ? c : K, K, vec != 0);
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) b = max(b, raw[p].top());
  b = __reduce_max_sync(0xffffffffu, b);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = b;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) b = max(b, red[j]);
  const float amax = group_amax(b);
  const Divider div(amax);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t m = m0 + p * 32;
    uint32_t w[4];
    raw[p].codes(amax, div, w);
    store16(codes + m * ldc, m < M ? c : K, K, w);
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

struct Codes {};  // tag: x holds e4m3 codes

// Rows of x as the columns of mma.sync m16n8k16 (NB blocks of 8), 16 weight rows per CTA as its rows; W warps split K
// by 128-groups and hold the next group's codes while they work on one.  e4m3 is exact in fp16, so the products are
// exact and sums are fp32.  The order of K within a group is free as long as both sides agree: lane t of a quad
// has bytes 16 t and 64 + 16 t of a group's 128, so that a quad reads 64 bytes at once.
// T other than Codes (NB = 1): every CTA quantizes the rows for itself into shared memory, which saves a launch.
// The weight's bytes bound it, with a start of about 2 us: 8 x 8192 x 4096 takes 8.5 us (4.0 TB/s), 8 x 4096 x 14336 12.5 (4.7
// TB/s), both with weights from HBM; one token 2048 x 2048 with its quantization 2.5 with weights in L2, 3.2 from HBM.
template <int W, int NB>
constexpr int kFewRed = W * 16 * (NB * 8 + 1) * 4;

__host__ __device__ constexpr int few_pitch(int G) { return G * BLK + 64; }  // 8 rows' 64 bytes in different banks

template <typename T, int W, int NB, int CTAS>
__global__ void __launch_bounds__(W * 32, CTAS) fp8_few_rows_kernel(const LinArgs a) {
  constexpr bool kCodes = std::is_same<T, Codes>::value;
  extern __shared__ __align__(16) uint8_t few_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  const int n0 = blockIdx.x * 16;
  const uint8_t* pw[2] = {a.w + min(n0 + g, a.N - 1) * a.ldw + 16 * t, a.w + min(n0 + g + 8, a.N - 1) * a.ldw + 16 * t};
  const float* ws = a.ws + static_cast<int64_t>(n0 / BLK) * a.G;
  const int pitch = few_pitch(a.G);
  float* sscale = reinterpret_cast<float*>(few_smem + 8 * pitch);  // [8][G]
  float acc[NB][4] = {};
  uint4 wv[2][2], xv[NB][2];
  float wsc = 0.f, xsc[NB][2];
  auto load = [&](int s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = s * BLK + 64 * j;
      const bool in = c + 16 * t < a.K;  // K is a multiple of 16
#pragma unroll
      for (int h = 0; h < 2; ++h) wv[h][j] = in ? load_once(pw[h] + c) : make_uint4(0, 0, 0, 0);
      if (kCodes)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          xv[b][j] = in && 8 * b + g < a.M
                         ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.x) + (8 * b + g) * a.ldx + c + 16 * t))
                         : make_uint4(0, 0, 0, 0);
    }
    wsc = s < a.G ? __ldg(ws + s) : 0.f;
    if (kCodes)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int m = 8 * b + 2 * t + i;
          xsc[b][i] = s < a.G && m < a.M ? __ldg(a.xs + static_cast<int64_t>(m) * a.G + s) : 0.f;
        }
  };
  load(warp);
  if constexpr (!kCodes) {
    const int l = threadIdx.x & 7, n = static_cast<int>(a.M) * a.G;
#pragma unroll 1
    for (int i = threadIdx.x >> 3; i - (threadIdx.x >> 3 & 3) < n; i += W * 4) {
      const int m = i < n ? i / a.G : 0, s = i - m * a.G;
      Raw16<T> raw;
      raw.load(static_cast<const T*>(a.x) + m * a.ldx, i < n ? s * BLK + 16 * l : a.K, a.K, a.vec != 0);
      uint32_t b = raw.top();
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
      const float amax = group_amax(b);
      uint32_t w[4];
      raw.codes(amax, Divider(amax), w);
      if (i < n) *reinterpret_cast<uint4*>(few_smem + m * pitch + s * BLK + 16 * l) = make_uint4(w[0], w[1], w[2], w[3]);
      if (l == 0 && i < n) sscale[i] = group_scale(amax);
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int s = warp; s < a.G; s += W) {
    if (!kCodes) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        xv[0][j] = g < a.M ? *reinterpret_cast<const uint4*>(few_smem + g * pitch + s * BLK + 64 * j + 16 * t)
                           : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 2; ++i) xsc[0][i] = 2 * t + i < a.M ? sscale[(2 * t + i) * a.G + s] : 0.f;
    }
    float d[NB][4] = {};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a0, a1, a2, a3;
        codes_to_f16(reinterpret_cast<const uint32_t*>(&wv[0][j])[k], a0, a2);
        codes_to_f16(reinterpret_cast<const uint32_t*>(&wv[1][j])[k], a1, a3);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t b0, b1;
          codes_to_f16(reinterpret_cast<const uint32_t*>(&xv[b][j])[k], b0, b1);
          mma_f16(d[b], a0, a1, a2, a3, b0, b1);
        }
      }
    }
    float f[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) f[b][i] = __fmul_rn(xsc[b][i], wsc);
    load(s + W);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[b][e] = __fmaf_rn(f[b][e & 1], d[b][e], acc[b][e]);
  }
  if (!kCodes) __syncthreads();  // the parts go over the codes
  float(*red)[16][NB * 8 + 1] = reinterpret_cast<float(*)[16][NB * 8 + 1]>(few_smem);
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][g + 8 * (e >> 1)][8 * b + 2 * t + (e & 1)] = acc[b][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * NB * 8; i += W * 32) {
    const int r = i % 16, m = i / 16, n = n0 + r;
    if (n >= a.N || m >= a.M) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v = __fadd_rn(v, red[w][r][m]);
    if (a.bias != nullptr) v = __fadd_rn(v, load_as_f32(a.bias, a.out_type, n));
    store_from_f32(a.out, a.out_type, static_cast<int64_t>(m) * a.N + n, v);
  }
}

template <typename T, int W, int NB, int CTAS>
int launch_few(const LinArgs& a, cudaStream_t st) {
  int smem = kFewRed<W, NB>;
  if (!std::is_same<T, Codes>::value) smem = std::max(smem, 8 * few_pitch(a.G) + 32 * a.G);
  if (smem > 48 * 1024) {
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = once_per_device(ready, [] {
      return cudaFuncSetAttribute(fp8_few_rows_kernel<T, W, NB, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  8 * few_pitch(kOwnK / BLK) + 32 * static_cast<int>(kOwnK / BLK));
    });
    if (e != cudaSuccess) return fail(LLQ_ECUDA, "fp8_few_rows_kernel: %s", cudaGetErrorString(e));
  }
  launch_pdl(fp8_few_rows_kernel<T, W, NB, CTAS>, dim3((a.N + 15) / 16), dim3(W * 32), smem, st, a);
  return check_launch("fp8_few_rows_kernel");
}

// Up to 8 rows.  16 warps share a CTA's 16 weight rows, two CTAs per SM; where these do not fit at once, 8 warps and four CTAs (us,
// 16 warps / 8 warps: 8 x 2048 x 2048 2.6 / 2.7, 8 x 4096 x 14336 12.5 / 16.2, 8 x 5120 x 4096 7.5 / 6.9, 8 x 16384 x 2048 10.6 / 9.2,
// 1 x 8192 x 2048 with its quantization 7.3 / 5.9).
template <typename T>
int launch_eight(const LinArgs& a, cudaStream_t st) {
  if (a.N > 32 * num_sms()) return launch_few<T, 8, 1, 4>(a, st);
  return launch_few<T, 16, 1, 2>(a, st);
}

template <typename T>
int launch_rows(const void* x, int64_t M, int64_t K, int64_t ldx, int block_rows, uint8_t* codes, int64_t ldc, float* scale,
                cudaStream_t st) {
  const int vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * sizeof(T)) % 16 == 0;
  const int64_t G = (K + BLK - 1) / BLK;
  if (block_rows == 1) {
    const int64_t n = M * G;
    int64_t blocks = (n + 31) / 32;
    const int64_t most = static_cast<int64_t>(num_sms()) * kRowsBlocks<T>;
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
             static_cast<const T*>(x), M, K, ldx, vec, static_cast<uint32_t>(G), codes, ldc, scale);
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

// Does the product run on fp8_few_rows_kernel (else on fp8_tc_kernel)?  Up to 8 rows it is faster, from 9 to 16 with all but the
// largest weights, where the rule costs up to 9 % (us: 8 x 2048 x 2048 2.4 against 6.4, 8 x 8192 x 4096 8.6 against 11, 16 x 4096 x 4096 6.9 against 10.3, 16 x 8192 x 4096 12.0
// against 11.0, 16 x 4096 x 14336 17.2 against 18.2); with 32, where a CTA reads more of x than of the weight, for few
// and small weight rows, at the end of that range 5 % slower (32 x 2048 x 2048 4.4 against 6.4, 32 x 2048 x 4096 7.2 against 8.1, 32 x 4096 x 2048 6.7 against 6.4, 32 x
// 8192 x 1024 7.9 against 4.7, 32 x 8192 x 4096 18.5 against 11.0).
static bool few_rows(int64_t M, int64_t K, int64_t N) { return M <= 16 || (M <= 32 && N <= 4096 && N * K <= 1 << 24); }

// Do its CTAs quantize the rows for themselves?  Each does all of them again, N / 16 times together, which beats a launch for
// few values (1 x 1024 x 1024 2.2 us against 3.1, 8 x 2048 x 2048 4.0 against 4.2, 1 x 3000 x 7168 9.1 against 10.1) and not
// for many (1 x 8192 x 4096 9.4 against 9.5, 8 x 8192 x 4096 20.0 against 10.0).
static bool few_quantizes(int64_t M, int64_t K, int64_t N) {
  return M <= 8 && K <= kOwnK && M * K * ((N + 15) / 16) <= 1 << 21;
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
  if (K > 1 << 30) return fail(LLQ_EINVAL, "K too large");
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
  const bool own = x_dtype != LLQ_E4M3 && few_quantizes(M, K, N);  // the product's own kernel quantizes the rows
  const uint8_t* codes = static_cast<const uint8_t*>(x);
  if (x_dtype != LLQ_E4M3 && !own) {  // quantized once into the workspace
    const size_t need = fp8_linear_workspace(M, K, N, x_dtype);
    if (workspace == nullptr || bytes < need) return fail(LLQ_ENOSPACE, "workspace needs %zu bytes, got %zu", need, bytes);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(LLQ_EINVAL, "the workspace needs 16-byte alignment");
    uint8_t* to = static_cast<uint8_t*>(workspace);
    float* scale = reinterpret_cast<float*>(to + static_cast<size_t>(M) * K);
    const int rc = fp8_quantize(x, x_dtype, M, K, ldx, 1, to, K, scale, st);
    if (rc) return rc;
    codes = to;
    x_scale = scale;
    ldx = K;
  }
  if (!few_rows(M, K, N)) {
    Fp8Operands p{};
    p.x = codes;
    p.xs = x_scale;
    p.ldx = ldx;
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
  a.x = own ? x : codes;
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
  if (!own) {
    if (M > 16) return launch_few<Codes, 8, 4, 2>(a, st);
    if (M > 8) return launch_few<Codes, 8, 2, 2>(a, st);
    return launch_eight<Codes>(a, st);
  }
  switch (x_dtype) {
    case LLQ_F32: return launch_eight<float>(a, st);
    case LLQ_F16: return launch_eight<__half>(a, st);
    default: return launch_eight<__nv_bfloat16>(a, st);
  }
}

// codes [M][K] (K is a multiple of 16) and scales [M][G] of rows that are quantized before the tensor-core product
size_t fp8_linear_workspace(int64_t M, int K, int N, int x_dtype) {
  if (M < 1 || K < 1 || x_dtype == LLQ_E4M3 || few_quantizes(M, K, N)) return 0;
  return static_cast<size_t>(M) * K + static_cast<size_t>(M) * ((K + BLK - 1) / BLK) * 4;
}

}  // namespace llq
