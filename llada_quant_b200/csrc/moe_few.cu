// The PACKED MoE layer for at most 32 tokens, in two kernels.
//
//   z[t,e] = x[t] . gate[e] (+ bias[e])            fp32, never rounded to fewer bits
//   p = softmax(z[t]), the k largest z, ties to the lower expert, weight p or p / sum of the k
//   a = W1[e, n] . x[t],  b = W1[e, I + n] . x[t]   W = q * s in fp32, no bf16 rounding of a weight
//   h[t,e,n] = a / (1 + exp(-a)) * b * (weight of e in t)
//   out[t] = bf16(sum over the experts of t, ascending, of W2[e] . h[t,e])
//
// What bounds it: the packed bytes of the experts that some token chose, read once from HBM (one
// token of a 64-expert, 2048 x 1024, top-8 INT4 layer: 26.7 MB, 4.1 us at 6.55 TB/s).  There are
// too few tokens to fill a tcgen05 tile (8 of 64 experts get one token each), so the products run
// on mma.sync m16n8k16 with the weights as the 16 rows and up to 8 tokens as the columns, and the
// packed bytes go from HBM straight to the registers of the lane that feeds them to the MMA: a
// lane's 16 (INT4) or 32 (INT8) bytes of a row are its k slots of the 8 MMAs of one 128-group, so
// no shared memory, no transpose and no repacking stands between load and MMA.  The integer codes
// are exact in bf16; each group's partial sum is multiplied by the group's scale in fp32.
//
// Kernel 1 (router, GEMM1): the clusters of 8 CTAs each compute the whole router (256 KB of gate,
// an eighth per CTA, exchanged through distributed shared memory), so no grid-wide wait stands
// between router and experts.  A warp then takes 16-row tiles of 8 gate and the matching 8 up rows,
// so that SiLU(a) * b is local to a thread.
// Kernel 2 (GEMM2, combine): a cluster of 8 CTAs owns 128 output features and splits the list of
// (chosen expert, 128-group) steps evenly; the partial outputs meet in distributed shared memory
// and are added in rank order, so no atomics and a fixed order of sums.
// h travels between them as two bf16 numbers, hi + lo (17 significant bits), so that the bf16 MMAs
// add no visible rounding: the layer rounds once, at its end.
#include <cooperative_groups.h>

#include "llq_common.cuh"
#include "llq_internal.cuh"

namespace llq {

namespace {

namespace cg = cooperative_groups;

constexpr int MAX_T = 32;     // a token is a bit of an expert's 32-bit mask
constexpr int MAX_EXP = 256;
constexpr int MAX_K = 32;
constexpr int CL = 8;         // CTAs of a cluster (the largest portable size)
constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int KG = 128;       // K elements of a step: 32 for each of a quad's four lanes

// what kernel 1 tells kernel 2 about the routing
struct FewPlan {
  int32_t nhit;               // experts that some token chose
  int32_t expert[MAX_EXP];    // their ids, ascending
  int32_t row[MAX_EXP + 1];   // first row of h of each
  uint32_t mask[MAX_EXP];     // their tokens
};

struct FewArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* gate;
  const float* bias;
  int renormalize;
  int T, E, H, I, k;
  const int8_t* q1;
  const float* s1;
  const int8_t* q2;
  const float* s2;
  int groups1, gsteps1;  // scales per row of w1, 128-steps per scale (0: one scale per row)
  int groups2, gsteps2;
  float* logits;
  float* topk_w;
  int32_t* topk_ids;
  FewPlan* plan;
  __nv_bfloat16* h_hi;
  __nv_bfloat16* h_lo;
  int h_pitch;
  __nv_bfloat16* out;
};

// D += A (16 x 16, rows) * B (16 x 8, columns), bf16 in, fp32 sums.  Lane (g = lane / 4, t = lane % 4)
// holds of A the k pairs (2t, 2t+1) and (2t+8, 2t+9) of rows g (a0, a2) and g + 8 (a1, a3), of B the
// same pairs of column g, of D the columns 2t, 2t+1 of rows g (d0, d1) and g + 8 (d2, d3).
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// weights pass through once: no L1 line is kept for them
__device__ __forceinline__ uint4 load_weights(const int8_t* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}

// two int4 codes of a word (nibbles j and j + 4, j the shift / 4) as a bf16 pair: the xor puts
// q + 8 into the low mantissa bits of 128, and 128 + 8 is subtracted exactly
__device__ __forceinline__ uint32_t int4_pair(uint32_t w) {
  uint32_t t, o;
  asm("lop3.b32 %0, %1, 0x000F000F, 0x43084308, 0x6A;" : "=r"(t) : "r"(w));
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(o) : "r"(t), "r"(0xC308C308u));
  return o;
}

// two int8 codes, one in the low byte of each half: the low seven bits in the mantissa of 128, minus
// 128 (code >= 0) or 256 (code < 0: its sign bit is the exponent step between the two)
__device__ __forceinline__ uint32_t int8_pair(uint32_t b) {
  uint32_t m, c, o;
  asm("lop3.b32 %0, %1, 0x007F007F, 0x43004300, 0xEA;" : "=r"(m) : "r"(b));
  asm("lop3.b32 %0, %1, 0x00800080, 0xC300C300, 0xEA;" : "=r"(c) : "r"(b));
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(o) : "r"(m), "r"(c));
  return o;
}

// one row's 32 codes of a lane
template <int BITS>
struct Codes {
  uint4 v[BITS == 4 ? 1 : 2];
  __device__ __forceinline__ void load(const int8_t* p) {
#pragma unroll
    for (int i = 0; i < (BITS == 4 ? 1 : 2); ++i) v[i] = load_weights(p + 16 * i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (BITS == 4 ? 1 : 2); ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  // codes 8j .. 8j + 7 as four bf16 pairs: INT4 (0,4) (1,5) (2,6) (3,7), INT8 (0,1) (2,3) (4,5) (6,7)
  __device__ __forceinline__ void pairs(int j, uint32_t (&p)[4]) const {
    if (BITS == 4) {
      const uint32_t w = j == 0 ? v[0].x : j == 1 ? v[0].y : j == 2 ? v[0].z : v[0].w;
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = int4_pair(w >> (4 * i));
    } else {
      const uint4 u = v[j >> 1];
      const uint32_t w0 = (j & 1) ? u.z : u.x, w1 = (j & 1) ? u.w : u.y;
      p[0] = int8_pair(__byte_perm(w0, 0, 0x4140));
      p[1] = int8_pair(__byte_perm(w0, 0, 0x4342));
      p[2] = int8_pair(__byte_perm(w1, 0, 0x4140));
      p[3] = int8_pair(__byte_perm(w1, 0, 0x4342));
    }
  }
};

// 8 bf16 of a token in natural order -> the pairs of Codes::pairs
template <int BITS>
__device__ __forceinline__ void token_pairs(uint4 x, uint32_t (&p)[4]) {
  if (BITS == 4) {
    p[0] = __byte_perm(x.x, x.z, 0x5410);
    p[1] = __byte_perm(x.x, x.z, 0x7632);
    p[2] = __byte_perm(x.y, x.w, 0x5410);
    p[3] = __byte_perm(x.y, x.w, 0x7632);
  } else {
    p[0] = x.x;
    p[1] = x.y;
    p[2] = x.z;
    p[3] = x.w;
  }
}

// position of feature n of h in the order of Codes::pairs
template <int BITS>
__device__ __forceinline__ int pair_pos(int n) {
  if (BITS != 4) return n;
  const int j = n & 7;
  return (n & ~7) | (j < 4 ? 2 * j : 2 * j - 7);
}

// the i-th set bit of m, or -1
__device__ __forceinline__ int nth_bit(uint32_t m, int i) {
  const uint32_t p = __fns(m, 0, i + 1);
  return p == 0xffffffffu ? -1 : static_cast<int>(p);
}

// unsigned key that orders floats as their values; NaN lowest
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t b = __float_as_uint(z);
  if (!(z == z)) return 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct Smem1 {
  float logit[MAX_EXP][MAX_T];   // z; then the weight of expert e in token t
  union {
    float red[WARPS][8][MAX_T];  // router: a tile of 8 experts, one K slice per warp
    struct {
      float w[MAX_T][MAX_K];     // the routing, as the caller brings it or gets it
      int32_t ids[MAX_T][MAX_K];
    };
  };
  uint32_t mask[MAX_EXP];
  int32_t expert[MAX_EXP];
  int32_t row[MAX_EXP + 1];
  int32_t nhit;
};

// the router: this CTA's experts (8 at a time) against all tokens, into every CTA of the cluster
__device__ void router_logits(const FewArgs& a, Smem1& sm, cg::cluster_group& cluster) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ntiles = (a.T + 7) / 8;
  const int rank = static_cast<int>(cluster.block_rank());
  for (int e0 = rank * 8; e0 < a.E; e0 += CL * 8) {
    float d[MAX_T / 8][4];
#pragma unroll
    for (int n = 0; n < MAX_T / 8; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
    const int e = e0 + g;
    for (int c = warp * 32; c < a.H; c += WARPS * 32) {
      const uint4 w = e < a.E ? __ldg(reinterpret_cast<const uint4*>(a.gate + static_cast<int64_t>(e) * a.H + c + 8 * t))
                              : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int n = 0; n < MAX_T / 8; ++n) {
        if (n < ntiles) {
          const int tok = n * 8 + g;
          const uint4 x = tok < a.T ? __ldg(reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(tok) * a.H + c + 8 * t))
                                    : make_uint4(0, 0, 0, 0);
          mma_bf16(d[n], w.x, 0, w.y, 0, x.x, x.y);
          mma_bf16(d[n], w.z, 0, w.w, 0, x.z, x.w);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < MAX_T / 8; ++n) {
      sm.red[warp][g][n * 8 + 2 * t] = d[n][0];
      sm.red[warp][g][n * 8 + 2 * t + 1] = d[n][1];
    }
    __syncthreads();
    const int r = threadIdx.x / MAX_T, tok = threadIdx.x % MAX_T;  // 8 experts x 32 tokens
    if (e0 + r < a.E && tok < a.T) {
      float z = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) z = __fadd_rn(z, sm.red[w][r][tok]);
      if (a.bias != nullptr) z = __fadd_rn(z, a.bias[e0 + r]);
#pragma unroll
      for (int c = 0; c < CL; ++c) *cluster.map_shared_rank(&sm.logit[e0 + r][tok], c) = z;
      if (a.logits != nullptr && blockIdx.x < CL) a.logits[static_cast<int64_t>(tok) * a.E + e0 + r] = z;
    }
    __syncthreads();
  }
}

// softmax and top-k of one token by one warp, into sm.ids and sm.w
__device__ void choose(const FewArgs& a, Smem1& sm, int tok) {
  int32_t* ids = sm.ids[tok];
  float* ws = sm.w[tok];
  const int lane = threadIdx.x & 31;
  constexpr int PER = MAX_EXP / 32;
  float z[PER];
  float m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 32 * j;
    z[j] = e < a.E ? __fadd_rn(sm.logit[e][tok], 0.f) : -INFINITY;  // -0 ranks as +0
    bad |= !(z[j] == z[j]);
    m = fmaxf(m, z[j]);
  }
  m = warp_max(m);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) s = __fadd_rn(s, lane + 32 * j < a.E ? expf(z[j] - m) : 0.f);
  s = warp_sum(s);
  if (__any_sync(0xffffffffu, bad)) s = NAN;  // as softmax over a row with a NaN
  float total = 0.f;
  uint32_t taken = 0;  // bit j: this lane's expert lane + 32 j is chosen
  for (int i = 0; i < a.k; ++i) {
    uint32_t best = 0;
    int bj = -1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (lane + 32 * j < a.E && !((taken >> j) & 1u)) {
        const uint32_t key = order_key(z[j]);
        if (bj < 0 || key > best) {
          best = key;
          bj = j;
        }
      }
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, bj < 0 ? 0u : best);
    const int mine = (bj >= 0 && best == top) ? lane + 32 * bj : 0x7fffffff;
    const int e = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<uint32_t>(mine)));
    if (mine == e) taken |= 1u << bj;
    const float p = __fdiv_rn(expf(sm.logit[e][tok] - m), s);
    total = __fadd_rn(total, p);
    if (lane == 0) {
      ids[i] = e;
      ws[i] = p;
    }
  }
  __syncwarp();
  if (a.renormalize)
    for (int i = lane; i < a.k; i += 32) ws[i] = __fdiv_rn(ws[i], total);
}

template <int BITS>
__global__ void __launch_bounds__(THREADS, 2) few_gemm1_kernel(const FewArgs a) {
  __shared__ Smem1 sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();

  if (a.gate != nullptr) {
    router_logits(a, sm, cluster);
    cluster.sync();  // every CTA's logits are in every CTA
    for (int tok = warp; tok < a.T; tok += WARPS) choose(a, sm, tok);
    __syncthreads();
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i < a.T * a.k; i += THREADS) {
        a.topk_w[i] = sm.w[i / a.k][i % a.k];
        a.topk_ids[i] = sm.ids[i / a.k][i % a.k];
      }
    }
  } else {
    for (int i = threadIdx.x; i < a.T * a.k; i += THREADS) {
      sm.w[i / a.k][i % a.k] = a.topk_w[i];
      sm.ids[i / a.k][i % a.k] = a.topk_ids[i];
    }
  }
  // share[e][t]: sum of the token's weights of expert e; mask[e]: the tokens that chose it
  for (int i = threadIdx.x; i < a.E * MAX_T; i += THREADS) (&sm.logit[0][0])[i] = 0.f;
  for (int i = threadIdx.x; i < a.E; i += THREADS) sm.mask[i] = 0;
  __syncthreads();
  if (threadIdx.x < a.T) {
    const int tok = threadIdx.x;
    for (int i = 0; i < a.k; ++i) {
      const int e = sm.ids[tok][i];
      if (e >= 0 && e < a.E) {
        sm.logit[e][tok] = __fadd_rn(sm.logit[e][tok], sm.w[tok][i]);
        atomicOr(&sm.mask[e], 1u << tok);
      }
    }
  }
  __syncthreads();
  if (warp == 0) {  // the chosen experts, ascending, and their rows of h
    int n = 0, rows = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + lane;
      const uint32_t m = e < a.E ? sm.mask[e] : 0;
      const uint32_t hits = __ballot_sync(0xffffffffu, m != 0);
      int incl = __popc(m);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (m != 0) {
        const int at = n + __popc(hits & ((1u << lane) - 1));
        sm.expert[at] = e;
        sm.row[at] = rows + incl - __popc(m);
      }
      n += __popc(hits);
      rows += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      sm.nhit = n;
      sm.row[n] = rows;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < sm.nhit; i += THREADS) {
      a.plan->expert[i] = sm.expert[i];
      a.plan->row[i] = sm.row[i];
      a.plan->mask[i] = sm.mask[sm.expert[i]];
    }
    if (threadIdx.x == 0) a.plan->nhit = sm.nhit;
  }
  pdl_trigger();

  const int tiles = a.I / 8;
  const int units = sm.nhit * tiles;
  const int kb = a.H * BITS / 8;  // bytes of a row of w1
  const int steps = (a.H + KG - 1) / KG;
  for (int u = blockIdx.x + warp * gridDim.x; u < units; u += gridDim.x * WARPS) {
    const int hit = u / tiles, rb = u - hit * tiles;
    const int e = sm.expert[hit];
    const uint32_t mask = sm.mask[e];
    const int ntok = __popc(mask);
    const int64_t row_g = static_cast<int64_t>(e) * 2 * a.I + rb * 8 + g;  // gate row; up row I further
    const int8_t* pg = a.q1 + row_g * kb + t * (32 * BITS / 8);
    const int8_t* pu = pg + static_cast<int64_t>(a.I) * kb;
    const float* sg = a.s1 + row_g * a.groups1;
    const float* su = sg + static_cast<int64_t>(a.I) * a.groups1;
    for (int c0 = 0; c0 < ntok; c0 += 8) {
      const int tok = nth_bit(mask, c0 + g);
      const uint4* px = tok < 0 ? nullptr
                                : reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(tok) * a.H + 32 * t);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < steps; ++s) {
        const bool in = s * KG + 32 * t < a.H;  // H is a multiple of 32
        Codes<BITS> wg, wu;
        if (in) {
          wg.load(pg + s * (KG * BITS / 8));
          wu.load(pu + s * (KG * BITS / 8));
        } else {
          wg.zero();
          wu.zero();
        }
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 xv = (in && px != nullptr) ? __ldg(px + s * (KG / 8) + j) : make_uint4(0, 0, 0, 0);
          uint32_t ag[4], au[4], b[4];
          wg.pairs(j, ag);
          wu.pairs(j, au);
          token_pairs<BITS>(xv, b);
          mma_bf16(d, ag[0], au[0], ag[1], au[1], b[0], b[1]);
          mma_bf16(d, ag[2], au[2], ag[3], au[3], b[2], b[3]);
        }
        const int gi = a.gsteps1 == 0 ? 0 : s / a.gsteps1;
        const float f = sg[gi], v = su[gi];
        acc[0] = __fmaf_rn(f, d[0], acc[0]);
        acc[1] = __fmaf_rn(f, d[1], acc[1]);
        acc[2] = __fmaf_rn(v, d[2], acc[2]);
        acc[3] = __fmaf_rn(v, d[3], acc[3]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = c0 + 2 * t + i;
        if (col < ntok) {
          const float ga = acc[i], up = acc[2 + i];
          const float h = __fdiv_rn(ga, 1.f + expf(-ga)) * up * sm.logit[e][nth_bit(mask, col)];
          const __nv_bfloat16 hi = __float2bfloat16_rn(h);
          const int64_t at = static_cast<int64_t>(sm.row[hit] + col) * a.h_pitch + pair_pos<BITS>(rb * 8 + g);
          a.h_hi[at] = hi;
          a.h_lo[at] = __float2bfloat16_rn(h - __bfloat162float(hi));
        }
      }
    }
  }
}

constexpr int PANEL = WARPS * 16;  // output features of a cluster of kernel 2

template <int BITS>
__global__ void __launch_bounds__(THREADS, 2) few_gemm2_kernel(const FewArgs a) {
  __shared__ float part[PANEL][MAX_T + 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(cluster.block_rank());
  const int panel = blockIdx.x / CL;
  for (int i = threadIdx.x; i < PANEL * (MAX_T + 1); i += THREADS) (&part[0][0])[i] = 0.f;
  pdl_wait();
  __syncthreads();

  const int steps = (a.I + KG - 1) / KG;
  const int kb = a.I * BITS / 8;
  const int total = a.plan->nhit * steps;
  const int begin = static_cast<int>(static_cast<int64_t>(total) * rank / CL);
  const int end = static_cast<int>(static_cast<int64_t>(total) * (rank + 1) / CL);
  const int r0 = warp * 16 + g, r1 = r0 + 8;  // this lane's rows of the panel
  const int n0 = min(panel * PANEL + r0, a.H - 1), n1 = min(panel * PANEL + r1, a.H - 1);
  const bool alive = panel * PANEL + warp * 16 < a.H;
  for (int at = begin; at < end && alive;) {
    const int hit = at / steps, s0 = at - hit * steps;
    const int s1 = min(steps, s0 + end - at);
    const int e = a.plan->expert[hit];
    const uint32_t mask = a.plan->mask[hit];
    const int ntok = __popc(mask);
    const int64_t row0 = static_cast<int64_t>(e) * a.H + n0, row1 = static_cast<int64_t>(e) * a.H + n1;
    const int8_t* p0 = a.q2 + row0 * kb + t * (32 * BITS / 8);
    const int8_t* p1 = a.q2 + row1 * kb + t * (32 * BITS / 8);
    const float* f0 = a.s2 + row0 * a.groups2;
    const float* f1 = a.s2 + row1 * a.groups2;
    for (int c0 = 0; c0 < ntok; c0 += 8) {
      const bool col_in = c0 + g < ntok;
      const int64_t hrow = static_cast<int64_t>(a.plan->row[hit] + c0 + g) * a.h_pitch + 32 * t;
      const uint4* ph = reinterpret_cast<const uint4*>(a.h_hi + hrow);
      const uint4* pl = reinterpret_cast<const uint4*>(a.h_lo + hrow);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int s = s0; s < s1; ++s) {
        const bool in = s * KG + 32 * t < a.I;
        Codes<BITS> w0, w1;
        if (in) {
          w0.load(p0 + s * (KG * BITS / 8));
          w1.load(p1 + s * (KG * BITS / 8));
        } else {
          w0.zero();
          w1.zero();
        }
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 hv = make_uint4(0, 0, 0, 0), lv = hv;
          if (in && col_in) {
            hv = ph[s * (KG / 8) + j];
            lv = pl[s * (KG / 8) + j];
          }
          uint32_t a0[4], a1[4];
          w0.pairs(j, a0);
          w1.pairs(j, a1);
          mma_bf16(d, a0[0], a1[0], a0[1], a1[1], hv.x, hv.y);
          mma_bf16(d, a0[2], a1[2], a0[3], a1[3], hv.z, hv.w);
          mma_bf16(d, a0[0], a1[0], a0[1], a1[1], lv.x, lv.y);
          mma_bf16(d, a0[2], a1[2], a0[3], a1[3], lv.z, lv.w);
        }
        const int gi = a.gsteps2 == 0 ? 0 : s / a.gsteps2;
        const float f = f0[gi], v = f1[gi];
        acc[0] = __fmaf_rn(f, d[0], acc[0]);
        acc[1] = __fmaf_rn(f, d[1], acc[1]);
        acc[2] = __fmaf_rn(v, d[2], acc[2]);
        acc[3] = __fmaf_rn(v, d[3], acc[3]);
      }
      // rows belong to this warp alone, and the tokens of an expert are distinct
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = c0 + 2 * t + i;
        if (col < ntok) {
          const int tok = nth_bit(mask, col);
          part[r0][tok] += acc[i];
          part[r1][tok] += acc[2 + i];
        }
      }
      __syncwarp();
    }
    at += s1 - s0;
  }
  cluster.sync();
  // 16 rows of the panel per CTA of the cluster
  for (int i = threadIdx.x; i < 16 * a.T; i += THREADS) {
    const int r = rank * 16 + (i & 15), tok = i >> 4;
    float v = 0.f;
#pragma unroll
    for (int c = 0; c < CL; ++c) v = __fadd_rn(v, *cluster.map_shared_rank(&part[r][tok], c));
    if (panel * PANEL + r < a.H)
      a.out[static_cast<int64_t>(tok) * a.H + panel * PANEL + r] = __float2bfloat16_rn(v);
  }
  cluster.sync();  // the others may still read this CTA's part
}

template <typename K>
int launch_cluster(K kernel, int grid, cudaStream_t st, const FewArgs& a, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CL;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(LLQ_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  return LLQ_OK;
}

template <int BITS>
int launch_few(const FewArgs& a, cudaStream_t st) {
  const int grid = num_sms() * 2 / CL * CL;
  int rc = launch_cluster(few_gemm1_kernel<BITS>, grid, st, a, "few_gemm1_kernel");
  if (rc) return rc;
  return launch_cluster(few_gemm2_kernel<BITS>, (a.H + PANEL - 1) / PANEL * CL, st, a, "few_gemm2_kernel");
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

inline bool few_group_ok(int K, int group) { return group <= 0 || K % group != 0 || group % KG == 0; }

}  // namespace

size_t moe_few_workspace(int64_t T, int k, int I) {
  if (T < 1 || k < 1 || I < 1) return 0;
  const size_t pitch = (static_cast<size_t>(I) + 7) / 8 * 8;
  return up256(sizeof(FewPlan)) + 2 * up256(static_cast<size_t>(T) * k * pitch * 2);
}

int moe_few(const llq_few_layer& L, const void* x, int64_t T, float* logits, float* topk_w, int32_t* topk_ids,
            void* out, void* workspace, size_t bytes, cudaStream_t st) {
  if (T < 0 || L.E < 1 || L.H < 1 || L.I < 1 || L.k < 1 || L.k > L.E)
    return fail(LLQ_EINVAL, "bad shape T=%lld E=%d H=%d I=%d k=%d", (long long)T, L.E, L.H, L.I, L.k);
  if (L.bits != 4 && L.bits != 8) return fail(LLQ_EUNSUPPORTED, "bits must be 8 or 4, got %d", L.bits);
  if (T > MAX_T) return fail(LLQ_EUNSUPPORTED, "the few-token layer takes at most %d tokens, got %lld", MAX_T, (long long)T);
  if (L.E > MAX_EXP || L.k > MAX_K) return fail(LLQ_EUNSUPPORTED, "the few-token layer takes E <= 256 and k <= 32");
  if (L.H % 32 != 0 || L.I % 32 != 0 || L.H > 32768 || L.I > 32768)
    return fail(LLQ_EUNSUPPORTED, "the few-token layer needs H and I in multiples of 32, at most 32768 (H=%d I=%d)", L.H, L.I);
  if (!few_group_ok(L.H, L.group_size) || !few_group_ok(L.I, L.group_size))
    return fail(LLQ_EUNSUPPORTED, "the few-token layer needs a group size in multiples of 128, got %d", L.group_size);
  if (T == 0) return LLQ_OK;
  if (x == nullptr || out == nullptr || topk_w == nullptr || topk_ids == nullptr || L.qw1 == nullptr ||
      L.sw1 == nullptr || L.qw2 == nullptr || L.sw2 == nullptr)
    return fail(LLQ_EINVAL, "null pointer");
  const uintptr_t al = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(L.gate_w) |
                       reinterpret_cast<uintptr_t>(L.qw1) | reinterpret_cast<uintptr_t>(L.qw2) |
                       reinterpret_cast<uintptr_t>(workspace);
  if (al & 15) return fail(LLQ_EINVAL, "x, gate_w, the packed weights and the workspace need 16-byte alignment");
  const size_t need = moe_few_workspace(T, L.k, L.I);
  if (workspace == nullptr || bytes < need)
    return fail(LLQ_ENOSPACE, "workspace needs %zu bytes, got %zu", need, bytes);
  FewArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.gate = static_cast<const __nv_bfloat16*>(L.gate_w);
  a.bias = L.bias;
  a.renormalize = L.renormalize;
  a.T = static_cast<int>(T);
  a.E = L.E;
  a.H = L.H;
  a.I = L.I;
  a.k = L.k;
  a.q1 = L.qw1;
  a.s1 = L.sw1;
  a.q2 = L.qw2;
  a.s2 = L.sw2;
  const bool g1 = L.group_size > 0 && L.H % L.group_size == 0, g2 = L.group_size > 0 && L.I % L.group_size == 0;
  a.groups1 = g1 ? L.H / L.group_size : 1;
  a.gsteps1 = g1 ? L.group_size / KG : 0;
  a.groups2 = g2 ? L.I / L.group_size : 1;
  a.gsteps2 = g2 ? L.group_size / KG : 0;
  a.logits = logits;
  a.topk_w = topk_w;
  a.topk_ids = topk_ids;
  char* ws = static_cast<char*>(workspace);
  a.plan = reinterpret_cast<FewPlan*>(ws);
  a.h_pitch = (L.I + 7) / 8 * 8;
  const size_t plane = up256(static_cast<size_t>(T) * L.k * a.h_pitch * 2);
  a.h_hi = reinterpret_cast<__nv_bfloat16*>(ws + up256(sizeof(FewPlan)));
  a.h_lo = reinterpret_cast<__nv_bfloat16*>(ws + up256(sizeof(FewPlan)) + plane);
  a.out = static_cast<__nv_bfloat16*>(out);
  return L.bits == 4 ? launch_few<4>(a, st) : launch_few<8>(a, st);
}

}  // namespace llq
