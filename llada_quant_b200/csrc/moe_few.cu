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
// on mma.sync m16n8k16 with the weights as the 16 rows and up to 8 tokens as the columns: a lane's
// 16 (INT4) or 32 (INT8) contiguous bytes of a row are its k slots of the 8 MMAs of one 128-group,
// so nothing is transposed or repacked between memory and MMA.  The integer codes become exact
// 16-bit numbers; each group's partial sum is multiplied by the group's scale in fp32.
//
// Kernel 1 (router, GEMM1): each cluster of 2 CTAs computes the whole router (half of K per CTA,
// exchanged through distributed shared memory), so no grid-wide wait stands between router and
// experts.  The work is a list of segments (expert, up to 8 of its tokens), each of I / 8 jobs: 8
// gate and the 8 up rows, so that SiLU(a) * b is local to a thread.  The CTAs take equal runs of jobs.
// Kernel 2 (GEMM2, combine): the CTAs of a panel of 128 output features split the list of (segment,
// 128-group) steps evenly; each stores its partial outputs, and the one that finishes last adds them
// in the order of the steps: no waits, and a fixed order of sums.
// The tokens enter kernel 1 as fp16, each 128-group scaled by a power of two so that its largest
// magnitude lies in [2^14, 2^15): exact for every bf16 value within 2^-31 of the largest, and what is
// lost below is 2^-40 of it.  (fp16 rather than bf16 because its ten mantissa bits take an INT8 code, or
// the upper nibble of a byte, where it lies: 40 instead of 56 logic instructions per lane and 128-group at
// INT4, 48 instead of 96 at INT8; the logic pipe is what bounds the arithmetic.)  h travels between the
// kernels as two bf16 numbers, hi + lo (16 significant bits).  So no MMA adds a visible rounding: the
// layer rounds once, at its end.
//
// The packed bytes and their scales reach shared memory by TMA (swizzled) into rings that are deep
// enough for HBM's latency; the tokens lie in shared memory in MMA order.  Measured on the way
// (32 tokens, INT4, both kernels): lanes loading their own bytes with cp.async and their tokens from L1,
// 132 us, bound by the L1 wavefronts that eight scattered rows per instruction cost; a register ring
// unrolled over its slots, 527 us, its code larger than the instruction cache; TMA rings whose refill one
// lane computed while its warp waited, 94 us.
#include <algorithm>

#include <cooperative_groups.h>

#include "llq_internal.cuh"
#include "tc_ptx.cuh"

namespace llq {

namespace {

namespace cg = cooperative_groups;

constexpr int MAX_T = 32;     // a token is a bit of an expert's 32-bit mask
constexpr int MAX_EXP = 256;
constexpr int MAX_K = 32;
constexpr int MAX_SEG = MAX_EXP + MAX_T * MAX_K / 8;
constexpr int CL1 = 2;        // CTAs of a cluster of kernel 1: all 148 SMs hold one (of 8, with this much
                              // shared memory, only 120 CTAs fit at once)
constexpr int WARPS = 16;
constexpr int THREADS = WARPS * 32;
constexpr int KG = 128;       // K elements of a step: 32 for each of a quad's four lanes

constexpr int MAX_SPLIT = 16;  // CTAs of a panel in kernel 2
constexpr int MAX_PANELS = 64;

// an expert and up to 8 of its tokens, ascending: the columns of its MMAs
struct Segment {
  int32_t expert, n;
  uint64_t tokens;  // a byte each
  __device__ __forceinline__ int token(int c) const { return static_cast<int>(tokens >> (8 * c)) & 0xff; }
};

// what kernel 1 tells kernel 2 about the routing
struct FewPlan {
  Segment seg[MAX_SEG];
  int32_t n;
  int32_t done[MAX_PANELS];  // kernel 2's CTAs that have stored their part of a panel
};

struct FewArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* gate;
  const float* bias;
  int renormalize;
  int T, E, H, I, k;
  const float* s1;
  const int8_t* q2;
  const float* s2;
  int groups1, gsteps1;  // scales per row of w1, 128-steps per scale (0: one scale per row)
  int groups2, gsteps2;
  int depth1;            // slots of a warp's ring in kernel 1
  int nbuf;              // segments whose tokens kernel 1 holds at a time
  int depth2;            // stages of a group's ring in kernel 2
  float* logits;
  float* topk_w;
  int32_t* topk_ids;
  FewPlan* plan;
  // [segment][step of I][plane][piece j of 4][lane], 4 KB a step: the B operand of kernel 2's MMAs.  Columns are the
  // segment's tokens; plane 0 holds the hi parts, plane 1 the lo parts, but with at most 4 tokens the lo parts are
  // columns 4 to 7 of plane 0 and half of the bytes and MMAs fall away.
  uint4* h;
  float* partial;        // [panel][split][128 features][T]
  int split;             // CTAs of a panel in kernel 2
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

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float lds4(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t and_xor(uint32_t x, uint32_t mask, uint32_t k) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(x), "r"(mask), "r"(k));
  return r;
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// Eight codes as four pairs of 16-bit numbers, exactly: INT4 (0,4) (1,5) (2,6) (3,7), INT8 (0,2) (1,3) (4,6) (5,7).
// fp16, for kernel 1.  INT4: the xor puts q + 8 into the low mantissa bits of 1024 (one is 1) or the next four (one is
// 16), and 1032, or a sixteenth and 72, bring it back.  INT8: the byte xor 128 is q + 128 in the mantissa of 1024.
__device__ __forceinline__ void pairs4_f16(uint32_t w, uint32_t (&p)[4]) {
  const uint32_t y = w >> 8;
  p[0] = add_f16x2(and_xor(w, 0x000F000Fu, 0x64086408u), 0xE408E408u);
  p[1] = fma_f16x2(and_xor(w, 0x00F000F0u, 0x64806480u), 0x2C002C00u, 0xD480D480u);
  p[2] = add_f16x2(and_xor(y, 0x000F000Fu, 0x64086408u), 0xE408E408u);
  p[3] = fma_f16x2(and_xor(y, 0x00F000F0u, 0x64806480u), 0x2C002C00u, 0xD480D480u);
}
__device__ __forceinline__ void pairs8_f16(uint32_t w, uint32_t& p0, uint32_t& p1) {
  const uint32_t x = w ^ 0x80808080u;
  p0 = add_f16x2(__byte_perm(x, 0x64646464u, 0x4240u), 0xE480E480u);
  p1 = add_f16x2(__byte_perm(x, 0x64646464u, 0x4341u), 0xE480E480u);
}
// bf16, for kernel 2, whose h has no bound that fp16 could be scaled by.  INT4: q + 8 in the low mantissa bits of 128.
// INT8: the low seven bits in the mantissa of 128, minus 128 (code >= 0) or 256 (code < 0: its sign bit is the
// exponent step between the two).
__device__ __forceinline__ void pairs4_bf16(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = add_bf16x2(and_xor(w >> (4 * i), 0x000F000Fu, 0x43084308u), 0xC308C308u);
}
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t k) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(k));
  return r;
}
__device__ __forceinline__ void pairs8_bf16(uint32_t w, uint32_t& p0, uint32_t& p1) {
  const uint32_t y = w >> 8;
  p0 = add_bf16x2(and_or(w, 0x007F007Fu, 0x43004300u), and_or(w, 0x00800080u, 0xC300C300u));
  p1 = add_bf16x2(and_or(y, 0x007F007Fu, 0x43004300u), and_or(y, 0x00800080u, 0xC300C300u));
}

// A lane's 32 codes of a row for one step, from rows of 128 bytes (128-byte swizzle).
template <int BITS>
struct Codes {
  static constexpr int STEPS = BITS == 4 ? 2 : 1;  // steps in 128 bytes
  uint4 v[BITS == 4 ? 1 : 2];
  // `row` is the address of row r (mod 8), `step` the step in it.  With row_of(g) as lane g's row
  // the eight lanes that a shared-memory access serves at a time (two rows) meet eight different 16-byte columns.
  static __device__ __forceinline__ int row_of(int g) { return BITS == 4 ? ((g & 1) << 2) | (g >> 1) : g; }
  __device__ __forceinline__ void load128(uint32_t row, int r, int step, int t) {
    if (BITS == 4) {
      v[0] = lds16(row + (((step * 4 + t) ^ r) << 4));
    } else {
      v[0] = lds16(row + (((2 * t) ^ r) << 4));
      v[1] = lds16(row + (((2 * t + 1) ^ r) << 4));
    }
  }
  // codes 8j .. 8j + 7
  template <bool F16>
  __device__ __forceinline__ void pairs(int j, uint32_t (&p)[4]) const {
    if (BITS == 4) {
      const uint32_t w = j == 0 ? v[0].x : j == 1 ? v[0].y : j == 2 ? v[0].z : v[0].w;
      if (F16) pairs4_f16(w, p);
      else pairs4_bf16(w, p);
    } else {
      const uint4 u = v[j >> 1];
      const uint32_t w0 = (j & 1) ? u.z : u.x, w1 = (j & 1) ? u.w : u.y;
      if (F16) {
        pairs8_f16(w0, p[0], p[1]);
        pairs8_f16(w1, p[2], p[3]);
      } else {
        pairs8_bf16(w0, p[0], p[1]);
        pairs8_bf16(w1, p[2], p[3]);
      }
    }
  }
};

// the element of 8 that stands at place i of the pairs, and the place of element n of h
template <int BITS>
__device__ __forceinline__ constexpr int pair_element(int i) {
  return BITS == 4 ? (i >> 1) + 4 * (i & 1) : (i & 4) + ((i >> 1) & 1) + 2 * (i & 1);
}
template <int BITS>
__device__ __forceinline__ int pair_place(int n) {
  const int j = n & 7;
  return BITS == 4 ? (j < 4 ? 2 * j : 2 * j - 7) : (j & 4) + 2 * (j & 1) + ((j >> 1) & 1);
}

// The scale of step s of a row: where a row has a multiple of 4 of them, a copy brings the aligned four that hold it
// (a slot never straddles them: they cover a multiple of 4 steps), else lanes load it (those of a quad share a row
// pair: even lanes its first row, odd lanes its second).
__device__ __forceinline__ int scale_index(int s, int gsteps) { return gsteps == 0 ? 0 : gsteps == 1 ? s : s / gsteps; }

__device__ __forceinline__ float load_scale(const float* a, const float* b, int s, int steps, int gsteps, int t) {
  return s < steps ? __ldg(((t & 1) ? b : a) + scale_index(s, gsteps)) : 0.f;
}

__device__ __forceinline__ void quad_scales(float v, float& a, float& b) {
  const int src = threadIdx.x & 28;
  a = __shfl_sync(0xffffffffu, v, src);
  b = __shfl_sync(0xffffffffu, v, src + 1);
}

// key > 0 that orders floats as their values; NaN lowest
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t b = __float_as_uint(z);
  if (!(z == z)) return 1;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int MAX_DEPTH1 = 2;
constexpr int TILE1 = 2048;      // 8 gate and 8 up rows of 128 bytes: one copy
constexpr int SLOT1 = 2 * TILE1;
constexpr int SCALE1 = 256;      // the same 16 rows' four scales
constexpr int RED_SLICES = 8;
constexpr int RED_PITCH = MAX_T + 1;
constexpr int RED_BYTES = RED_SLICES * 64 * RED_PITCH * 4;
constexpr int ROUTER_BYTES = RED_BYTES + CL1 * MAX_EXP * MAX_T * 4;  // over the rings and tokens, before they are used

struct Smem1 {
  float w[MAX_T][MAX_K];         // the routing, as the caller brings it or gets it
  int16_t ids[MAX_T][MAX_K];     // (experts out of range as -1)
  uint32_t mask[MAX_EXP];        // tokens of every expert
  Segment seg[MAX_SEG];
  float col_w[2][8];             // the columns' weights of the segments at hand
  float col_scale[2][64][8];     // what undoes the scaling of a step of a column's token
  float4 head[WARPS][32];        // a warp's part of a job that an earlier warp began
  uint64_t full[WARPS][MAX_DEPTH1];  // a slot of a warp's ring has landed
  int32_t nseg;
  int abort_flag;
};

using LogitPart = float[MAX_T][MAX_EXP];

// The router: K is split over the CTAs of the cluster and eight slices of warps in each; half of the warps take 32 of
// 64 experts at a time, the others the next 32.  A slice's sums meet in `red`, a CTA's in parts[rank] of both CTAs.
__device__ void router_logits(const FewArgs& a, float (*red)[64][RED_PITCH], LogitPart* parts, cg::cluster_group& cluster) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ntiles = (a.T + 7) / 8;
  const int rank = static_cast<int>(cluster.block_rank());
  const int slice = warp % RED_SLICES, half = warp / RED_SLICES;
  const int pairs = (a.H + 63) / 64;  // 128 bytes of a row: two chunks of 32
  const int p0 = pairs * rank / CL1, p1 = pairs * (rank + 1) / CL1;
  for (int eg = 0; eg < a.E; eg += 64) {
    float d[2][MAX_T / 8][4] = {};
    const __nv_bfloat16* w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // experts beyond the last read it and are not kept
      w[i] = a.gate + static_cast<int64_t>(min(eg + half * 32 + i * 8 + g, a.E - 1)) * a.H + 8 * t;
    for (int p = p0 + slice; p < p1; p += RED_SLICES) {
      uint4 u[2][4], x[2][MAX_T / 8];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int at = p * 64 + c * 32;
        const bool in = at < a.H;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          u[c][i] = in ? __ldg(reinterpret_cast<const uint4*>(w[i] + at)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < MAX_T / 8; ++n)
          x[c][n] = in && n < ntiles ? __ldg(reinterpret_cast<const uint4*>(
                                           a.x + static_cast<int64_t>(min(n * 8 + g, a.T - 1)) * a.H + 8 * t + at))
                                     : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int n = 0; n < MAX_T / 8; ++n)
          if (n < ntiles) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              mma_bf16(d[m][n], u[c][2 * m].x, u[c][2 * m + 1].x, u[c][2 * m].y, u[c][2 * m + 1].y, x[c][n].x, x[c][n].y);
              mma_bf16(d[m][n], u[c][2 * m].z, u[c][2 * m + 1].z, u[c][2 * m].w, u[c][2 * m + 1].w, x[c][n].z, x[c][n].w);
            }
          }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < MAX_T / 8; ++n)
        if (n < ntiles) {
          float* r = &red[slice][half * 32 + m * 16 + g][n * 8 + 2 * t];
          r[0] = d[m][n][0];
          r[1] = d[m][n][1];
          r[8 * RED_PITCH] = d[m][n][2];
          r[8 * RED_PITCH + 1] = d[m][n][3];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * a.T; i += THREADS) {
      const int r = i & 63, tok = i >> 6;
      if (eg + r < a.E) {
        float z = 0.f;
#pragma unroll
        for (int k = 0; k < RED_SLICES; ++k) z = __fadd_rn(z, red[k][r][tok]);
#pragma unroll
        for (int c = 0; c < CL1; ++c) *cluster.map_shared_rank(&parts[rank][tok][eg + r], c) = z;
      }
    }
    if (eg + 64 < a.E) __syncthreads();
  }
}

__device__ __forceinline__ float logit_of(const FewArgs& a, const LogitPart* parts, int e, int tok) {
  float z = __fadd_rn(parts[0][tok][e], parts[1][tok][e]);
  if (a.bias != nullptr) z = __fadd_rn(z, __ldg(a.bias + e));
  return z;
}

// softmax and top-k of N tokens (WARPS apart) by one warp, 32 PER experts at most, into sm.ids, sm.w and sm.mask; the
// tokens' chains of dependent steps overlap
template <int PER, int N>
__device__ void choose(const FewArgs& a, Smem1& sm, const LogitPart* parts, int tok0) {
  const int lane = threadIdx.x & 31;
  float p[N][PER], s[N], wt[N];
  uint32_t key[N][PER];  // 0: no expert, or one that is taken
  int id[N];             // lane i: choice i
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int tok = min(tok0 + n * WARPS, a.T - 1);
    float m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = lane + 32 * j;
      p[n][j] = e < a.E ? __fadd_rn(logit_of(a, parts, e, tok), 0.f) : -INFINITY;  // -0 ranks as +0
      key[n][j] = e < a.E ? order_key(p[n][j]) : 0;
      bad |= !(p[n][j] == p[n][j]);
      m = fmaxf(m, p[n][j]);
    }
    m = warp_max(m);
    s[n] = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      p[n][j] = lane + 32 * j < a.E ? expf(p[n][j] - m) : 0.f;
      s[n] = __fadd_rn(s[n], p[n][j]);
    }
    s[n] = warp_sum(s[n]);
    if (__any_sync(0xffffffffu, bad)) s[n] = NAN;  // as softmax over a row with a NaN
    wt[n] = 0.f;
    id[n] = 0;
  }
  for (int i = 0; i < a.k; ++i) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t best = key[n][0];
      float q = p[n][0];
      int bj = 0;
#pragma unroll
      for (int j = 1; j < PER; ++j) {
        if (key[n][j] > best) {
          best = key[n][j];
          q = p[n][j];
          bj = j;
        }
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      const uint32_t mine = best == top ? static_cast<uint32_t>(lane + 32 * bj) : 0xffffffffu;
      const uint32_t e = __reduce_min_sync(0xffffffffu, mine);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (mine == e && j == bj) key[n][j] = 0;
      q = __shfl_sync(0xffffffffu, q, e & 31);
      if (lane == i) {
        id[n] = static_cast<int>(e);
        wt[n] = q;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int tok = tok0 + n * WARPS;
    if (lane < a.k) wt[n] = __fdiv_rn(wt[n], s[n]);
    if (a.renormalize) {
      float total = 0.f;
      for (int i = 0; i < a.k; ++i) total = __fadd_rn(total, __shfl_sync(0xffffffffu, wt[n], i));
      wt[n] = __fdiv_rn(wt[n], total);
    }
    if (lane < a.k && tok < a.T) {
      sm.ids[tok][lane] = static_cast<int16_t>(id[n]);
      sm.w[tok][lane] = wt[n];
      atomicOr(&sm.mask[id[n]], 1u << tok);
    }
  }
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// TS: scales by copies
template <int BITS, bool TS>
__global__ void __launch_bounds__(THREADS, 1)
    few_gemm1_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_s, const FewArgs a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int SS = Codes<BITS>::STEPS;  // steps of a tile
  const int steps = (a.H + KG - 1) / KG, slots = (steps + 2 * SS - 1) / (2 * SS);
  // [rings of codes][rings of scales][tokens in MMA order, nbuf segments][Smem1]; the router's sums before all but the last
  const int ring_bytes = WARPS * a.depth1 * (SLOT1 + SCALE1);
  const int xf_pieces = slots * 2 * SS * 128;  // of a segment: 2 KB a step
  uint4* xf = reinterpret_cast<uint4*>(base + ring_bytes);
  Smem1& sm = *reinterpret_cast<Smem1*>(base + max(ring_bytes + a.nbuf * xf_pieces * 16, ROUTER_BYTES));
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int grid = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
  if (threadIdx.x < WARPS * MAX_DEPTH1) mbar_init(&sm.full[threadIdx.x / MAX_DEPTH1][threadIdx.x % MAX_DEPTH1], 1);
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    prefetch_map(&tm_w);
    if (TS) prefetch_map(&tm_s);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = threadIdx.x; i < a.E; i += THREADS) sm.mask[i] = 0;
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  pdl_wait();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // both CTAs run: their shared memory may be written to

  if (a.gate != nullptr) {
    LogitPart* parts = reinterpret_cast<LogitPart*>(base + RED_BYTES);
    router_logits(a, reinterpret_cast<float (*)[64][RED_PITCH]>(base), parts, cluster);
    cluster.sync();  // every CTA's sums are in every CTA
    if (a.E > 64) {
      for (int tok = warp; tok < a.T; tok += WARPS) choose<MAX_EXP / 32, 1>(a, sm, parts, tok);
    } else if (warp + WARPS < a.T) {
      choose<2, 2>(a, sm, parts, warp);
    } else if (warp < a.T) {
      choose<2, 1>(a, sm, parts, warp);
    }
    if (a.logits != nullptr && cta == grid - 1)
      for (int i = threadIdx.x; i < a.T * a.E; i += THREADS) a.logits[i] = logit_of(a, parts, i % a.E, i / a.E);
    __syncthreads();
    if (cta == 0) {
      for (int i = threadIdx.x; i < a.T * a.k; i += THREADS) {
        a.topk_w[i] = sm.w[i / a.k][i % a.k];
        a.topk_ids[i] = sm.ids[i / a.k][i % a.k];
      }
    }
  } else {
    __syncthreads();
    for (int i = threadIdx.x; i < a.T * a.k; i += THREADS) {
      const int e = a.topk_ids[i];
      const bool in = e >= 0 && e < a.E;
      sm.w[i / a.k][i % a.k] = a.topk_w[i];
      sm.ids[i / a.k][i % a.k] = static_cast<int16_t>(in ? e : -1);
      if (in) atomicOr(&sm.mask[e], 1u << (i / a.k));
    }
    __syncthreads();
  }
  if (warp == 0) {  // the segments: the chosen experts, ascending, 8 tokens at a time
    int n = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      uint32_t m = e0 + lane < a.E ? sm.mask[e0 + lane] : 0;
      const int mine = (__popc(m) + 7) >> 3;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      for (int i = n + incl - mine; m != 0; ++i) {
        Segment g1{e0 + lane, 0, 0};
        for (; m != 0 && g1.n < 8; m &= m - 1) g1.tokens |= static_cast<uint64_t>(__ffs(m) - 1) << (8 * g1.n++);
        sm.seg[i] = g1;
      }
      n += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) sm.nseg = n;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the router's sums lay where the copies land
  __syncthreads();
  pdl_trigger();

  // ---- GEMM1: this CTA's run [begin, end) of the jobs, with few segments inside one of them
  const int tiles = a.I / 8, nseg = sm.nseg;
  int begin, end;
  if (nseg > 0 && grid / nseg >= 8) {
    const int per = grid / nseg, s = cta / per, c = cta - s * per;  // CTAs of a segment
    begin = s < nseg ? s * tiles + tiles * c / per : 0;
    end = s < nseg ? s * tiles + tiles * (c + 1) / per : 0;
  } else {
    const int64_t jobs = static_cast<int64_t>(nseg) * tiles;
    begin = static_cast<int>(jobs * cta / grid);
    end = static_cast<int>(jobs * (cta + 1) / grid);
  }
  // The run goes in windows of nbuf segments; the slots of a window's jobs are split evenly over the warps, so that a
  // job may begin in one warp and end in another.
  const int kb = a.H * BITS / 8;  // bytes of a row of w1
  uint8_t* ring = base + warp * a.depth1 * SLOT1;
  uint8_t* sring = base + WARPS * a.depth1 * SLOT1 + warp * a.depth1 * SCALE1;
  volatile int* abort_flag = &sm.abort_flag;
  auto window_end = [&](int wb) { return min(end, (wb / tiles + a.nbuf) * tiles); };
  // the units (slots of jobs, in order) of window [wb, we) that warp w begins at
  auto unit = [&](int wb, int we, int w) { return static_cast<int>(static_cast<int64_t>(we - wb) * slots * w / WARPS); };

  // what is copied next: slot lz of row block lrow of expert half lhalf; lleft units are left in the window at lwb
  int lwb = begin, lleft = 0, lz = 0, lseg = 0, lrow = 0, lhalf = 0, lslot = 0;
  auto open = [&]() {  // the first window from lwb on in which this warp has units
    for (; lwb < end; lwb = window_end(lwb)) {
      const int we = window_end(lwb), u = unit(lwb, we, warp);
      lleft = unit(lwb, we, warp + 1) - u;
      if (lleft > 0) {
        const int job = lwb + u / slots;
        lz = u % slots;
        lseg = job / tiles;
        lrow = (job - lseg * tiles) * 8;
        lhalf = sm.seg[lseg].expert * 2;
        return;
      }
    }
  };
  // The whole warp follows the cursor and three lanes issue a copy each (two tiles, the scales): one lane doing it all
  // held the warp up for 950 cycles a slot.
  const CUtensorMap* lmap = lane == 2 ? &tm_s : &tm_w;
  auto fetch = [&]() {
    uint64_t* bar = &sm.full[warp][lslot];
    const bool two = lz * 256 + 128 < kb;
    if (lane == 0) mbar_expect_tx(bar, SLOT1 - (two ? 0 : TILE1) + (TS ? SCALE1 : 0));
    __syncwarp();
    uint8_t* dst = lane == 2 ? sring + lslot * SCALE1 : ring + lslot * SLOT1 + lane * TILE1;
    const int x = lane == 2 ? scale_index(lz * 2 * SS, a.gsteps1) & ~3 : lz * 256 + lane * 128;
    if (lane == 0 || (lane == 1 && two) || (lane == 2 && TS)) tma_load_3d(dst, lmap, x, lrow, lhalf, bar);
    if (++lslot == a.depth1) lslot = 0;
    if (--lleft == 0) {
      lwb = window_end(lwb);
      open();
    } else if (++lz == slots) {
      lz = 0;
      lrow += 8;
      if (lrow == a.I) {
        lrow = 0;
        lhalf = sm.seg[++lseg].expert * 2;
      }
    }
  };
  open();
  for (int i = 0; i < a.depth1 && lwb < end; ++i) fetch();
  if (cta == 0) {
    for (int i = threadIdx.x; i < nseg; i += THREADS) a.plan->seg[i] = sm.seg[i];
    if (threadIdx.x < MAX_PANELS) a.plan->done[threadIdx.x] = 0;
    if (threadIdx.x == 0) a.plan->n = nseg;
  }

  const int r = Codes<BITS>::row_of(g);
  const int hsteps = (a.I + KG - 1) / KG;
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int wb = begin; wb < end; wb = window_end(wb)) {
    const int we = window_end(wb), seg0 = wb / tiles, nsegs = (we - 1) / tiles - seg0 + 1;
    if (wb > begin) __syncthreads();  // the tokens of the window before are done with
    // the segments' tokens to fp16 in MMA order, eight 16-byte pieces in flight per thread
    const int row = xf_pieces / 8;  // pieces of a token with the zeros behind it, a multiple of 16
    const int n0 = sm.seg[seg0].n, cols = n0 + (nsegs > 1 ? sm.seg[seg0 + 1].n : 0);
    for (int i0 = 0; i0 < row * cols; i0 += 8 * THREADS) {
      uint4 v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int i = i0 + q * THREADS + static_cast<int>(threadIdx.x), cc = i / row, p = i - cc * row;
        const int b = cc >= n0;
        v[q] = make_uint4(0, 0, 0, 0);
        if (cc < cols && p * 8 < a.H)
          v[q] = __ldg(reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(sm.seg[seg0 + b].token(cc - b * n0)) * a.H) + p);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int i = i0 + q * THREADS + static_cast<int>(threadIdx.x), cc = i / row, p = i - cc * row;
        const int b = cc >= n0, c = cc - b * n0;
        const int s = p >> 4, pt = (p >> 2) & 3, pj = p & 3;  // step, lane of the quad, piece of the lane
        const uint32_t w[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
        float f[8];
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[2 * k] = __uint_as_float(w[k] << 16);
          f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
          m = max(m, max(w[k] & 0x7fff0000u, (w[k] << 16) & 0x7fffffffu));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));  // the step's 16 pieces
        const uint32_t e = min(max(m >> 23, 15u), 254u);  // largest magnitude in [2^(e-127), 2^(e-126))
        const float up = __uint_as_float((268u - e) << 23);
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __half2 pr = __floats2half2_rn(f[pair_element<BITS>(2 * k)] * up, f[pair_element<BITS>(2 * k + 1)] * up);
          h[k] = *reinterpret_cast<const uint32_t*>(&pr);
        }
        if (cc < cols) {
          xf[b * xf_pieces + (s * 4 + pj) * 32 + c * 4 + pt] = make_uint4(h[0], h[1], h[2], h[3]);
          if ((p & 15) == 0) sm.col_scale[b][s][c] = __uint_as_float((e - 14u) << 23);
        }
      }
    }
    if (threadIdx.x < cols) {
      const int b = static_cast<int>(threadIdx.x) >= n0, c = static_cast<int>(threadIdx.x) - b * n0;
      const Segment sg = sm.seg[seg0 + b];
      const int tok = sg.token(c);
      float w = 0.f;
      for (int i = 0; i < a.k; ++i)
        if (sm.ids[tok][i] == sg.expert) w = __fadd_rn(w, sm.w[tok][i]);
      sm.col_w[b][c] = w;
    }
    __syncthreads();

    // h of a finished job
    auto emit = [&](int job, const float (&acc)[4]) {
      const int seg = job / tiles, rb = job - seg * tiles, ntok = sm.seg[seg].n;
      const bool packed = ntok <= 4;
      // feature n = 8 rb + r of columns 2t and 2t + 1: its place in the 16 bytes of 8 features that rb is
      const int n = rb * 8 + r, s = n / KG, pt = (n % KG) / 32, pj = (n % 32) / 8;
      uint4* step = a.h + (static_cast<int64_t>(seg) * hsteps + s) * 256 + pj * 32 + pt;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = 2 * t + i;
        if (col < ntok) {
          const float ga = acc[i], up = acc[2 + i];
          const float h = __fdiv_rn(ga, 1.f + expf(-ga)) * up * sm.col_w[seg - seg0][col];
          const __nv_bfloat16 hi = __float2bfloat16_rn(h);
          __nv_bfloat16* at = reinterpret_cast<__nv_bfloat16*>(step + col * 4) + pair_place<BITS>(n);
          at[0] = hi;
          at[(packed ? 16 : 128) * 8] = __float2bfloat16_rn(h - __bfloat162float(hi));  // four columns, or a plane, further
        }
      }
      if (rb == tiles - 1) {  // zeros behind the last feature of the last step
        for (int p = tiles; p < hsteps * 16; ++p) {
          uint4* piece = a.h + (static_cast<int64_t>(seg) * hsteps + p / 16) * 256 + p % 4 * 32 + p % 16 / 4;
          if (lane < 2 * ntok) piece[(lane & 1) * (packed ? 16 : 128) + (lane >> 1) * 4] = make_uint4(0, 0, 0, 0);
        }
      }
    };
    int left = unit(wb, we, warp + 1) - unit(wb, we, warp);
    int job = wb + unit(wb, we, warp) / slots, za = unit(wb, we, warp) % slots;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    int open_job = -1;  // a job that this warp began and a later one ends
    while (left > 0 && ok) {
      const int zb = min(slots, za + left), seg = job / tiles, b = seg - seg0;
      left -= zb - za;
      const int64_t wrow = static_cast<int64_t>(sm.seg[seg].expert) * 2 * a.I + (job - seg * tiles) * 8 + r;
      const float* fg = a.s1 + wrow * a.groups1;
      const float* fu = fg + static_cast<int64_t>(a.I) * a.groups1;
      float sc = TS ? 0.f : load_scale(fg, fu, za * 2 * SS, steps, a.gsteps1, t);
      acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
      uint32_t xb = smem_u32(xf + b * xf_pieces + lane) + za * (2 * SS * 2048);
      uint32_t cb = smem_u32(&sm.col_scale[b][za * 2 * SS][2 * t]);
      for (int z = za; z < zb && ok; ++z) {
        ok = mbar_wait(&sm.full[warp][slot], phase, abort_flag, 0x600 + warp);
        const uint32_t tile = smem_u32(ring + slot * SLOT1) + r * 128, sa = smem_u32(sring + slot * SCALE1) + r * 16;
#pragma unroll
        for (int h = 0; h < 2 * SS; ++h) {  // behind the last step codes and tokens are zero
          float f, v;
          if (TS) {
            const uint32_t at = sa + (scale_index(z * 2 * SS + h, a.gsteps1) & 3) * 4;
            f = lds4(at);
            v = lds4(at + SCALE1 / 2);
          } else {
            quad_scales(sc, f, v);
            sc = load_scale(fg, fu, z * 2 * SS + h + 1, steps, a.gsteps1, t);
          }
          const float c0 = lds4(cb + h * 32), c1 = lds4(cb + h * 32 + 4);
          Codes<BITS> wg, wu;
          wg.load128(tile + h / SS * TILE1, r, h % SS, t);
          wu.load128(tile + h / SS * TILE1 + TILE1 / 2, r, h % SS, t);
          float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of MMAs
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 x = lds16(xb + h * 2048 + j * 512);
            uint32_t ag[4], au[4];
            wg.template pairs<true>(j, ag);
            wu.template pairs<true>(j, au);
            mma_f16(d0, ag[0], au[0], ag[1], au[1], x.x, x.y);
            mma_f16(d1, ag[2], au[2], ag[3], au[3], x.z, x.w);
          }
          acc[0] = __fmaf_rn(f * c0, __fadd_rn(d0[0], d1[0]), acc[0]);
          acc[1] = __fmaf_rn(f * c1, __fadd_rn(d0[1], d1[1]), acc[1]);
          acc[2] = __fmaf_rn(v * c0, __fadd_rn(d0[2], d1[2]), acc[2]);
          acc[3] = __fmaf_rn(v * c1, __fadd_rn(d0[3], d1[3]), acc[3]);
        }
        xb += 2 * SS * 2048;
        cb += 2 * SS * 32;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // our reads of the slot before its refill
        __syncwarp();
        if (lwb < end && ok) fetch();
        if (++slot == a.depth1) {
          slot = 0;
          phase ^= 1;
        }
      }
      if (za == 0 && zb == slots) {
        emit(job, acc);
      } else if (za > 0) {
        sm.head[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      } else {
        open_job = job;
      }
      ++job;
      za = 0;
    }
    __syncthreads();
    if (open_job >= 0) {  // its parts in the order of K
      const int stop = (open_job - wb + 1) * slots;
      for (int w = warp + 1; w < WARPS && unit(wb, we, w) < stop; ++w) {
        if (unit(wb, we, w) == unit(wb, we, w + 1)) continue;
        const float4 v = sm.head[w][lane];
        acc[0] = __fadd_rn(acc[0], v.x);
        acc[1] = __fadd_rn(acc[1], v.y);
        acc[2] = __fadd_rn(acc[2], v.z);
        acc[3] = __fadd_rn(acc[3], v.w);
      }
      emit(open_job, acc);
    }
  }
  // never leave copies in flight into this CTA's shared memory
  if (!ok && lane == 0) {
    const long long t0 = clock64();
    for (int i = 0; i < a.depth1; ++i) {
      const int q = (slot + i) % a.depth1;
      while (!mbar_try_wait(&sm.full[warp][q], q < slot ? phase ^ 1 : phase) && clock64() - t0 < kTimeoutCycles) {
      }
    }
  }
}

constexpr int MT = 8;                  // 16-row tiles of a panel, one warp of a group each
constexpr int PANEL = MT * 16;         // output features of a CTA of kernel 2
constexpr int GROUPS = WARPS / MT;     // groups of a CTA, each with a part of the steps
constexpr int MAX_DEPTH2 = 4;
constexpr int THREADS2 = THREADS + 32;  // and a warp that issues the copies

template <int BITS>
struct Stage2 {  // 128 bytes of the panel's packed rows (two steps at INT4, one at INT8), h, four scales of the rows
  static constexpr int STEPS = Codes<BITS>::STEPS;
  static constexpr int W = PANEL * 128;
  static constexpr int H = STEPS * 4096;
  static constexpr int S = PANEL * 16;
  static constexpr int BYTES = W + H + S;
};

struct Smem2 {
  Segment seg[MAX_SEG];
  uint64_t full[GROUPS][MAX_DEPTH2];
  uint64_t empty[GROUPS][MAX_DEPTH2];
  int abort_flag;
  int last;
};

template <int BITS, bool TS>
__global__ void __launch_bounds__(THREADS2, 1)
    few_gemm2_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_s, const FewArgs a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  using S = Stage2<BITS>;
  constexpr int SS = S::STEPS;
  const int depth = a.depth2;
  Smem2& sm = *reinterpret_cast<Smem2*>(base + GROUPS * depth * S::BYTES);
  float* parts = reinterpret_cast<float*>(base + GROUPS * depth * S::BYTES + sizeof(Smem2));  // [GROUPS][PANEL][pitch]
  const int pitch = a.T | 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int panel = blockIdx.x / a.split, rank = blockIdx.x % a.split, tile = warp % MT, group = warp / MT;
  if (threadIdx.x < GROUPS * MAX_DEPTH2) {
    mbar_init(&sm.full[threadIdx.x / MAX_DEPTH2][threadIdx.x % MAX_DEPTH2], 1);
    mbar_init(&sm.empty[threadIdx.x / MAX_DEPTH2][threadIdx.x % MAX_DEPTH2], MT);
  }
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    prefetch_map(&tm_w);
    if (TS) prefetch_map(&tm_s);
  }
  for (int i = threadIdx.x; i < GROUPS * PANEL * pitch; i += THREADS2) parts[i] = 0.f;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  asm volatile("fence.proxy.async.global;" ::: "memory");  // kernel 1's stores of h before the copies read them
  const int nseg = a.plan->n;
  if (threadIdx.x < MAX_SEG) sm.seg[threadIdx.x] = a.plan->seg[threadIdx.x];  // (those behind the last are not looked at)
  __syncthreads();

  // the slots (a stage each) of all segments in a row; a group has [begin, end) of them
  const int steps = (a.I + KG - 1) / KG, slots = (steps + SS - 1) / SS;
  const int64_t total = static_cast<int64_t>(nseg) * slots;
  auto bound = [&](int grp) { return static_cast<int>(total * (rank * GROUPS + grp) / (a.split * GROUPS)); };
  volatile int* abort_flag = &sm.abort_flag;

  if (warp == WARPS) {
    // ---- copies: the groups' next slots in turn
    int at[GROUPS], seg[GROUPS], z[GROUPS], st[GROUPS], issued[GROUPS];
    uint32_t ph[GROUPS];
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) {
      at[q] = bound(q);
      seg[q] = at[q] / slots;
      z[q] = at[q] - seg[q] * slots;
      st[q] = issued[q] = 0;
      ph[q] = 1;
    }
    bool ok = true;
    while (ok && (at[0] < bound(1) || at[GROUPS - 1] < bound(GROUPS))) {
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) {
        if (ok && at[q] < bound(q + 1)) {
          ok = mbar_wait(&sm.empty[q][st[q]], ph[q], abort_flag, 0x620 + q);
          if (!ok) break;
          const Segment sg = sm.seg[seg[q]];
          uint64_t* bar = &sm.full[q][st[q]];
          uint8_t* dst = base + (q * depth + st[q]) * S::BYTES;
          const int n = min(SS, steps - z[q] * SS);
          const int hb = sg.n <= 4 ? 2048 : 4096;  // of a step
          const int y = sg.expert * a.H + panel * PANEL;
          if (lane == 0) mbar_expect_tx(bar, S::W + n * hb + (TS ? S::S : 0));
          __syncwarp();
          if (lane == 0) {
            tma_load_2d(dst, &tm_w, z[q] * 128, y, bar);
            if (TS) tma_load_2d(dst + S::W + S::H, &tm_s, scale_index(z[q] * SS, a.gsteps2) & ~3, y, bar);
          } else if (lane <= n) {
            bulk_load(dst + S::W + (lane - 1) * 4096, a.h + (static_cast<int64_t>(seg[q]) * steps + z[q] * SS + lane - 1) * 256,
                      hb, bar);
          }
          ++at[q];
          ++issued[q];
          if (++z[q] == slots) {
            z[q] = 0;
            ++seg[q];
          }
          if (++st[q] == depth) {
            st[q] = 0;
            ph[q] ^= 1;
          }
        }
      }
    }
    if (!ok && lane == 0) {  // never leave copies in flight into this CTA's shared memory
      const long long t0 = clock64();
#pragma unroll
      for (int q = 0; q < GROUPS; ++q)
        for (int i = max(0, issued[q] - depth); i < issued[q]; ++i)
          while (!mbar_try_wait(&sm.full[q][i % depth], (i / depth) & 1) && clock64() - t0 < kTimeoutCycles) {
          }
    }
  } else {
    const int begin = bound(group), end = bound(group + 1);
    const int r = Codes<BITS>::row_of(g), r0 = tile * 16 + r;  // this lane's rows of the panel: r0 and r0 + 8
    const int n0 = min(panel * PANEL + r0, a.H - 1), n1 = min(panel * PANEL + r0 + 8, a.H - 1);
    bool ok = true;
    int st = 0;
    uint32_t phase = 0;
    for (int at = begin; at < end && ok;) {
      const int si = at / slots, za = at - si * slots, zb = min(slots, za + end - at);
      const Segment sg = sm.seg[si];
      const bool packed = sg.n <= 4;
      const float* f0 = a.s2 + (static_cast<int64_t>(sg.expert) * a.H + n0) * a.groups2;
      const float* f1 = a.s2 + (static_cast<int64_t>(sg.expert) * a.H + n1) * a.groups2;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      float sc = TS ? 0.f : load_scale(f0, f1, za * SS, steps, a.gsteps2, t);
      for (int z = za; z < zb; ++z, ++at) {
        ok = mbar_wait(&sm.full[group][st], phase, abort_flag, 0x610 + group);
        if (!ok) break;
        const uint32_t stage = smem_u32(base + (group * depth + st) * S::BYTES);
#pragma unroll
        for (int h = 0; h < SS; ++h) {
          const int s = z * SS + h;
          if (s < steps) {
            const uint32_t ha = stage + S::W + h * 4096 + lane * 16;
            Codes<BITS> w0, w1;
            w0.load128(stage + r0 * 128, r, h, t);
            w1.load128(stage + (r0 + 8) * 128, r, h, t);
            float f, v;
            if (TS) {
              const uint32_t fa = stage + S::W + S::H + r0 * 16 + (scale_index(s, a.gsteps2) & 3) * 4;
              f = lds4(fa);
              v = lds4(fa + 128);
            } else {
              quad_scales(sc, f, v);
              sc = load_scale(f0, f1, s + 1, steps, a.gsteps2, t);
            }
            float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};  // chains of MMAs
            if (packed) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint4 hv = lds16(ha + j * 512);
                uint32_t p0[4], p1[4];
                w0.template pairs<false>(j, p0);
                w1.template pairs<false>(j, p1);
                mma_bf16(d0, p0[0], p1[0], p0[1], p1[1], hv.x, hv.y);
                mma_bf16(d1, p0[2], p1[2], p0[3], p1[3], hv.z, hv.w);
              }
            } else {
              float d2[4] = {0.f, 0.f, 0.f, 0.f}, d3[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint4 hv = lds16(ha + j * 512), lv = lds16(ha + 2048 + j * 512);
                uint32_t p0[4], p1[4];
                w0.template pairs<false>(j, p0);
                w1.template pairs<false>(j, p1);
                mma_bf16(d0, p0[0], p1[0], p0[1], p1[1], hv.x, hv.y);
                mma_bf16(d1, p0[2], p1[2], p0[3], p1[3], hv.z, hv.w);
                mma_bf16(d2, p0[0], p1[0], p0[1], p1[1], lv.x, lv.y);
                mma_bf16(d3, p0[2], p1[2], p0[3], p1[3], lv.z, lv.w);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) d0[i] = __fadd_rn(d0[i], __fadd_rn(d2[i], d3[i]));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __fmaf_rn(i < 2 ? f : v, __fadd_rn(d0[i], d1[i]), acc[i]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // our reads of the stage before its refill
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[group][st]);
        if (++st == depth) {
          st = 0;
          phase ^= 1;
        }
      }
      if (packed) {  // columns 4 to 7 are the lo parts of 0 to 3
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = __fadd_rn(acc[i], __shfl_xor_sync(0xffffffffu, acc[i], 2));
      }
      // rows belong to this warp alone, and the tokens of a segment are distinct
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = 2 * t + i;
        if (col < sg.n) {
          float* p = parts + (group * PANEL + r0) * pitch + sg.token(col);
          p[0] += acc[i];
          p[8 * pitch] += acc[2 + i];
        }
      }
      __syncwarp();
    }
  }
  __syncthreads();
  // the groups' parts in the order of their steps; with one CTA a panel that is all
  float* mine = a.partial + (static_cast<int64_t>(panel) * a.split + rank) * (PANEL * a.T);
  auto store = [&](int i, float v) {  // i = token * PANEL + row
    const int n = panel * PANEL + i % PANEL;
    if (n < a.H) a.out[static_cast<int64_t>(i / PANEL) * a.H + n] = __float2bfloat16_rn(v);
  };
  for (int i = threadIdx.x; i < PANEL * a.T; i += THREADS2) {
    const float* p = parts + i % PANEL * pitch + i / PANEL;
    float v = p[0];
#pragma unroll
    for (int q = 1; q < GROUPS; ++q) v = __fadd_rn(v, p[q * PANEL * pitch]);
    if (a.split == 1) store(i, v);
    else __stcg(mine + i, v);
  }
  if (a.split == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) sm.last = atomicAdd(&a.plan->done[panel], 1) == a.split - 1;
  __syncthreads();
  if (!sm.last) return;
  __threadfence();
  // the CTA that finishes last adds the CTAs' parts, again in the order of their steps
  const float* all = a.partial + static_cast<int64_t>(panel) * a.split * (PANEL * a.T);
  for (int i = threadIdx.x; i < PANEL * a.T; i += THREADS2) {
    float v[MAX_SPLIT];
#pragma unroll
    for (int c = 0; c < MAX_SPLIT; ++c) v[c] = c < a.split ? __ldcg(all + static_cast<int64_t>(c) * (PANEL * a.T) + i) : 0.f;
#pragma unroll
    for (int c = 1; c < MAX_SPLIT; ++c) v[0] = __fadd_rn(v[0], v[c]);
    store(i, v[0]);
  }
}

template <typename K>
int launch_few_kernel(K kernel, int grid, int cluster, int threads, int smem, cudaStream_t st, const CUtensorMap& tw,
                      const CUtensorMap& ts, const FewArgs& a, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tw, ts, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(LLQ_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  return LLQ_OK;
}

constexpr int kSmemMost = 232448;  // 227 KB

inline int panels_of(int H) { return (H + PANEL - 1) / PANEL; }

// CTAs of a panel: as many as fill the SMs once
inline int split_of(int H) { return std::max(1, std::min(MAX_SPLIT, num_sms() / panels_of(H))); }

template <typename K>
int allow_smem(K kernel, std::atomic<uint64_t>& ready) {
  const cudaError_t e = once_per_device(
      ready, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost); });
  return e == cudaSuccess ? LLQ_OK : fail(LLQ_ECUDA, "few-token layer: %s", cudaGetErrorString(e));
}

template <int BITS, bool TS>
int launch_gemm1(FewArgs& a, const int8_t* q1, cudaStream_t st) {
  // w1 as [2 E halves][I rows][bytes]: a copy takes 8 gate rows and the same up rows
  const uint64_t kb = static_cast<uint64_t>(a.H) * BITS / 8, gb = static_cast<uint64_t>(a.groups1) * 4;
  CUtensorMap tw, ts;
  int rc = make_map_3d(&tw, q1, CU_TENSOR_MAP_DATA_TYPE_UINT8, kb, a.I, 2 * static_cast<uint64_t>(a.E), kb, kb * a.I, 128, 8,
                       2, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  ts = tw;
  if (TS) {
    rc = make_map_3d(&ts, a.s1, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.groups1, a.I, 2 * static_cast<uint64_t>(a.E), gb, gb * a.I,
                     4, 8, 2, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc) return rc;
  }
  static std::atomic<uint64_t> ready{0};
  rc = allow_smem(few_gemm1_kernel<BITS, TS>, ready);
  if (rc) return rc;
  // two segments' tokens and two slots of every ring where they fit (H up to 2048), then one segment's, then one slot
  constexpr int SS = Codes<BITS>::STEPS;
  const int seg = ((a.H + KG - 1) / KG + 2 * SS - 1) / (2 * SS) * (2 * SS) * 2048, slot = WARPS * (SLOT1 + SCALE1);
  int smem = 0;
  for (int i = 0; i < 3; ++i) {
    a.nbuf = i == 0 ? 2 : 1;
    a.depth1 = i == 2 ? 1 : 2;
    smem = 1024 + std::max(a.nbuf * seg + a.depth1 * slot, ROUTER_BYTES) + static_cast<int>(sizeof(Smem1));
    if (smem <= kSmemMost) break;
  }
  if (smem > kSmemMost) return fail(LLQ_EUNSUPPORTED, "the few-token layer has no room for rows of %d", a.H);
  return launch_few_kernel(few_gemm1_kernel<BITS, TS>, num_sms() / CL1 * CL1, CL1, THREADS, smem, st, tw, ts, a, "few_gemm1_kernel");
}

template <int BITS, bool TS>
int launch_gemm2(FewArgs& a, cudaStream_t st) {
  const uint64_t kb = static_cast<uint64_t>(a.I) * BITS / 8, rows = static_cast<uint64_t>(a.E) * a.H;
  CUtensorMap tw, ts;
  int rc = make_map(&tw, a.q2, CU_TENSOR_MAP_DATA_TYPE_UINT8, kb, rows, kb, 128, PANEL, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  ts = tw;
  if (TS) {
    rc = make_map(&ts, a.s2, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.groups2, rows, static_cast<uint64_t>(a.groups2) * 4, 4, PANEL,
                  CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc) return rc;
  }
  static std::atomic<uint64_t> ready{0};
  rc = allow_smem(few_gemm2_kernel<BITS, TS>, ready);
  if (rc) return rc;
  // as deep as the partial outputs leave room for
  const int fixed = 1024 + static_cast<int>(sizeof(Smem2)) + GROUPS * PANEL * (a.T | 1) * 4;
  a.depth2 = std::min(MAX_DEPTH2, (kSmemMost - fixed) / (GROUPS * Stage2<BITS>::BYTES));
  return launch_few_kernel(few_gemm2_kernel<BITS, TS>, panels_of(a.H) * a.split, 1, THREADS2,
                           fixed + GROUPS * a.depth2 * Stage2<BITS>::BYTES, st, tw, ts, a, "few_gemm2_kernel");
}

template <int BITS>
int launch_few(FewArgs& a, const int8_t* q1, cudaStream_t st) {
  auto aligned = [](const float* s, int groups) { return groups % 4 == 0 && (reinterpret_cast<uintptr_t>(s) & 15) == 0; };
  const int rc = aligned(a.s1, a.groups1) ? launch_gemm1<BITS, true>(a, q1, st) : launch_gemm1<BITS, false>(a, q1, st);
  if (rc) return rc;
  return aligned(a.s2, a.groups2) ? launch_gemm2<BITS, true>(a, st) : launch_gemm2<BITS, false>(a, st);
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

inline bool few_group_ok(int K, int group) { return group <= 0 || K % group != 0 || group % KG == 0; }

// most segments of a call: every chosen expert has one with fewer than 8 tokens at most, the others are full
inline int64_t few_segments(int64_t T, int k, int E) { return std::min<int64_t>(T * k, E + T * k / 8); }

struct FewWorkspace {
  size_t h, partial, total;
};

// (sized for the most CTAs a panel can have, so that it does not hang on the device)
FewWorkspace few_workspace(int64_t T, int k, int E, int H, int I) {
  FewWorkspace w;
  w.h = up256(sizeof(FewPlan));
  w.partial = w.h + static_cast<size_t>(few_segments(T, k, E)) * ((I + KG - 1) / KG) * 4096;
  w.total = w.partial + static_cast<size_t>(panels_of(H)) * MAX_SPLIT * PANEL * T * 4;
  return w;
}

}  // namespace

size_t moe_few_workspace(int64_t T, int k, int E, int H, int I) {
  if (T < 1 || k < 1 || E < 1 || H < 1 || I < 1 || T > MAX_T || k > MAX_K || E > MAX_EXP) return 0;
  return few_workspace(T, k, E, H, I).total;
}

int moe_few(const llq_few_layer& L, const void* x, int64_t T, float* logits, float* topk_w, int32_t* topk_ids,
            void* out, void* workspace, size_t bytes, cudaStream_t st) {
  if (T < 0 || L.E < 1 || L.H < 1 || L.I < 1 || L.k < 1 || L.k > L.E)
    return fail(LLQ_EINVAL, "bad shape T=%lld E=%d H=%d I=%d k=%d", (long long)T, L.E, L.H, L.I, L.k);
  if (L.bits != 4 && L.bits != 8) return fail(LLQ_EUNSUPPORTED, "bits must be 8 or 4, got %d", L.bits);
  if (T > MAX_T) return fail(LLQ_EUNSUPPORTED, "the few-token layer takes at most %d tokens, got %lld", MAX_T, (long long)T);
  if (L.E > MAX_EXP || L.k > MAX_K) return fail(LLQ_EUNSUPPORTED, "the few-token layer takes E <= 256 and k <= 32");
  if (L.H % 32 != 0 || L.I % 32 != 0 || L.H > 8192 || L.I > 8192)
    return fail(LLQ_EUNSUPPORTED, "the few-token layer needs H and I in multiples of 32, at most 8192 (H=%d I=%d)", L.H, L.I);
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
  const size_t need = moe_few_workspace(T, L.k, L.E, L.H, L.I);
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
  const FewWorkspace w = few_workspace(T, L.k, L.E, L.H, L.I);
  a.h = reinterpret_cast<uint4*>(ws + w.h);
  a.partial = reinterpret_cast<float*>(ws + w.partial);
  a.split = split_of(L.H);
  a.out = static_cast<__nv_bfloat16*>(out);
  return L.bits == 4 ? launch_few<4>(a, L.qw1, st) : launch_few<8>(a, L.qw1, st);
}

}  // namespace llq
