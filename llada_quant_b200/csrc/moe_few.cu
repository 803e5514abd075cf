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
// experts.  The work is a list of segments (expert, up to 8 of its tokens), each of I / 16 jobs: 16
// gate and the 16 up rows, so that SiLU(a) * b is local to a thread.  The CTAs take equal runs of jobs.
// Kernel 2 (GEMM2, combine): the CTAs of a panel of 128 output features split the list of (segment,
// 128-group) steps evenly; each stores its partial outputs, and the one that finishes last adds them
// in the order of the steps: no waits, and a fixed order of sums.
// The tokens enter kernel 1 as fp16, each 128-group scaled by a power of two so that its largest
// magnitude lies in [2^14, 2^15): exact for every bf16 value within 2^-31 of the largest, and what is
// lost below is 2^-40 of it.  (fp16 rather than bf16 because its ten mantissa bits take an INT8 code, or
// the upper nibble of a byte, where it lies: 40 instead of 56 logic instructions per lane and 128-group at
// INT4, 48 instead of 96 at INT8.)  h travels between the
// kernels as three bf16 numbers that add up to the fp32 value (8 + 8 + 8 significant bits; the third is short only
// where h lies below 2^-110).  So no MMA adds a visible rounding: the layer rounds once, at its end.
//
// The packed bytes reach shared memory by TMA (swizzled) into rings that are deep enough for HBM's latency;
// their scales go from global memory to registers, up to eight steps ahead (RowScales); the tokens lie in
// shared memory in MMA order.  Other forms (32 tokens, INT4, both kernels, where this takes 83 us): lanes loading their
// own bytes with cp.async and their tokens from L1, 132 us, bound by the L1 wavefronts that eight scattered
// rows per instruction cost; a register ring unrolled over its slots, 527 us, its code larger than the
// instruction cache; rings whose refill the computing warps issue themselves, 4 us more (a copy holds its
// warp up for hundreds of cycles).
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
constexpr int WARPS = 15;     // of kernel 1 that compute, and one that issues the copies
constexpr int THREADS = (WARPS + 1) * 32;
constexpr int KG = 128;       // K elements of a step: 32 for each of a quad's four lanes

constexpr int MAX_SPLIT = 16;  // CTAs of a panel in kernel 2
constexpr int MAX_PANELS = 64;

// an expert and up to 8 of its tokens, ascending: the columns of its MMAs
struct Segment {
  int32_t expert, n;
  uint64_t tokens;  // a byte each
  __device__ __forceinline__ int token(int c) const { return static_cast<int>(tokens >> (8 * c)) & 0xff; }
};

// Planes of 8 columns that the three parts of h of a segment of n tokens take: side by side in one with at most 2 tokens;
// with 3 or 4 the first two in one and the third in another, behind it zeros; with more each in one of its own.
__host__ __device__ __forceinline__ constexpr int planes_of(int n) { return n <= 2 ? 1 : n <= 4 ? 2 : 3; }
// 16-byte pieces from the first part of a column to its part i (to the zeros where i is 3: n 3 or 4 alone)
__device__ __forceinline__ int part_piece(int n, int i) { return n <= 2 ? 8 * i : n <= 4 ? (i >> 1) * 128 + (i & 1) * 16 : 128 * i; }

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
  // [segment][step of I][plane][piece j of 4][lane], 2 KB a plane: the B operand of kernel 2's MMAs.  Columns are the
  // segment's tokens, a plane for each of h's three parts; with fewer tokens the parts share planes (part_piece), and
  // bytes and MMAs fall away.
  uint4* h;
  int planes;            // of a step in h: as many as a segment of min(T, 8) tokens has
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
  // With row_of(g) as lane g's row the eight lanes that a shared-memory access serves at a time (two rows) meet eight
  // different 16-byte columns; offset(g, t) is where lane (g, t)'s first 16 bytes lie in its row.
  static __device__ __forceinline__ int row_of(int g) { return BITS == 4 ? ((g & 1) << 2) | (g >> 1) : g; }
  static __device__ __forceinline__ uint32_t offset(int g, int t) {
    return static_cast<uint32_t>(((BITS == 4 ? t : 2 * t) ^ row_of(g)) << 4);
  }
  // `at`: the lane's first 16 bytes in its row, at INT4 of the step (the second step's lie 64 bytes, xor, further)
  __device__ __forceinline__ void load(uint32_t at) {
    v[0] = lds16(at);
    if (BITS == 8) v[1] = lds16(at ^ 16);
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

// The scales of a warp's 32 rows.  Lane t of a quad loads those of one of the quad's four rows (t = 2 q + i: the row
// that is i of MMA q), and shuffles hand them to the quad.  V4: a row has a multiple of four scales, one per step: the
// lane holds those of four steps and asks for the next four in time for HBM.  Else one is loaded per step, or one for
// the whole row.
template <int STEPS, bool V4>
struct RowScales {
  const float* p;
  int gsteps, steps;
  float4 cur, nxt;
  __device__ __forceinline__ float4 four(int s) const {
    return s < steps ? __ldg(reinterpret_cast<const float4*>(p + s)) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ float one(int s) const { return s < steps ? __ldg(p + (gsteps == 1 ? s : s / gsteps)) : 0.f; }
  // for steps from s on
  __device__ __forceinline__ void start(const float* row, int s, int nsteps, int gs) {
    p = row;
    steps = nsteps;
    gsteps = gs;
    if (V4) {
      cur = four(s & ~3);
      nxt = four((s & ~3) + 4);
    } else {
      cur.x = gs == 0 ? __ldg(p) : one(s);
    }
  }
  // of step s, for all four rows
  __device__ __forceinline__ void get(int s, float (&f)[2][2]) {
    float v;
    if (V4) {
      v = (s & 2) ? ((s & 1) ? cur.w : cur.z) : ((s & 1) ? cur.y : cur.x);
    } else {
      v = cur.x;
      if (gsteps != 0) cur.x = one(s + 1);
    }
    const int src = threadIdx.x & 28;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < 2; ++i) f[q][i] = __shfl_sync(0xffffffffu, v, src + 2 * q + i);
  }
  // behind the slot whose first step was `first`
  __device__ __forceinline__ void next(int first) {
    if (V4 && ((first + STEPS) & 3) == 0) {
      cur = nxt;
      nxt = four(first + STEPS + 4);
    }
  }
};

// key > 0 that orders floats as their values; NaN lowest
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t b = __float_as_uint(z);
  if (!(z == z)) return 1;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int MAX_DEPTH1 = 2;
constexpr int SLOT1 = 4096;      // 16 gate and 16 up rows of 128 bytes (two steps at INT4, one at INT8): one copy
constexpr int RED_SLICES = (WARPS + 1) / 2;
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
  float4 head[WARPS][2][32];     // a warp's part of a job that an earlier warp began
  uint64_t full[WARPS][MAX_DEPTH1];   // a slot of a warp's ring has landed
  uint64_t empty[WARPS][MAX_DEPTH1];  // and was read
  int32_t nseg;
  int abort_flag;
};

using LogitPart = float[MAX_T][MAX_EXP];

// The router: K is split over the CTAs of the cluster and eight slices of warps in each; half of the warps take 32 of
// 64 experts at a time, the others the next 32.  A slice's sums meet in `red`, a CTA's in parts[rank] of both CTAs.
template <int NT>  // tiles of 8 tokens
__device__ void router_logits(const FewArgs& a, float (*red)[64][RED_PITCH], LogitPart* parts, cg::cluster_group& cluster) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(cluster.block_rank());
  const int slice = warp % RED_SLICES, half = warp / RED_SLICES;
  const int pairs = (a.H + 63) / 64;  // 128 bytes of a row: two chunks of 32
  const int p0 = pairs * rank / CL1, p1 = pairs * (rank + 1) / CL1;
#pragma unroll 1
  for (int eg = 0; eg < a.E; eg += 64) {
    {
      float d[2][NT][4] = {};
      const __nv_bfloat16* w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)  // experts beyond the last read it and are not kept
        w[i] = a.gate + static_cast<int64_t>(min(eg + half * 32 + i * 8 + g, a.E - 1)) * a.H + 8 * t;
      constexpr int CH = NT == 1 ? 4 : 2;  // chunks whose loads are under way together
#pragma unroll 1
      for (int p = p0 + slice; p < p1; p += RED_SLICES * CH / 2) {
        uint4 u[CH][4], x[CH][NT];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int q = p + c / 2 * RED_SLICES, at = q * 64 + c % 2 * 32;
          const bool in = q < p1 && at < a.H;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            u[c][i] = in ? __ldg(reinterpret_cast<const uint4*>(w[i] + at)) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            x[c][n] = in ? __ldg(reinterpret_cast<const uint4*>(
                                             a.x + static_cast<int64_t>(min(n * 8 + g, a.T - 1)) * a.H + 8 * t + at))
                                       : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              mma_bf16(d[m][n], u[c][2 * m].x, u[c][2 * m + 1].x, u[c][2 * m].y, u[c][2 * m + 1].y, x[c][n].x, x[c][n].y);
              mma_bf16(d[m][n], u[c][2 * m].z, u[c][2 * m + 1].z, u[c][2 * m].w, u[c][2 * m + 1].w, x[c][n].z, x[c][n].w);
            }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          {
            float* r = &red[slice][half * 32 + m * 16 + g][n * 8 + 2 * t];
            r[0] = d[m][n][0];
            r[1] = d[m][n][1];
            r[8 * RED_PITCH] = d[m][n][2];
            r[8 * RED_PITCH + 1] = d[m][n][3];
          }
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

__device__ __forceinline__ float raw_logit(const LogitPart* parts, int e, int tok) {
  return __fadd_rn(parts[0][tok][e], parts[1][tok][e]);
}
__device__ __forceinline__ float logit_of(const FewArgs& a, const LogitPart* parts, int e, int tok) {
  const float z = raw_logit(parts, e, tok);
  return a.bias != nullptr ? __fadd_rn(z, __ldg(a.bias + e)) : z;
}

// softmax and top-k of one token by one warp, 32 PER experts at most, into sm.ids, sm.w and sm.mask.  (Here and in all
// that a call runs once the code is kept short: it comes from L2 or HBM, 128 bytes at a time, and unrolling this for
// three tokens made it 3 times slower.)
template <int PER>
__device__ void choose(const FewArgs& a, Smem1& sm, const LogitPart* parts, int tok) {
  const int lane = threadIdx.x & 31;
  float p[PER];
  uint32_t key[PER];  // 0: no expert, or one that is taken
  float m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 32 * j;
    p[j] = e < a.E ? __fadd_rn(logit_of(a, parts, e, tok), 0.f) : -INFINITY;  // -0 ranks as +0
    key[j] = e < a.E ? order_key(p[j]) : 0;
    bad |= !(p[j] == p[j]);
    m = fmaxf(m, p[j]);
  }
  m = warp_max(m);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    p[j] = lane + 32 * j < a.E ? expf(p[j] - m) : 0.f;
    s = __fadd_rn(s, p[j]);
  }
  s = warp_sum(s);
  if (__any_sync(0xffffffffu, bad)) s = NAN;  // as softmax over a row with a NaN
  float wt = 0.f;
  int id = 0;  // lane i: choice i
#pragma unroll 1
  for (int i = 0; i < a.k; ++i) {
    uint32_t best = key[0];
    float q = p[0];
    int bj = 0;
#pragma unroll
    for (int j = 1; j < PER; ++j) {
      if (key[j] > best) {
        best = key[j];
        q = p[j];
        bj = j;
      }
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const uint32_t mine = best == top ? static_cast<uint32_t>(lane + 32 * bj) : 0xffffffffu;
    const uint32_t e = __reduce_min_sync(0xffffffffu, mine);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (mine == e && j == bj) key[j] = 0;
    q = __shfl_sync(0xffffffffu, q, e & 31);
    if (lane == i) {
      id = static_cast<int>(e);
      wt = q;
    }
  }
  if (lane < a.k) wt = __fdiv_rn(wt, s);
  if (a.renormalize) {
    float total = 0.f;
#pragma unroll 1
    for (int i = 0; i < a.k; ++i) total = __fadd_rn(total, __shfl_sync(0xffffffffu, wt, i));
    wt = __fdiv_rn(wt, total);
  }
  if (lane < a.k) {
    sm.ids[tok][lane] = static_cast<int16_t>(id);
    sm.w[tok][lane] = wt;
    atomicOr(&sm.mask[id], 1u << tok);
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

// h of a finished job: features 16 rb and on of segment seg.  (Inlined at both of its calls: called, with three parts, it
// makes the compiler copy the arguments to each thread's stack, 3 us more for one token.)
template <int BITS>
__device__ __forceinline__ void emit(const FewArgs& a, const Segment& sg, const float* col_w, int seg, int rb,
                                  const float (&acc)[2][4]) {
  const int lane = threadIdx.x & 31, t = lane & 3, r = Codes<BITS>::row_of(lane >> 2);
  const int hsteps = (a.I + KG - 1) / KG, ntok = sg.n, nparts = planes_of(ntok) == 2 ? 4 : 3;  // the fourth is zero
  const int o1 = part_piece(ntok, 1) * 8, o2 = part_piece(ntok, 2) * 8;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    // feature n of columns 2t and 2t + 1: its place in the 16 bytes of the 8 features from n - r on
    const int n = rb * 16 + q * 8 + r, s = n / KG, pt = (n % KG) / 32, pj = (n % 32) / 8;
    uint4* step = a.h + (static_cast<int64_t>(seg) * hsteps + s) * (a.planes * 128) + pj * 32 + pt;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = 2 * t + i;
      if (col < ntok) {
        const float ga = acc[q][i], up = acc[q][2 + i];
        float h = __fdiv_rn(ga, 1.f + expf(-ga)) * up * col_w[col];
        __nv_bfloat16* at = reinterpret_cast<__nv_bfloat16*>(step + col * 4) + pair_place<BITS>(n);
        const __nv_bfloat16 hi = __float2bfloat16_rn(h);
        h = __hisinf(hi) ? 0.f : h - __bfloat162float(hi);  // (infinity minus itself is a NaN)
        const __nv_bfloat16 mid = __float2bfloat16_rn(h);
        at[0] = hi;
        at[o1] = mid;
        at[o2] = __float2bfloat16_rn(h - __bfloat162float(mid));
        if (nparts == 4) at[part_piece(ntok, 3) * 8] = __float2bfloat16_rn(0.f);
      }
    }
  }
  if (rb == a.I / 16 - 1) {  // zeros behind the last feature of the last step
    for (int p = a.I / 8; p < hsteps * 16; ++p) {
      uint4* piece = a.h + (static_cast<int64_t>(seg) * hsteps + p / 16) * (a.planes * 128) + p % 4 * 32 + p % 16 / 4;
      const int part = lane >> 3, col = lane & 7;
      if (part < nparts && col < ntok) piece[part_piece(ntok, part) + col * 4] = make_uint4(0, 0, 0, 0);
    }
  }
}

// Router, top-k, segments and GEMM1.  32 tokens of a 64 x 2048 x 1024, top-8 INT4 layer: 17 us until the first product
// (router 8, top-k and segments 4, tokens 4), then 31 us for 135 MB (4.3 TB/s): over the whole kernel the warps issue in 47 %
// of the cycles (9 instructions turn 8 INT4 codes into fp16 pairs) and otherwise wait, for scales first, then for the
// chain of a step's MMAs; four warps a scheduler are too few to cover for one another.  One token: 9 us, then 7.
template <int BITS, bool V4>
__global__ void __launch_bounds__(THREADS, 1)
    few_gemm1_kernel(const __grid_constant__ CUtensorMap tm_w, const FewArgs a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int SS = Codes<BITS>::STEPS;  // steps of a slot
  const int steps = (a.H + KG - 1) / KG, slots = (steps + SS - 1) / SS;
  // [rings of codes][tokens in MMA order, nbuf segments][Smem1]; the router's sums before all but the last
  const int ring_bytes = WARPS * a.depth1 * SLOT1;
  const int xf_pieces = slots * SS * 128;  // of a segment: 2 KB a step
  uint4* xf = reinterpret_cast<uint4*>(base + ring_bytes);
  Smem1& sm = *reinterpret_cast<Smem1*>(base + max(ring_bytes + a.nbuf * xf_pieces * 16, ROUTER_BYTES));
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int grid = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
  if (threadIdx.x < WARPS * MAX_DEPTH1) {
    mbar_init(&sm.full[threadIdx.x / MAX_DEPTH1][threadIdx.x % MAX_DEPTH1], 1);
    mbar_init(&sm.empty[threadIdx.x / MAX_DEPTH1][threadIdx.x % MAX_DEPTH1], 1);
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    prefetch_map(&tm_w);
  }
  for (int i = threadIdx.x; i < a.E; i += THREADS) sm.mask[i] = 0;
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  pdl_wait();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // both CTAs run: their shared memory may be written to

  if (a.gate != nullptr) {
    LogitPart* parts = reinterpret_cast<LogitPart*>(base + RED_BYTES);
    float (*red)[64][RED_PITCH] = reinterpret_cast<float (*)[64][RED_PITCH]>(base);
    if (a.T <= 8) router_logits<1>(a, red, parts, cluster);
    else router_logits<4>(a, red, parts, cluster);
    cluster.sync();  // every CTA's sums are in every CTA
    if (warp < WARPS) {
#pragma unroll 1
      for (int tok = warp; tok < a.T; tok += WARPS) {
        if (a.E <= 64) choose<2>(a, sm, parts, tok);
        else choose<MAX_EXP / 32>(a, sm, parts, tok);
      }
    }
    if (a.logits != nullptr && cta == grid - 1)
      for (int i = threadIdx.x; i < a.T * a.E; i += THREADS) a.logits[i] = raw_logit(parts, i % a.E, i / a.E);
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
  const int tiles = a.I / 16, nseg = sm.nseg;
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
  volatile int* abort_flag = &sm.abort_flag;
  auto window_end = [&](int wb) { return min(end, (wb / tiles + a.nbuf) * tiles); };
  // the units (slots of jobs, in order) of window [wb, we) that warp w begins at
  auto unit = [&](int wb, int we, int w) { return static_cast<int>(static_cast<int64_t>(we - wb) * slots * w / WARPS); };

  // Copies: lane w of the last warp follows warp w's jobs, slot lz of row block lrow of expert half lhalf next, `left`
  // units left in the window at lwb.
  int lwb = begin, left = 0, lz = 0, lseg = 0, lrow = 0, lhalf = 0, lslot = 0, issued = 0;
  uint32_t lphase = 1;
  auto open = [&]() {  // the first window from lwb on in which the warp has units
    for (; lwb < end; lwb = window_end(lwb)) {
      const int we = window_end(lwb), u = unit(lwb, we, lane);
      left = unit(lwb, we, lane + 1) - u;
      if (left > 0) {
        const int job = lwb + u / slots;
        lz = u % slots;
        lseg = job / tiles;
        lrow = (job - lseg * tiles) * 16;
        lhalf = sm.seg[lseg].expert * 2;
        return;
      }
    }
  };
  auto copy = [&]() {
    uint64_t* bar = &sm.full[lane][lslot];
    mbar_expect_tx(bar, SLOT1);
    tma_load_3d(base + (lane * a.depth1 + lslot) * SLOT1, &tm_w, lz * 128, lrow, lhalf, bar);
    ++issued;
    if (++lslot == a.depth1) {
      lslot = 0;
      lphase ^= 1;
    }
    if (--left == 0) {
      lwb = window_end(lwb);
      open();
    } else if (++lz == slots) {
      lz = 0;
      lrow += 16;
      if (lrow == a.I) {
        lrow = 0;
        lhalf = sm.seg[++lseg].expert * 2;
      }
    }
  };
  if (warp == WARPS) {
    if (lane < WARPS) open();
    else lwb = end;
    for (int i = 0; i < a.depth1; ++i)
      if (lwb < end) copy();
  }
  if (cta == 0) {
    for (int i = threadIdx.x; i < nseg; i += THREADS) a.plan->seg[i] = sm.seg[i];
    if (threadIdx.x < MAX_PANELS) a.plan->done[threadIdx.x] = 0;
    if (threadIdx.x == 0) a.plan->n = nseg;
  }

  const int r = Codes<BITS>::row_of(g);
  const uint32_t ring = smem_u32(base + warp * a.depth1 * SLOT1) + r * 128 + Codes<BITS>::offset(g, t);
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int wb = begin; wb < end; wb = window_end(wb)) {
    const int we = window_end(wb), seg0 = wb / tiles, nsegs = (we - 1) / tiles - seg0 + 1;
    if (wb > begin) __syncthreads();  // the tokens of the window before are done with
    // the segments' tokens in MMA order: every thread copies its 16-byte pieces, then makes them fp16 where they lie
    const int row = xf_pieces / 8;  // pieces of a token with the zeros behind it, a multiple of 16
    const int n0 = sm.seg[seg0].n, cols = n0 + (nsegs > 1 ? sm.seg[seg0 + 1].n : 0);
    auto piece = [&](int i, int& b, int& c, int& p) {
      const int cc = i / row;
      p = i - cc * row;
      b = cc >= n0;
      c = cc - b * n0;
      // step p / 16, lane p / 4 % 4 of the quad, piece p % 4 of the lane
      return xf + b * xf_pieces + ((p >> 4) * 4 + (p & 3)) * 32 + c * 4 + ((p >> 2) & 3);
    };
#pragma unroll 1
    for (int i = threadIdx.x; i < row * cols; i += THREADS) {
      int b, c, p;
      const uint32_t dst = smem_u32(piece(i, b, c, p));
      const bool in = p * 8 < a.H;
      const uint4* src = reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(sm.seg[seg0 + b].token(c)) * a.H) + (in ? p : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
    for (int i0 = 0; i0 < row * cols; i0 += THREADS) {
      const int i = i0 + static_cast<int>(threadIdx.x);
      const bool in = i < row * cols;  // (16 threads in a row share a step)
      int b, c, p;
      uint4* at = piece(in ? i : 0, b, c, p);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (in) v = *at;
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
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
      if (in) {
        *at = make_uint4(h[0], h[1], h[2], h[3]);
        if ((p & 15) == 0) sm.col_scale[b][p >> 4][c] = __uint_as_float((e - 14u) << 23);
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

    if (warp == WARPS) {  // the copies of this window, as the warps give slots back
      long long t0 = clock64();
      bool more = lwb < we && ok;
      while (__any_sync(0xffffffffu, more)) {
        const bool can = more && mbar_test(&sm.empty[lane][lslot], lphase);
        if (can) {
          copy();
          more = lwb < we;
        }
        if (__any_sync(0xffffffffu, can)) {
          t0 = clock64();
        } else if (*abort_flag || clock64() - t0 > kTimeoutCycles) {
          if (lane == 0 && !*abort_flag) atomicExch(&g_device_error, 0x620);
          *abort_flag = 1;
          ok = false;
          break;
        } else {
          __nanosleep(40);
        }
      }
      __syncthreads();
      continue;
    }
    int units = unit(wb, we, warp + 1) - unit(wb, we, warp);
    int job = wb + unit(wb, we, warp) / slots, za = unit(wb, we, warp) % slots;
    float acc[2][4] = {};
    int open_job = -1;  // a job that this warp began and a later one ends
    while (units > 0 && ok) {
      const int zb = min(slots, za + units), seg = job / tiles, b = seg - seg0;
      units -= zb - za;
      // of the quad's rows lane t has the scales of gate (t even) or up row t / 2 * 8 + r of the job
      const int64_t wrow = static_cast<int64_t>(sm.seg[seg].expert) * 2 * a.I + (t & 1) * a.I + (job - seg * tiles) * 16 + (t >> 1) * 8 + r;
      RowScales<SS, V4> scales;
      scales.start(a.s1 + wrow * a.groups1, za * SS, steps, a.gsteps1);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = 0.f;
      uint32_t xb = smem_u32(xf + b * xf_pieces + lane) + za * (SS * 2048);
      uint32_t cb = smem_u32(&sm.col_scale[b][za * SS][2 * t]);
      for (int z = za; z < zb; ++z) {
        ok = mbar_wait(&sm.full[warp][slot], phase, abort_flag, 0x600 + warp);
        if (!ok) break;
        uint32_t rows = ring + slot * SLOT1;
#pragma unroll 1
        for (int h = 0; h < SS; ++h, rows ^= 64) {  // behind the last step codes and tokens are zero
          Codes<BITS> w[2][2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            w[q][0].load(rows + q * 1024);
            w[q][1].load(rows + SLOT1 / 2 + q * 1024);
          }
          float f[2][2], d0[2][4] = {}, d1[2][4] = {};  // two chains of MMAs for each of the two row tiles
          scales.get(z * SS + h, f);
          const float c0 = lds4(cb), c1 = lds4(cb + 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 x = lds16(xb + j * 512);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t ag[4], au[4];
              w[q][0].template pairs<true>(j, ag);
              w[q][1].template pairs<true>(j, au);
              mma_f16(d0[q], ag[0], au[0], ag[1], au[1], x.x, x.y);
              mma_f16(d1[q], ag[2], au[2], ag[3], au[3], x.z, x.w);
            }
          }
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[q][i] = __fmaf_rn(f[q][i >> 1] * ((i & 1) ? c1 : c0), __fadd_rn(d0[q][i], d1[q][i]), acc[q][i]);
          xb += 2048;
          cb += 32;
        }
        scales.next(z * SS);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // our reads of the slot before its refill
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[warp][slot]);
        if (++slot == a.depth1) {
          slot = 0;
          phase ^= 1;
        }
      }
      if (za == 0 && zb == slots) {
        emit<BITS>(a, sm.seg[seg], sm.col_w[b], seg, job - seg * tiles, acc);
      } else if (za > 0) {
#pragma unroll
        for (int q = 0; q < 2; ++q) sm.head[warp][q][lane] = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
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
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4 v = sm.head[w][q][lane];
          acc[q][0] = __fadd_rn(acc[q][0], v.x);
          acc[q][1] = __fadd_rn(acc[q][1], v.y);
          acc[q][2] = __fadd_rn(acc[q][2], v.z);
          acc[q][3] = __fadd_rn(acc[q][3], v.w);
        }
      }
      const int seg = open_job / tiles;
      emit<BITS>(a, sm.seg[seg], sm.col_w[seg - seg0], seg, open_job - seg * tiles, acc);
    }
  }
  // never leave copies in flight into this CTA's shared memory
  if (warp == WARPS && lane < WARPS && *abort_flag) {
    const long long t0 = clock64();
    for (int i = max(0, issued - a.depth1); i < issued; ++i)
      while (!mbar_try_wait(&sm.full[lane][i % a.depth1], (i / a.depth1) & 1) && clock64() - t0 < kTimeoutCycles) {
      }
  }
}

constexpr int MT = 4;                  // warps of a group, 32 rows each
constexpr int PANEL = MT * 32;         // output features of a CTA of kernel 2
constexpr int GROUPS = 3;              // groups of a CTA, each with a part of the steps
constexpr int WARPS2 = MT * GROUPS;
constexpr int THREADS2 = (WARPS2 + 1) * 32;  // and a warp that issues the copies
constexpr int MAX_DEPTH2 = 4;

template <int BITS>
struct Stage2 {  // 128 bytes of the panel's packed rows (two steps at INT4, one at INT8), and h
  static constexpr int STEPS = Codes<BITS>::STEPS;
  static constexpr int W = PANEL * 128;
  static __host__ __device__ constexpr int bytes(int planes) { return W + STEPS * planes * 2048; }
};

struct Smem2 {
  Segment seg[MAX_SEG];
  uint64_t full[GROUPS][MAX_DEPTH2];
  uint64_t empty[GROUPS][MAX_DEPTH2];
  int abort_flag;
  int last;
};

// GEMM2 and the combine.  The same layer: 22 us for 71 MB at 32 tokens (waits and issue, 47 %, again: up to three MMAs for h's three
// parts), then 5 for the outputs' parts; one token 3 and 4.  All of it: 32 tokens 83 us (INT8 105), one token 26 (INT8 30), 8 tokens INT8
// with given routing 66 (4.1 TB/s).  (With two parts of h, 16 bits of it, 81 (105), 26 (30) and 67.)
template <int BITS, bool V4>
__global__ void __launch_bounds__(THREADS2, 1)
    few_gemm2_kernel(const __grid_constant__ CUtensorMap tm_w, const FewArgs a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  using S = Stage2<BITS>;
  constexpr int SS = S::STEPS;
  const int depth = a.depth2, stage_bytes = S::bytes(a.planes), hstep = a.planes * 2048;
  Smem2& sm = *reinterpret_cast<Smem2*>(base + GROUPS * depth * stage_bytes);
  float* parts = reinterpret_cast<float*>(base + GROUPS * depth * stage_bytes + sizeof(Smem2));  // [GROUPS][PANEL][pitch]
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
  }
  for (int i = threadIdx.x; i < GROUPS * PANEL * pitch; i += THREADS2) parts[i] = 0.f;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  asm volatile("fence.proxy.async.global;" ::: "memory");  // kernel 1's stores of h before the copies read them
  const int nseg = a.plan->n;
  for (int i = threadIdx.x; i < MAX_SEG; i += THREADS2) sm.seg[i] = a.plan->seg[i];  // (those behind the last are not looked at)
  __syncthreads();

  // the slots (a stage each) of all segments in a row; a group has [begin, end) of them
  const int steps = (a.I + KG - 1) / KG, slots = (steps + SS - 1) / SS;
  const int64_t total = static_cast<int64_t>(nseg) * slots;
  auto bound = [&](int grp) { return static_cast<int>(total * (rank * GROUPS + grp) / (a.split * GROUPS)); };
  volatile int* abort_flag = &sm.abort_flag;

  if (warp == WARPS2) {
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
    for (bool more = true; more && ok;) {
      more = false;
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) {
        if (ok && at[q] < bound(q + 1)) {
          more = true;
          ok = mbar_wait(&sm.empty[q][st[q]], ph[q], abort_flag, 0x620 + q);
          if (!ok) break;
          const Segment sg = sm.seg[seg[q]];
          uint64_t* bar = &sm.full[q][st[q]];
          uint8_t* dst = base + (q * depth + st[q]) * stage_bytes;
          const int n = min(SS, steps - z[q] * SS);
          const int hb = planes_of(sg.n) * 2048;  // of a step
          const int y = sg.expert * a.H + panel * PANEL;
          if (lane == 0) mbar_expect_tx(bar, S::W + n * hb);
          __syncwarp();
          if (lane == 0) {
            tma_load_2d(dst, &tm_w, z[q] * 128, y, bar);
          } else if (lane <= n) {
            bulk_load(dst + S::W + (lane - 1) * hstep,
                      a.h + (static_cast<int64_t>(seg[q]) * steps + z[q] * SS + lane - 1) * (a.planes * 128), hb, bar);
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
    const int r0 = tile * 32 + Codes<BITS>::row_of(g);  // this lane's rows of the panel: r0, and 8, 16 and 24 further
    const int ns = min(panel * PANEL + r0 + 8 * t, a.H - 1);  // the one that it has the scales of
    const uint32_t lane_row = r0 * 128 + Codes<BITS>::offset(g, t);
    bool ok = true;
    int st = 0;
    uint32_t phase = 0;
    for (int at = begin; at < end && ok;) {
      const int si = at / slots, za = at - si * slots, zb = min(slots, za + end - at);
      const Segment sg = sm.seg[si];
      const int planes = planes_of(sg.n), lo = planes > 2 ? 4096 : 2048;
      RowScales<SS, V4> scales;
      scales.start(a.s2 + (static_cast<int64_t>(sg.expert) * a.H + ns) * a.groups2, za * SS, steps, a.gsteps2);
      float acc[2][4] = {};
      for (int z = za; z < zb; ++z, ++at) {
        ok = mbar_wait(&sm.full[group][st], phase, abort_flag, 0x610 + group);
        if (!ok) break;
        const uint32_t stage = smem_u32(base + (group * depth + st) * stage_bytes);
        uint32_t rows = stage + lane_row, ha = stage + S::W + lane * 16;
#pragma unroll 1
        for (int h = 0; h < SS; ++h, rows ^= 64, ha += hstep) {
          if (z * SS + h < steps) {
            Codes<BITS> w[2][2];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int i = 0; i < 2; ++i) w[q][i].load(rows + (2 * q + i) * 1024);
            float f[2][2], d0[2][4] = {}, d1[2][4] = {};  // chains of MMAs
            scales.get(z * SS + h, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 hv = lds16(ha + j * 512);
              uint4 mv, lv;  // asked for together, ahead of the MMAs (32 tokens 83.4 us; each before its own 86.0)
              if (planes > 1) {
                mv = lds16(ha + 2048 + j * 512);
                lv = lds16(ha + lo + j * 512);
              }
              uint32_t p[2][2][4];
#pragma unroll
              for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int i = 0; i < 2; ++i) w[q][i].template pairs<false>(j, p[q][i]);
                mma_bf16(d0[q], p[q][0][0], p[q][1][0], p[q][0][1], p[q][1][1], hv.x, hv.y);
                mma_bf16(d1[q], p[q][0][2], p[q][1][2], p[q][0][3], p[q][1][3], hv.z, hv.w);
              }
              if (planes > 1) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  mma_bf16(d0[q], p[q][0][0], p[q][1][0], p[q][0][1], p[q][1][1], mv.x, mv.y);
                  mma_bf16(d1[q], p[q][0][2], p[q][1][2], p[q][0][3], p[q][1][3], mv.z, mv.w);
                }
              }
              if (planes > 2) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  mma_bf16(d0[q], p[q][0][0], p[q][1][0], p[q][0][1], p[q][1][1], lv.x, lv.y);
                  mma_bf16(d1[q], p[q][0][2], p[q][1][2], p[q][0][3], p[q][1][3], lv.z, lv.w);
                }
              }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[q][i] = __fmaf_rn(f[q][i >> 1], __fadd_rn(d0[q][i], d1[q][i]), acc[q][i]);
          }
        }
        scales.next(z * SS);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // our reads of the stage before its refill
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[group][st]);
        if (++st == depth) {
          st = 0;
          phase ^= 1;
        }
      }
      if (planes < 3) {  // the other parts of a quad's lane 0 (and 1): in lanes 1 and 2 with at most 2 tokens, else in 2 (and 3)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = acc[q][i], far = __shfl_sync(0xffffffffu, v, lane + 2), near = __shfl_sync(0xffffffffu, v, lane + 1);
            acc[q][i] = __fadd_rn(v, planes == 1 ? __fadd_rn(near, far) : far);
          }
      }
      // rows belong to this warp alone, and the tokens of a segment are distinct
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = 2 * t + i;
        if (col < sg.n) {
          float* p = parts + (group * PANEL + r0) * pitch + sg.token(col);
#pragma unroll
          for (int q = 0; q < 4; ++q) p[8 * q * pitch] += acc[q >> 1][2 * (q & 1) + i];
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
  __syncthreads();
  if (threadIdx.x == 0) {  // (its fences hold for what the CTA's threads stored before and load behind the barriers)
    __threadfence();
    sm.last = atomicAdd(&a.plan->done[panel], 1) == a.split - 1;
    __threadfence();
  }
  __syncthreads();
  if (!sm.last) return;
  // the CTA that finishes last adds the CTAs' parts, again in the order of their steps
  const float4* all = reinterpret_cast<const float4*>(a.partial + static_cast<int64_t>(panel) * a.split * (PANEL * a.T));
  const int vecs = PANEL * a.T / 4;
  for (int i = threadIdx.x; i < vecs; i += THREADS2) {
    float4 v[MAX_SPLIT];
#pragma unroll
    for (int c = 0; c < MAX_SPLIT; ++c) v[c] = c < a.split ? __ldcg(all + c * vecs + i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 1; c < MAX_SPLIT; ++c) {
      v[0].x = __fadd_rn(v[0].x, v[c].x);
      v[0].y = __fadd_rn(v[0].y, v[c].y);
      v[0].z = __fadd_rn(v[0].z, v[c].z);
      v[0].w = __fadd_rn(v[0].w, v[c].w);
    }
    store(4 * i, v[0].x);
    store(4 * i + 1, v[0].y);
    store(4 * i + 2, v[0].z);
    store(4 * i + 3, v[0].w);
  }
}

template <typename K>
int launch_few_kernel(K kernel, int grid, int cluster, int threads, int smem, cudaStream_t st, const CUtensorMap& tw,
                      const FewArgs& a, const char* what) {
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tw, a);
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

template <int BITS, bool V4>
int launch_gemm1(FewArgs& a, const int8_t* q1, cudaStream_t st) {
  // w1 as [2 E halves][I rows][bytes]: a copy takes 16 gate rows and the same up rows
  const uint64_t kb = static_cast<uint64_t>(a.H) * BITS / 8;
  CUtensorMap tw;
  int rc = make_map_3d(&tw, q1, CU_TENSOR_MAP_DATA_TYPE_UINT8, kb, a.I, 2 * static_cast<uint64_t>(a.E), kb, kb * a.I, 128, 16,
                       2, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  static std::atomic<uint64_t> ready{0};
  rc = allow_smem(few_gemm1_kernel<BITS, V4>, ready);
  if (rc) return rc;
  // two segments' tokens and two slots of every ring where they fit, then one segment's, then one slot
  constexpr int SS = Codes<BITS>::STEPS;
  const int seg = ((a.H + KG - 1) / KG + SS - 1) / SS * SS * 2048, slot = WARPS * SLOT1;
  int smem = 0;
  for (int i = 0; i < 3; ++i) {
    a.nbuf = i == 0 ? 2 : 1;
    a.depth1 = i == 2 ? 1 : 2;
    smem = 1024 + std::max(a.nbuf * seg + a.depth1 * slot, ROUTER_BYTES) + static_cast<int>(sizeof(Smem1));
    if (smem <= kSmemMost) break;
  }
  if (smem > kSmemMost) return fail(LLQ_EUNSUPPORTED, "the few-token layer has no room for rows of %d", a.H);
  return launch_few_kernel(few_gemm1_kernel<BITS, V4>, num_sms() / CL1 * CL1, CL1, THREADS, smem, st, tw, a, "few_gemm1_kernel");
}

template <int BITS, bool V4>
int launch_gemm2(FewArgs& a, cudaStream_t st) {
  const uint64_t kb = static_cast<uint64_t>(a.I) * BITS / 8;
  CUtensorMap tw;
  int rc = make_map(&tw, a.q2, CU_TENSOR_MAP_DATA_TYPE_UINT8, kb, static_cast<uint64_t>(a.E) * a.H, kb, 128, PANEL,
                    CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  static std::atomic<uint64_t> ready{0};
  rc = allow_smem(few_gemm2_kernel<BITS, V4>, ready);
  if (rc) return rc;
  // as deep as the partial outputs leave room for
  const int fixed = 1024 + static_cast<int>(sizeof(Smem2)) + GROUPS * PANEL * (a.T | 1) * 4;
  const int stage = GROUPS * Stage2<BITS>::bytes(a.planes);
  a.depth2 = std::min(MAX_DEPTH2, (kSmemMost - fixed) / stage);
  return launch_few_kernel(few_gemm2_kernel<BITS, V4>, panels_of(a.H) * a.split, 1, THREADS2,
                           fixed + a.depth2 * stage, st, tw, a, "few_gemm2_kernel");
}

template <int BITS>
int launch_few(FewArgs& a, const int8_t* q1, cudaStream_t st) {
  auto v4 = [](const float* s, int groups, int gsteps) {
    return gsteps == 1 && groups % 4 == 0 && (reinterpret_cast<uintptr_t>(s) & 15) == 0;
  };
  const int rc = v4(a.s1, a.groups1, a.gsteps1) ? launch_gemm1<BITS, true>(a, q1, st) : launch_gemm1<BITS, false>(a, q1, st);
  if (rc) return rc;
  return v4(a.s2, a.groups2, a.gsteps2) ? launch_gemm2<BITS, true>(a, st) : launch_gemm2<BITS, false>(a, st);
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
  w.partial = w.h + static_cast<size_t>(few_segments(T, k, E)) * ((I + KG - 1) / KG) * planes_of(static_cast<int>(T)) * 2048;
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
  a.planes = planes_of(a.T);
  a.partial = reinterpret_cast<float*>(ws + w.partial);
  a.split = split_of(L.H);
  a.out = static_cast<__nv_bfloat16*>(out);
  return L.bits == 4 ? launch_few<4>(a, L.qw1, st) : launch_few<8>(a, L.qw1, st);
}

}  // namespace llq
