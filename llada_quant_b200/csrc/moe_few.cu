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
// so nothing is transposed or repacked between memory and MMA.  The integer codes are exact in
// bf16; each group's partial sum is multiplied by the group's scale in fp32.
//
// Kernel 1 (router, GEMM1): each cluster of 2 CTAs computes the whole router (half per CTA, exchanged
// through distributed shared memory), so no grid-wide wait stands between router and experts.  The
// work is a list of segments (expert, up to 8 of its tokens), each of I / 8 jobs: 8 gate and the 8 up
// rows, so that SiLU(a) * b is local to a thread.  The CTAs take equal runs of jobs.
// Kernel 2 (GEMM2, combine): a cluster of 4 CTAs owns 64 output features and splits the list of
// (segment, 128-group) steps evenly over its 16 warp groups; the partial outputs meet in distributed
// shared memory and are added in the order of the steps: no atomics, a fixed order of sums.
// h travels between them as two bf16 numbers, hi + lo (16 significant bits), in the order in which
// kernel 2's lanes want it, so that the bf16 MMAs add no visible rounding: the layer rounds once, at
// its end.
//
// The packed bytes and their scales reach shared memory by TMA (swizzled) into rings that are deep
// enough for HBM's latency; the tokens lie in shared memory in MMA order.  Measured on the way
// (32 tokens, INT4, both kernels): lanes loading their own bytes with cp.async and their tokens from L1,
// 132 us, bound by the L1 wavefronts that eight scattered rows per instruction cost; a register ring
// unrolled over its slots, 527 us, its code larger than the instruction cache.
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
constexpr int CL2 = 4;        // of kernel 2: 132 fit
constexpr int WARPS = 16;
constexpr int THREADS = WARPS * 32;
constexpr int KG = 128;       // K elements of a step: 32 for each of a quad's four lanes

// what kernel 1 tells kernel 2 about the routing: the segments
struct FewPlan {
  int32_t n;
  int32_t expert[MAX_SEG];
  uint32_t mask[MAX_SEG];     // tokens, at most 8: the columns of the segment, ascending
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

// two int4 codes of a word (its nibbles 0 and 4) as a bf16 pair, 136 too large: the xor puts q + 8 into the low
// mantissa bits of 128
constexpr float kBias4 = 136.f;
__device__ __forceinline__ uint32_t int4_biased(uint32_t w) {
  uint32_t t;
  asm("lop3.b32 %0, %1, 0x000F000F, 0x43084308, 0x6A;" : "=r"(t) : "r"(w));
  return t;
}
// and exactly
__device__ __forceinline__ uint32_t int4_pair(uint32_t w) {
  uint32_t o;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(o) : "r"(int4_biased(w)), "r"(0xC308C308u));
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

// A lane's 32 codes of a row for one step, from rows of 128 bytes (128-byte swizzle) or 64 bytes (64-byte swizzle).
template <int BITS>
struct Codes {
  static constexpr int STEPS = BITS == 4 ? 2 : 1;  // steps in 128 bytes
  uint4 v[BITS == 4 ? 1 : 2];
  // Rows of 128 bytes; `row` is the address of row r (mod 8), `step` the step in it.  With row_of(g) as lane g's row
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
  // rows of one step, 64 bytes at INT4; lane g's row is g
  __device__ __forceinline__ void load_step(uint32_t row, int g, int t) {
    if (BITS == 4) v[0] = lds16(row + ((t ^ (g >> 1)) << 4));
    else load128(row, g, 0, t);
  }
  // codes 8j .. 8j + 7 as four bf16 pairs: INT4 (0,4) (1,5) (2,6) (3,7), INT8 (0,1) (2,3) (4,5) (6,7)
  // (BIASED: INT4 ones 136 too large)
  template <bool BIASED>
  __device__ __forceinline__ void pairs(int j, uint32_t (&p)[4]) const {
    if (BITS == 4) {
      const uint32_t w = j == 0 ? v[0].x : j == 1 ? v[0].y : j == 2 ? v[0].z : v[0].w;
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = BIASED ? int4_biased(w >> (4 * i)) : int4_pair(w >> (4 * i));
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

// the i-th set bit of m (i below the number of its bits, at most 8 here)
__device__ __forceinline__ int nth_bit(uint32_t m, int i) {
  for (; i > 0; --i) m &= m - 1;
  return __ffs(m) - 1;
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
constexpr int RED_BYTES = RED_SLICES * 64 * MAX_T * 4;
constexpr int ROUTER_BYTES = RED_BYTES + CL1 * MAX_EXP * MAX_T * 4;  // over the rings and tokens, before they are used

struct Smem1 {
  float w[MAX_T][MAX_K];         // the routing, as the caller brings it or gets it
  int16_t ids[MAX_T][MAX_K];     // (experts out of range as -1)
  uint32_t mask[MAX_EXP];        // tokens of every expert
  int32_t expert[MAX_SEG];       // the segments
  uint32_t seg_mask[MAX_SEG];
  float col_w[2][8];             // the columns' weights of the segments at hand
  float sum[2][64][8];           // and 136 times the sums of the steps of their tokens
  float4 head[WARPS][32];        // a warp's part of a job that an earlier warp began
  uint64_t full[WARPS][MAX_DEPTH1];  // a slot of a warp's ring has landed
  int32_t nseg;
  int abort_flag;
};

using LogitPart = float[MAX_EXP][MAX_T];

// The router: K is split over the CTAs of the cluster and eight slices of warps in each; half of the warps take 32 of
// 64 experts at a time, the others the next 32.  A slice's sums meet in `red`, a CTA's in parts[rank] of both CTAs.
__device__ void router_logits(const FewArgs& a, float (*red)[64][MAX_T], LogitPart* parts, cg::cluster_group& cluster) {
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
          r[8 * MAX_T] = d[m][n][2];
          r[8 * MAX_T + 1] = d[m][n][3];
        }
    __syncthreads();
    const int tw = ntiles * 8;
    for (int i = threadIdx.x; i < 64 * tw; i += THREADS) {
      const int r = i / tw, tok = i - r * tw;
      if (eg + r < a.E) {
        float z = 0.f;
#pragma unroll
        for (int k = 0; k < RED_SLICES; ++k) z = __fadd_rn(z, red[k][r][tok]);
#pragma unroll
        for (int c = 0; c < CL1; ++c) *cluster.map_shared_rank(&parts[rank][eg + r][tok], c) = z;
      }
    }
    if (eg + 64 < a.E) __syncthreads();
  }
}

__device__ __forceinline__ float logit_of(const FewArgs& a, const LogitPart* parts, int e, int tok) {
  float z = __fadd_rn(parts[0][e][tok], parts[1][e][tok]);
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

__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
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
    router_logits(a, reinterpret_cast<float (*)[64][MAX_T]>(base), parts, cluster);
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
        uint32_t rest = 0;
        if (__popc(m) > 8) {  // the lowest 8 tokens, then the others
          rest = m;
          for (int b = 0; b < 8; ++b) rest &= rest - 1;
        }
        sm.expert[i] = e0 + lane;
        sm.seg_mask[i] = m ^ rest;
        m = rest;
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
  // this warp's units of window [wb, we): [first, last)
  auto unit = [&](int wb, int we, int w) { return static_cast<int>(static_cast<int64_t>(we - wb) * slots * w / WARPS); };

  // what is copied next: slot lz of row block lrow of expert half lhalf; lleft units are left in the window at lwb
  int lwb = begin, lu = 0, lleft = 0, lz = 0, lrow = 0, lhalf = 0, lslot = 0;
  auto place = [&]() {
    const int job = lwb + lu / slots, seg = job / tiles;
    lz = lu % slots;
    lrow = (job - seg * tiles) * 8;
    lhalf = sm.expert[seg] * 2;
  };
  auto open = [&]() {  // the first window from lwb on in which this warp has units
    for (; lwb < end; lwb = window_end(lwb)) {
      const int we = window_end(lwb);
      lu = unit(lwb, we, warp);
      lleft = unit(lwb, we, warp + 1) - lu;
      if (lleft > 0) {
        place();
        return;
      }
    }
  };
  auto fetch = [&]() {  // (lane 0; lwb < end)
    uint64_t* bar = &sm.full[warp][lslot];
    uint8_t* dst = ring + lslot * SLOT1;
    const bool two = lz * 256 + 128 < kb;
    mbar_expect_tx(bar, SLOT1 - (two ? 0 : TILE1) + (TS ? SCALE1 : 0));
    tma_load_3d(dst, &tm_w, lz * 256, lrow, lhalf, bar);
    if (two) tma_load_3d(dst + TILE1, &tm_w, lz * 256 + 128, lrow, lhalf, bar);
    if (TS) tma_load_3d(sring + lslot * SCALE1, &tm_s, scale_index(lz * 2 * SS, a.gsteps1) & ~3, lrow, lhalf, bar);
    if (++lslot == a.depth1) lslot = 0;
    if (--lleft == 0) {
      lwb = window_end(lwb);
      open();
    } else {
      ++lu;
      if (++lz == slots) place();
    }
  };
  // once its own copies are on their way, every warp asks for its share of w2 and its scales: HBM stays busy until
  // kernel 2 runs, which then finds them in L2 (while they fit: half of it)
  bool asked = lane != 0 || static_cast<int64_t>(nseg) * a.H * a.I * BITS / 8 > (64 << 20);
  auto ask = [&]() {
    asked = true;
    const int64_t wbytes = static_cast<int64_t>(a.H) * a.I * BITS / 8, sbytes = static_cast<int64_t>(a.H) * a.groups2 * 4;
    constexpr int PIECE = 8192;
    const int wp = static_cast<int>((wbytes + PIECE - 1) / PIECE);
    const int sp = (reinterpret_cast<uintptr_t>(a.s2) & 15) ? 0 : static_cast<int>((sbytes + PIECE - 1) / PIECE);
    for (int64_t i = static_cast<int64_t>(cta) * WARPS + warp; i < static_cast<int64_t>(nseg) * (wp + sp); i += grid * WARPS) {
      const int s = static_cast<int>(i / (wp + sp)), p = static_cast<int>(i - static_cast<int64_t>(s) * (wp + sp));
      const int64_t e = sm.expert[s];
      if (s > 0 && sm.expert[s - 1] == e) continue;
      const int64_t off = static_cast<int64_t>(p < wp ? p : p - wp) * PIECE, all = p < wp ? wbytes : sbytes;
      const char* at = p < wp ? reinterpret_cast<const char*>(a.q2) + e * wbytes : reinterpret_cast<const char*>(a.s2) + e * sbytes;
      prefetch_l2(at + off, static_cast<uint32_t>(min(static_cast<int64_t>(PIECE), all - off)) & ~15u);
    }
  };
  if (lane == 0) {
    open();
    for (int i = 0; i < a.depth1 && lwb < end; ++i) fetch();
    if (lwb >= end && !asked) ask();
  }
  __syncwarp();
  if (cta == 0) {
    for (int i = threadIdx.x; i < nseg; i += THREADS) {
      a.plan->expert[i] = sm.expert[i];
      a.plan->mask[i] = sm.seg_mask[i];
    }
    if (threadIdx.x == 0) a.plan->n = nseg;
  }

  const int r = Codes<BITS>::row_of(g);
  const int hsteps = (a.I + KG - 1) / KG;
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int wb = begin; wb < end; wb = window_end(wb)) {
    const int we = window_end(wb), seg0 = wb / tiles, nsegs = (we - 1) / tiles - seg0 + 1;
    __syncthreads();  // the tokens of the window before are done with
    for (int b = 0; b < nsegs; ++b) {
      const int e = sm.expert[seg0 + b];
      const uint32_t mask = sm.seg_mask[seg0 + b];
      const int ntok = __popc(mask), row = xf_pieces / 8;  // 16-byte pieces of a token, a multiple of 16
      for (int i0 = warp * 32; i0 < row * ntok; i0 += THREADS) {
        const int i = i0 + lane;
        const int c = i / row, p = i - c * row;               // column, piece of its row
        const int s = p >> 4, pt = (p >> 2) & 3, pj = p & 3;  // step, lane of the quad, piece of the lane
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c < ntok && p * 8 < a.H)
          v = __ldg(reinterpret_cast<const uint4*>(a.x + static_cast<int64_t>(nth_bit(mask, c)) * a.H) + p);
        uint32_t q[4];
        token_pairs<BITS>(v, q);
        if (c < ntok) xf[b * xf_pieces + (s * 4 + pj) * 32 + c * 4 + pt] = make_uint4(q[0], q[1], q[2], q[3]);
        if (BITS == 4) {  // the token's sum over the step, for the bias of the codes
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            sum = __fadd_rn(sum, __fadd_rn(__uint_as_float(q[k] << 16), __uint_as_float(q[k] & 0xffff0000u)));
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
          if ((lane & 15) == 0 && c < ntok) sm.sum[b][s][c] = sum * kBias4;
        }
      }
      if (threadIdx.x < ntok) {
        const int tok = nth_bit(mask, threadIdx.x);
        float w = 0.f;
        for (int i = 0; i < a.k; ++i)
          if (sm.ids[tok][i] == e) w = __fadd_rn(w, sm.w[tok][i]);
        sm.col_w[b][threadIdx.x] = w;
      }
    }
    __syncthreads();

    // h of a finished job
    auto emit = [&](int job, const float (&acc)[4]) {
      const int seg = job / tiles, rb = job - seg * tiles, ntok = __popc(sm.seg_mask[seg]);
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
          __nv_bfloat16* at = reinterpret_cast<__nv_bfloat16*>(step + col * 4) + (pair_pos<BITS>(n) & 7);
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
    const int first = unit(wb, we, warp), last = unit(wb, we, warp + 1);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    int open_job = -1;  // a job that this warp began and a later one ends
    for (int u = first; u < last && ok;) {
      const int job = wb + u / slots, za = u % slots, zb = min(slots, za + last - u);
      const int seg = job / tiles, b = seg - seg0;
      const int64_t row = static_cast<int64_t>(sm.expert[seg]) * 2 * a.I + (job - seg * tiles) * 8 + r;
      const float* fg = a.s1 + row * a.groups1;
      const float* fu = fg + static_cast<int64_t>(a.I) * a.groups1;
      float sc = TS ? 0.f : load_scale(fg, fu, za * 2 * SS, steps, a.gsteps1, t);
      acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
      const uint32_t xb = smem_u32(xf + b * xf_pieces + lane), sb = smem_u32(&sm.sum[b][0][2 * t]);
      for (int z = za; z < zb && ok; ++z) {
        ok = mbar_wait(&sm.full[warp][slot], phase, abort_flag, 0x600 + warp);
        const uint32_t tile = smem_u32(ring + slot * SLOT1) + r * 128, sa = smem_u32(sring + slot * SCALE1) + r * 16;
#pragma unroll
        for (int h = 0; h < 2 * SS; ++h) {  // behind the last step codes and tokens are zero
          const int s = z * 2 * SS + h;
          float f, v;
          if (TS) {
            const uint32_t at = sa + (scale_index(s, a.gsteps1) & 3) * 4;
            f = lds4(at);
            v = lds4(at + SCALE1 / 2);
          } else {
            quad_scales(sc, f, v);
            sc = load_scale(fg, fu, s + 1, steps, a.gsteps1, t);
          }
          Codes<BITS> wg, wu;
          wg.load128(tile + h / SS * TILE1, r, h % SS, t);
          wu.load128(tile + h / SS * TILE1 + TILE1 / 2, r, h % SS, t);
          float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of MMAs
          if (BITS == 4) {
            d0[0] = d0[2] = -lds4(sb + s * 32);
            d0[1] = d0[3] = -lds4(sb + s * 32 + 4);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 x = lds16(xb + s * 2048 + j * 512);
            uint32_t ag[4], au[4];
            wg.template pairs<true>(j, ag);
            wu.template pairs<true>(j, au);
            mma_bf16(d0, ag[0], au[0], ag[1], au[1], x.x, x.y);
            mma_bf16(d1, ag[2], au[2], ag[3], au[3], x.z, x.w);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = __fmaf_rn(i < 2 ? f : v, __fadd_rn(d0[i], d1[i]), acc[i]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // our reads of the slot before its refill
        __syncwarp();
        if (lane == 0 && ok) {
          if (lwb < end) fetch();
          else if (!asked) ask();
        }
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
      u += zb - za;
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

constexpr int MT = 4;                  // 16-row tiles of a panel, one warp of a group each
constexpr int PANEL = MT * 16;         // output features of a cluster of kernel 2
constexpr int GROUPS = WARPS / MT;     // groups of a CTA, each with a part of the steps
constexpr int MAX_DEPTH2 = 6;

template <int BITS>
struct Stage2 {  // one step: the panel's packed rows, h, four scales of the rows
  static constexpr int W = PANEL * KG * BITS / 8;
  static constexpr int H = 4096;
  static constexpr int S = PANEL * 16;
  static constexpr int BYTES = W + H + S;
};

struct Smem2 {
  int32_t expert[MAX_SEG];
  uint32_t mask[MAX_SEG];
  uint64_t full[GROUPS][MAX_DEPTH2];
  uint64_t empty[GROUPS][MAX_DEPTH2];
  int abort_flag;
};

template <int BITS, bool TS>
__global__ void __launch_bounds__(THREADS, 1)
    few_gemm2_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_s, const FewArgs a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  using S = Stage2<BITS>;
  const int depth = a.depth2;
  Smem2& sm = *reinterpret_cast<Smem2*>(base + GROUPS * depth * S::BYTES);
  float* parts = reinterpret_cast<float*>(base + GROUPS * depth * S::BYTES + sizeof(Smem2));  // [GROUPS][PANEL][pitch]
  const int pitch = a.T | 1;
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(cluster.block_rank());
  const int panel = blockIdx.x / CL2, tile = warp % MT, group = warp / MT;
  if (threadIdx.x < GROUPS * MAX_DEPTH2) {
    mbar_init(&sm.full[threadIdx.x / MAX_DEPTH2][threadIdx.x % MAX_DEPTH2], 1);
    mbar_init(&sm.empty[threadIdx.x / MAX_DEPTH2][threadIdx.x % MAX_DEPTH2], MT);
  }
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    prefetch_map(&tm_w);
    if (TS) prefetch_map(&tm_s);
  }
  for (int i = threadIdx.x; i < GROUPS * PANEL * pitch; i += THREADS) parts[i] = 0.f;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  asm volatile("fence.proxy.async.global;" ::: "memory");  // kernel 1's stores of h before the copies read them
  const int nseg = a.plan->n;
  if (threadIdx.x < MAX_SEG) {  // what lies behind the last segment is not looked at
    sm.expert[threadIdx.x] = a.plan->expert[threadIdx.x];
    sm.mask[threadIdx.x] = a.plan->mask[threadIdx.x];
  }
  __syncthreads();

  // the steps of all segments in a row; this group has [begin, end) of them
  const int steps = (a.I + KG - 1) / KG;
  const int64_t total = static_cast<int64_t>(nseg) * steps;
  const int piece = rank * GROUPS + group;
  const int begin = static_cast<int>(total * piece / (CL2 * GROUPS)), end = static_cast<int>(total * (piece + 1) / (CL2 * GROUPS));
  uint8_t* ring = base + group * depth * S::BYTES;
  volatile int* abort_flag = &sm.abort_flag;
  int lat = begin, lseg = begin / steps, ls = begin - lseg * steps, lst = 0, lrow = 0, lh = 0;  // the step to be copied next
  auto place = [&]() {
    lrow = sm.expert[lseg] * a.H + panel * PANEL;
    lh = __popc(sm.mask[lseg]) <= 4 ? S::H / 2 : S::H;
  };
  if (begin < end) place();
  auto fetch = [&]() {  // (one lane of the group)
    uint64_t* bar = &sm.full[group][lst];
    uint8_t* dst = ring + lst * S::BYTES;
    mbar_expect_tx(bar, S::W + lh + (TS ? S::S : 0));
    tma_load_2d(dst, &tm_w, ls * (KG * BITS / 8), lrow, bar);
    bulk_load(dst + S::W, a.h + static_cast<int64_t>(lat) * 256, lh, bar);
    if (TS) tma_load_2d(dst + S::W + S::H, &tm_s, scale_index(ls, a.gsteps2) & ~3, lrow, bar);
    if (++lst == depth) lst = 0;
    ++lat;
    if (++ls == steps) {
      ls = 0;
      if (++lseg < nseg) place();
    }
  };
  if (tile == 0 && lane == 0)
    for (int i = 0; i < depth && lat < end; ++i) fetch();

  const int r0 = tile * 16 + g;  // this lane's rows of the panel: r0 and r0 + 8
  const int n0 = min(panel * PANEL + r0, a.H - 1), n1 = min(panel * PANEL + r0 + 8, a.H - 1);
  bool ok = true;
  int st = 0, prev = 0;  // the stage to be read, and the one read before
  uint32_t phase = 0, pphase = 0;
  for (int at = begin; at < end && ok;) {
    const int seg = at / steps, sa = at - seg * steps, sb = min(steps, sa + end - at);
    const int64_t e = sm.expert[seg];
    const uint32_t mask = sm.mask[seg];
    const int ntok = __popc(mask);
    const bool packed = ntok <= 4;
    const float* f0 = a.s2 + (e * a.H + n0) * a.groups2;
    const float* f1 = a.s2 + (e * a.H + n1) * a.groups2;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    float sc = TS ? 0.f : load_scale(f0, f1, sa, sb, a.gsteps2, t);
    for (int s = sa; s < sb; ++s, ++at) {
      const float scn = TS ? 0.f : load_scale(f0, f1, s + 1, sb, a.gsteps2, t);
      // the stage read before takes the next step once the group's four warps have read it
      if (tile == 0 && lane == 0 && at > begin && lat < end &&
          mbar_wait(&sm.empty[group][prev], pphase, abort_flag, 0x620 + group))
        fetch();
      __syncwarp();
      ok = mbar_wait(&sm.full[group][st], phase, abort_flag, 0x610 + group);
      if (!ok) break;
      const uint32_t w = smem_u32(ring + st * S::BYTES) + r0 * (KG * BITS / 8);
      const uint32_t ha = smem_u32(ring + st * S::BYTES + S::W) + lane * 16;
      Codes<BITS> w0, w1;
      w0.load_step(w, g, t);
      w1.load_step(w + 8 * (KG * BITS / 8), g, t);
      float f, v;
      if (TS) {
        const uint32_t fa = smem_u32(ring + st * S::BYTES + S::W + S::H) + r0 * 16 + (scale_index(s, a.gsteps2) & 3) * 4;
        f = lds4(fa);
        v = lds4(fa + 128);
      } else {
        quad_scales(sc, f, v);
        sc = scn;
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
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // our reads of the stage before its refill
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[group][st]);
      prev = st;
      pphase = phase;
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
      if (col < ntok) {
        float* p = parts + (group * PANEL + r0) * pitch + nth_bit(mask, col);
        p[0] += acc[i];
        p[8 * pitch] += acc[2 + i];
      }
    }
    __syncwarp();
  }
  if (!ok && tile == 0 && lane == 0) {  // never leave copies in flight into this CTA's shared memory
    const long long t0 = clock64();
    for (int i = 0; i < depth; ++i) {
      const int q = (st + i) % depth;
      while (!mbar_try_wait(&sm.full[group][q], q < st ? phase ^ 1 : phase) && clock64() - t0 < kTimeoutCycles) {
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < PANEL * pitch; i += THREADS) {  // the groups' parts in the order of their steps
    float v = parts[i];
#pragma unroll
    for (int q = 1; q < GROUPS; ++q) v = __fadd_rn(v, parts[q * PANEL * pitch + i]);
    parts[i] = v;
  }
  cluster.sync();
  // then the CTAs', a share of the panel's rows in each
  constexpr int ROWS = PANEL / CL2;
  for (int i = threadIdx.x; i < ROWS * a.T; i += THREADS) {
    const int row = rank * ROWS + i % ROWS, tok = i / ROWS;
    float v[CL2];
#pragma unroll
    for (int c = 0; c < CL2; ++c) v[c] = cluster.map_shared_rank(parts, c)[row * pitch + tok];
#pragma unroll
    for (int c = 1; c < CL2; ++c) v[0] = __fadd_rn(v[0], v[c]);
    if (panel * PANEL + row < a.H)
      a.out[static_cast<int64_t>(tok) * a.H + panel * PANEL + row] = __float2bfloat16_rn(v[0]);
  }
  cluster.sync();  // the others may still read this CTA's part
}

template <typename K>
int launch_cluster(K kernel, int grid, int cluster, int smem, cudaStream_t st, const CUtensorMap& tw, const CUtensorMap& ts,
                   const FewArgs& a, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tw, ts, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(LLQ_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  return LLQ_OK;
}

constexpr int kSmemMost = 232448;  // 227 KB

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
  return launch_cluster(few_gemm1_kernel<BITS, TS>, num_sms() / CL1 * CL1, CL1, smem, st, tw, ts, a, "few_gemm1_kernel");
}

template <int BITS, bool TS>
int launch_gemm2(FewArgs& a, cudaStream_t st) {
  const uint64_t kb = static_cast<uint64_t>(a.I) * BITS / 8, rows = static_cast<uint64_t>(a.E) * a.H;
  CUtensorMap tw, ts;
  int rc = make_map(&tw, a.q2, CU_TENSOR_MAP_DATA_TYPE_UINT8, kb, rows, kb, KG * BITS / 8, PANEL,
                    BITS == 4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
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
  return launch_cluster(few_gemm2_kernel<BITS, TS>, (a.H + PANEL - 1) / PANEL * CL2, CL2,
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

}  // namespace

size_t moe_few_workspace(int64_t T, int k, int E, int I) {
  if (T < 1 || k < 1 || E < 1 || I < 1 || T > MAX_T || k > MAX_K || E > MAX_EXP) return 0;
  return up256(sizeof(FewPlan)) + static_cast<size_t>(few_segments(T, k, E)) * ((I + KG - 1) / KG) * 4096;
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
  const size_t need = moe_few_workspace(T, L.k, L.E, L.I);
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
  a.h = reinterpret_cast<uint4*>(ws + up256(sizeof(FewPlan)));
  a.out = static_cast<__nv_bfloat16*>(out);
  return L.bits == 4 ? launch_few<4>(a, L.qw1, st) : launch_few<8>(a, L.qw1, st);
}

}  // namespace llq
