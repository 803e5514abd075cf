// Product of e4m3 rows with an e4m3 weight, one fp32 scale per 128 of a row and per 128 x 128 of the
// weight, on the tensor cores:
//
//   out[m, n] = sum over blocks g of xs[m, g] ws[n / 128, g] (sum_{k in g} x[m, k] w[n, k])  (+ bias[n])
//
// The scales are fp32, so no block sum may be added to another inside the tensor core: each 128-block of K
// is its own tcgen05.mma group (four kind::f8f6f4 MMAs of K = 32) into its own TMEM buffer, and the
// epilogue warps read it back, multiply by the block's scale and add in fp32 registers while the next
// block is being multiplied into another buffer.
//
// A tile is 128 rows (TMEM lanes, so a row's scale is one number per thread) by BN weight rows.
//   warp 0      TMA producer: per block the 128 x 128 and BN x 128 byte boxes (128-byte swizzle)
//   warp 1      TMEM allocator and MMA issuer (one elected lane)
//   warps 2, 3  bring the rows' scales to shared memory: as loads of the epilogue's threads, one line each, they held up
//               its waits and took as many cycles as its sums
//   warps 4-11  epilogue: one TMEM lane quarter each, half of the columns; BN / 2 sums per thread
// What bounds a large product is the chain of these hand-overs: of about 950 cycles that 128 x 256 x 128 takes, the tensor
// core works 510 and the epilogue's threads 600 (its reads of TMEM and its 128 sums are 256 each), and they overlap
// only as far as two accumulator buffers let them.  So a thread asks for its next 32 columns before it adds the last,
// which takes 216 registers at BN = 256.  8192 x 8192 x 2048: 140 us, 1.96 PFLOP/s, at the full clock (call after call the
// card's power limit holds it at 1.5 GHz and 165 us).  Other forms: fma.rn.f32x2 for the sums (three instructions a pair) 4 %
// slower, three column parts of 64 at BN = 192 8 %; a pair of CTAs on 256 x 256 (cta_group::2) 4 % faster there, 6 % slower at
// 1024 x 4096 x 4096, and not built in.
// Persistent over tiles when K is not split.  When the tiles do not cover the SMs, a cluster of `split`
// CTAs shares one tile, each takes a part of K, and the parts meet in distributed shared memory and are
// added in rank order.
//
// This file is compiled without relocatable device code (build.py), which setmaxnreg needs; so it has an error word of
// its own.
#define LLQ_OWN_ERROR_WORD
#include <cooperative_groups.h>

#include "fp8.cuh"
#include "tc_ptx.cuh"

namespace llq {

namespace {

namespace cg = cooperative_groups;

constexpr int BM = 128;
constexpr int BK = 128;

template <int BN>
struct F8Cfg {
  static constexpr int A_BYTES = BM * BK;
  static constexpr int STAGE_BYTES = A_BYTES + BN * BK;
  static constexpr int ACC_BUFS = BN == 256 ? 2 : 4;
  static constexpr int TMEM_COLS = ACC_BUFS * BN;
  static constexpr int EPI_WARPS = 8;
  static constexpr int COLS = BN / 2;  // columns of an epilogue thread
  static constexpr int FIRST_EPI = 4;
  static constexpr int THREADS = (FIRST_EPI + EPI_WARPS) * 32;
  static constexpr int OUT_BYTES = EPI_WARPS * 4096;  // per warp twice 32 rows of 64 bytes
  static constexpr int HEAD_BYTES = 3 * 1024;  // barriers (1 KB) and the rows' scales, one vector per accumulator buffer
  static constexpr int STAGES = (232448 - HEAD_BYTES - OUT_BYTES) / STAGE_BYTES;
  static constexpr size_t SMEM_BYTES = HEAD_BYTES + static_cast<size_t>(STAGES) * STAGE_BYTES + OUT_BYTES;
  static_assert(1024 + ACC_BUFS * BM * 4 <= HEAD_BYTES, "head");
  static_assert(128 * BN * 4 <= STAGES * STAGE_BYTES, "the parts of a split tile reuse the stages");
  static_assert(SMEM_BYTES <= 232448, "shared memory");
};

struct F8Args {
  const float* xs;   // [M][G]
  const float* ws;   // [ceil(N / 128)][G]
  const void* bias;  // [N] of the output's type, or null
  void* out;         // [M][N]
  int64_t M;
  int N, G;
  int mtiles, tiles;
  int split;
  int tma_out;       // rows of out are 16-byte aligned
  int box;           // rows of x that a copy brings
};

// instruction descriptor of kind::f8f6f4: D f32, A and B e4m3 (0), both K-major
__device__ __forceinline__ uint32_t f8_idesc(int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(BM >> 4) << 24);
}

__device__ __forceinline__ void tc_mma_f8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate,
                                          uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(issue)
      : "memory");
}

// 32 consecutive fp32 columns of this thread's TMEM lane; complete after tc_wait_ld()
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// the loads into v are complete (v is an operand, so that nothing that uses it moves up)
__device__ __forceinline__ void tc_wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
               :
               : "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
}

// a load that stays where it is written: the compiler would move it down to its first use, behind the wait it is to overlap
__device__ __forceinline__ float load_ahead(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

template <typename O>
__device__ __forceinline__ float bias_at(const void* b, int n) {
  return to_f32(static_cast<const O*>(b)[n]);
}

// 16 bytes of outputs from consecutive sums
__device__ __forceinline__ uint4 pack_out(const float* v, float) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}
template <typename O>
__device__ __forceinline__ uint4 pack_out(const float* v, O o) {
  return make_uint4(pack2(v[0], v[1], o), pack2(v[2], v[3], o), pack2(v[4], v[5], o), pack2(v[6], v[7], o));
}

// A wait that polls: each 128 of K runs through a chain of commit, epilogue, release and issue, and waking from a long
// suspension is part of it (256 x 8192 x 2048 9.9 us suspended, 9.0 polled; 8192 x 8192 x 2048 140 both).
__device__ __forceinline__ bool poll(uint64_t* b, uint32_t parity, volatile int* abort_flag, int code) {
  const long long t0 = clock64();
  for (int n = 1; !mbar_try_wait(b, parity); ++n) {
    if ((n & 255) == 0) {
      if (*abort_flag) return false;
      if (clock64() - t0 > kTimeoutCycles) {
        *abort_flag = 1;
        atomicExch(&g_device_error, code);
        return false;
      }
    }
  }
  return true;
}

template <int BN, typename O>
__global__ void __launch_bounds__(F8Cfg<BN>::THREADS, 1)
    fp8_tc_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_o, const F8Args a) {
  using C = F8Cfg<BN>;
  extern __shared__ __align__(1024) uint8_t smem_head[];  // 1024: what the 128-byte swizzle counts from
  float* row_scale = reinterpret_cast<float*>(smem_head + 1024);  // [ACC_BUFS][BM]
  uint8_t* smem = smem_head + C::HEAD_BYTES;
  uint8_t* so = smem + C::STAGES * C::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_head);
  uint64_t* empty = full + C::STAGES;
  uint64_t* acc_full = empty + C::STAGES;
  uint64_t* acc_empty = acc_full + C::ACC_BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + C::ACC_BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::ACC_BUFS; ++i) {
      mbar_init(&acc_full[i], 1 + 2);  // the MMAs' commit and the scale warps
      mbar_init(&acc_empty[i], C::EPI_WARPS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  // the codes may come from generic stores of the kernel before
  asm volatile("fence.proxy.async.global;" ::: "memory");

  const int rank = blockIdx.x % a.split;
  const int stride = gridDim.x / a.split;
  const int g0 = static_cast<int>(static_cast<int64_t>(a.G) * rank / a.split);
  const int g1 = static_cast<int>(static_cast<int64_t>(a.G) * (rank + 1) / a.split);

  // the epilogue's threads take over the others' registers: 128 x 64 + 256 x 216 of the block's 384 x 168
  if (warp < C::FIRST_EPI) {
    if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  }
  if (warp == 0) {
    if (lane == 0) {
      int issued = 0, rs = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = blockIdx.x / a.split; u < a.tiles && ok; u += stride) {
        const int m0 = u % a.mtiles * BM, n0 = u / a.mtiles * BN;
        for (int g = g0; g < g1; ++g) {
          if (!mbar_wait(&empty[rs], ph ^ 1, abort_flag, 0x500 + rs)) { ok = false; break; }
          mbar_expect_tx(&full[rs], a.box * BK + BN * BK);
          uint8_t* dst = smem + rs * C::STAGE_BYTES;
          tma_load_2d(dst, &tm_x, g * BK, m0, &full[rs]);
          tma_load_2d(dst + C::A_BYTES, &tm_w, g * BK, n0, &full[rs]);
          ++issued;
          if (++rs == C::STAGES) {
            rs = 0;
            ph ^= 1;
          }
        }
      }
      // never leave copies in flight into this CTA's shared memory
      for (int i = (issued > C::STAGES ? issued - C::STAGES : 0); i < issued; ++i) {
        const long long t0 = clock64();
        while (!mbar_try_wait(&full[i % C::STAGES], (i / C::STAGES) & 1) && clock64() - t0 < kTimeoutCycles) {
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_one();
    const uint32_t idesc = f8_idesc(BN);
    int rs = 0, ab = 0;
    uint32_t ph = 0, aph = 0;
    bool ok = true;
    for (int u = blockIdx.x / a.split; u < a.tiles && ok; u += stride) {
      for (int g = g0; g < g1; ++g) {
        if (!poll(&full[rs], ph, abort_flag, 0x520 + rs)) { ok = false; break; }
        if (!poll(&acc_empty[ab], aph ^ 1, abort_flag, 0x510 + ab)) { ok = false; break; }
        tc_fence_after();
        const uint64_t ad = make_sdesc(smem_u32(smem + rs * C::STAGE_BYTES));
        const uint64_t bd = make_sdesc(smem_u32(smem + rs * C::STAGE_BYTES + C::A_BYTES));
#pragma unroll
        for (int j = 0; j < 4; ++j)  // 32 bytes of K each: two 16-byte units of the descriptors
          tc_mma_f8(tmem + ab * BN, ad + 2 * j, bd + 2 * j, idesc, j > 0 ? 1u : 0u, leader);
        tc_commit(&empty[rs], leader);
        tc_commit(&acc_full[ab], leader);
        if (++rs == C::STAGES) {
          rs = 0;
          ph ^= 1;
        }
        if (++ab == C::ACC_BUFS) {
          ab = 0;
          aph ^= 1;
        }
      }
    }
  } else if (warp < C::FIRST_EPI) {
    // the scales of 64 rows, four blocks at a time, one block ahead of the accumulators
    const int r0 = (warp - 2) * 64 + lane;
    const bool vec = a.G % 4 == 0 && g0 % 4 == 0 && (reinterpret_cast<uintptr_t>(a.xs) & 15) == 0;
    int ab = 0;
    uint32_t aph = 0;
    bool ok = true;
    for (int u = blockIdx.x / a.split; u < a.tiles && ok; u += stride) {
      const int64_t m = static_cast<int64_t>(u % a.mtiles) * BM + r0;
      const float* p0 = a.xs + (m < a.M ? m : 0) * a.G;  // rows behind the last are not stored, whatever scales them
      const float* p1 = a.xs + (m + 32 < a.M ? m + 32 : 0) * a.G;
      auto fetch = [&](const float* p, int g) {
        if (vec && g < g1) return __ldg(reinterpret_cast<const float4*>(p + g));
        return make_float4(g < g1 ? __ldg(p + g) : 0.f, g + 1 < g1 ? __ldg(p + g + 1) : 0.f, g + 2 < g1 ? __ldg(p + g + 2) : 0.f,
                           g + 3 < g1 ? __ldg(p + g + 3) : 0.f);
      };
      float4 n0 = fetch(p0, g0), n1 = fetch(p1, g0);
      for (int g = g0; g < g1 && ok; g += 4) {
        const float v[2][4] = {{n0.x, n0.y, n0.z, n0.w}, {n1.x, n1.y, n1.z, n1.w}};
        n0 = fetch(p0, g + 4);
        n1 = fetch(p1, g + 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (g + k >= g1) break;
          if (!mbar_wait(&acc_empty[ab], aph ^ 1, abort_flag, 0x540 + ab)) { ok = false; break; }
          row_scale[ab * BM + r0] = v[0][k];
          row_scale[ab * BM + r0 + 32] = v[1][k];
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_full[ab]);
          if (++ab == C::ACC_BUFS) {
            ab = 0;
            aph ^= 1;
          }
        }
      }
    }
  } else {
    if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int part_of = (warp - C::FIRST_EPI) >> 2;  // this warp's columns
    const int q = warp & 3;  // the TMEM lanes a warp may read
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q * 32) << 16) + part_of * C::COLS;
    int ab = 0;
    uint32_t aph = 0;
    bool ok = true;
    for (int u = blockIdx.x / a.split; u < a.tiles && ok; u += stride) {
      const int m0 = u % a.mtiles * BM, n0 = u / a.mtiles * BN + part_of * C::COLS;
      const float* ws = a.ws + static_cast<int64_t>(min(n0, a.N - 1) / 128) * a.G;
      float acc[C::COLS];
#pragma unroll
      for (int i = 0; i < C::COLS; ++i) acc[i] = 0.f;
      float next = g0 < g1 ? load_ahead(ws + g0) : 0.f;
      for (int g = g0; g < g1; ++g) {
        const float sw = next;
        if (g + 1 < g1) next = load_ahead(ws + g + 1);
        if (!poll(&acc_full[ab], aph, abort_flag, 0x530 + ab)) { ok = false; break; }
        tc_fence_after();
        constexpr int CH = C::COLS / 32;
        const uint32_t at = lane_addr + ab * BN;
        uint32_t v[CH > 1 ? 2 : 1][32];
        tc_ld32(at, v[0]);
        const float s = __fmul_rn(row_scale[ab * BM + q * 32 + lane], sw);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          tc_wait_ld32(v[c & 1]);
          if (c + 1 < CH) {
            tc_ld32(at + (c + 1) * 32, v[(c + 1) & 1]);
          } else {  // all is read: the buffer goes back before the last sums
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[ab]);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c * 32 + i] = __fmaf_rn(__uint_as_float(v[c & 1][i]), s, acc[c * 32 + i]);
        }
        if (++ab == C::ACC_BUFS) {
          ab = 0;
          aph ^= 1;
        }
      }
      if (!ok) break;
      if (a.split > 1) {  // this CTA's part of the tile, column by column, over the drained stages
        float* part = reinterpret_cast<float*>(smem) + (part_of * C::COLS) * BM + q * 32 + lane;
#pragma unroll
        for (int i = 0; i < C::COLS; ++i) part[i * BM] = acc[i];
        break;
      }
      // 64 bytes of every row at a time through one of this warp's two pieces of shared memory
      constexpr int PER = 16 / sizeof(O);  // outputs of 16 bytes
      constexpr int CC = 64 / sizeof(O);   // columns of a round
#pragma unroll
      for (int c = 0; c < C::COLS / CC; ++c) {
        uint8_t* stage = so + (warp - C::FIRST_EPI) * 4096 + (c & 1) * 2048;  // an even number of rounds, or one
        if (a.tma_out) {
          if (lane == 0) {
            if (C::COLS / CC > 1) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          }
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < CC / PER; ++j) {
          float v[PER];
#pragma unroll
          for (int i = 0; i < PER; ++i) v[i] = acc[c * CC + j * PER + i];
          if (a.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
              v[i] = __fadd_rn(v[i], bias_at<O>(a.bias, min(n0 + c * CC + j * PER + i, a.N - 1)));
          }
          *reinterpret_cast<uint4*>(stage + lane * 64 + ((j ^ (lane >> 1 & 3)) * 16)) = pack_out(v, O());
        }
        if (a.tma_out) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (n0 + c * CC < a.N && m0 + q * 32 < a.M) tma_store_2d(&tm_o, stage, n0 + c * CC, m0 + q * 32);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // also an empty one: the waits count them
          }
        } else {
          __syncwarp();
          for (int r = 0; r < 32 && m0 + q * 32 + r < a.M; ++r) {
            O* dst = static_cast<O*>(a.out) + (static_cast<int64_t>(m0) + q * 32 + r) * a.N;
            for (int i = lane; i < CC; i += 32) {
              const int n = n0 + c * CC + i;
              if (n < a.N)
                dst[n] = *reinterpret_cast<const O*>(stage + r * 64 + (((i / PER) ^ (r >> 1 & 3)) * 16) + i % PER * sizeof(O));
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  if (a.split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    // BN / split columns each: a thread adds 8 of one row over the ranks, in rank order
    const int u = blockIdx.x / a.split;
    const int m0 = u % a.mtiles * BM, n0 = u / a.mtiles * BN;
    const int mine = BN / a.split, c0 = rank * mine;
    for (int i = threadIdx.x; i < BM * mine / 8; i += C::THREADS) {
      const int r = i % BM, c = c0 + i / BM * 8;
      float v[8] = {};
      for (int k = 0; k < a.split; ++k) {
        const float* part = cluster.map_shared_rank(reinterpret_cast<float*>(smem), k) + c * BM + r;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(v[j], part[j * BM]);
      }
      const int64_t m = static_cast<int64_t>(m0) + r;
      if (m < a.M) {
        O* dst = static_cast<O*>(a.out) + m * a.N + n0 + c;
        if (a.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(v[j], bias_at<O>(a.bias, min(n0 + c + j, a.N - 1)));
        }
        constexpr int PER = 16 / sizeof(O);
        if (a.tma_out && n0 + c + 8 <= a.N) {
#pragma unroll
          for (int j = 0; j < 8; j += PER) *reinterpret_cast<uint4*>(dst + j) = pack_out(v + j, O());
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n0 + c + j < a.N) dst[j] = from_f32<O>(v[j]);
        }
      }
    }
    cluster.sync();  // the others may still read this CTA's part
  }
  tc_fence_before();
  __syncthreads();
  pdl_trigger();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
  }
}

template <int BN, typename O>
int launch_tc(const Fp8Operands& p, const F8Args& in, CUtensorMapDataType ot, cudaStream_t st) {
  using C = F8Cfg<BN>;
  F8Args a = in;
  CUtensorMap tx, tw, to;
  int rc = make_map(&tx, p.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.K, p.M, p.ldx, BK, a.box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = make_map(&tw, p.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.K, p.N, p.ldw, BK, BN, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  to = tx;
  const bool aligned = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && (static_cast<size_t>(p.N) * sizeof(O)) % 16 == 0;
  a.tma_out = aligned;
  if (a.tma_out && a.split == 1) {
    rc = make_map(&to, p.out, ot, p.N, p.M, static_cast<uint64_t>(p.N) * sizeof(O), 64 / sizeof(O), 32,
                  CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc) return rc;
  }
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = once_per_device(ready, [] {
    return cudaFuncSetAttribute(fp8_tc_kernel<BN, O>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(C::SMEM_BYTES));
  });
  if (e != cudaSuccess) return fail(LLQ_ECUDA, "fp8_tc_kernel: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.split > 1 ? a.tiles * a.split : std::min(a.tiles, num_sms()));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, fp8_tc_kernel<BN, O>, tx, tw, to, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(LLQ_ECUDA, "fp8_tc_kernel: %s", cudaGetErrorString(e));
  }
  return LLQ_OK;
}

template <int BN>
int launch_out(const Fp8Operands& p, const F8Args& a, cudaStream_t st) {
  switch (p.out_type) {
    case LLQ_F32: return launch_tc<BN, float>(p, a, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, st);
    case LLQ_F16: return launch_tc<BN, __half>(p, a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, st);
    default: return launch_tc<BN, __nv_bfloat16>(p, a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, st);
  }
}

}  // namespace

cudaError_t fp8_tc_error(int32_t* code) { return cudaMemcpyFromSymbol(code, g_device_error, sizeof(int32_t)); }

cudaError_t fp8_tc_clear_error() {
  const int32_t zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int32_t));
}

int fp8_gemm_tc(const Fp8Operands& p, cudaStream_t st) {
  const int64_t mt = (p.M + BM - 1) / BM;
  const int sms = num_sms();
  auto tiles = [&](int bn) { return mt * ((p.N + bn - 1) / bn); };
  // Tile width and K split by an estimate in ns, fitted to sweeps with each forced: the start, then per 128 of K the chain of
  // hand-overs or the bytes that all CTAs together bring from L2 (13.6 TB/s), whichever is longer, and for a split the
  // cluster's start and the exchange of the parts.  Its clusters must fit at once (148 SMs hold 132 CTAs in clusters of
  // four, 120 in clusters of eight).  Measured (us): 64 wide 48 x 2048 x 2048 6.5 whole, 7.6 in two, 7.8 in four; 64 x 2048 x 4096
  // 10.2, 9.5, 8.2; 48 x 1024 x 8192 17.2, 13.0, 9.6; 256 x 8192 x 2048 256 wide 13.1, 128 wide 9.0, 64 wide 16; 1024 x 4096 x
  // 4096 19.6, 26.3, 46.
  int bn = 64, split = 1;
  int64_t best = INT64_MAX;
  for (int w : {256, 128, 64}) {
    const int64_t start = w == 64 ? 2800 : w == 128 ? 3400 : 4000, chain = w == 64 ? 235 : w == 128 ? 260 : 600;
    for (int sp = 1, exchange = 0; sp <= 8; sp *= 2, exchange = (exchange == 0 ? (w == 64 ? 2000 : 3000) : exchange) + 750) {
      const int room = sp == 8 ? sms * 120 / 148 : sp == 4 ? sms * 132 / 148 : sms;
      if (sp > 1 && (tiles(w) * sp > room || sp * 2 > p.G || w == 256)) break;
      const int64_t at_once = std::min<int64_t>(tiles(w) * sp, sms), waves = (tiles(w) * sp + sms - 1) / sms;
      const int64_t cost = start + exchange + waves * ((p.G + sp - 1) / sp) * std::max(chain, (BM + w) * BK * at_once / 13600);
      if (cost < best) {
        best = cost;
        bn = w;
        split = sp;
      }
    }
  }
  F8Args a{};
  a.xs = p.xs;
  a.ws = p.ws;
  a.bias = p.bias;
  a.out = p.out;
  a.M = p.M;
  a.N = p.N;
  a.G = p.G;
  if (tiles(bn) > 0x7fffffff) return fail(LLQ_EINVAL, "too many tiles");
  a.mtiles = static_cast<int>(mt);
  a.tiles = static_cast<int>(tiles(bn));
  a.split = split;
  // with fewer rows than a tile has, the copies bring these alone (the other lanes' sums are not stored): filling the rest
  // with zeros cost 15.0 us against 11.0 at 16 x 8192 x 4096, 12.2 against 10.3 at 24 x 4096 x 4096
  a.box = static_cast<int>(std::min<int64_t>(BM, (p.M + 7) / 8 * 8));
  return bn == 256 ? launch_out<256>(p, a, st) : bn == 128 ? launch_out<128>(p, a, st) : launch_out<64>(p, a, st);
}

}  // namespace llq
