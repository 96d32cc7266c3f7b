// harp_gemm_s8: C[M, N] = (A B^T) * sa[m] * sb[n] + bias[n] with A [M, K] and
// B [N, K] in signed 8-bit integers, a scale for each row of A (token) and of B
// (output channel), 32-bit integer sums and a bf16 or fp32 result.
//
// The integer sum is exact (K <= 131071 keeps 128 * 128 * K below 2^31), so the
// result is one rounding of the sum to fp32, two products and an addition, and
// does not depend on the order of the K loop, its split or the kernel chosen.
//
// Two kernels:
//   gemm_s8_pair  CTA pairs (cta_group::2), persistent over 256 x BN tiles: many
//                 tokens and many channels.  17408 x 9216 x 1152 in 137 us alone
//                 (2.7 PFLOP/s) and 161 us run for seconds, where the GPU sits at its
//                 1000 W and 1.31 GHz (zeros for operands: 117 us at 1.97 GHz);
//                 17408 x 1152 x 4608 in 68 to 73 us alone and 80 us run for seconds
//   gemm_s8_rows  128 channels x up to 256 tokens a CTA, the K loop split over a
//                 cluster that adds its integer sums through distributed shared
//                 memory: few tokens (down to one) or few channels.  Bound by
//                 latency: 4 x 6912 x 1152 in 4.4 us and 4 x 1152 x 4608 in 4.7 us back to
//                 back, of which the weights' bytes are 1.2 and 0.8 us
// Operands whose rows TMA cannot address are first copied to rows that it can
// (1061 x 1003 x 1155 in 17 us, 12 without the copies).
#include "common.cuh"
#include "dependent_launch.cuh"
#include "gemm_common.cuh"
#include "gemm_sm100.h"
#include "per_device.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

namespace harp {

namespace {

using bf16 = __nv_bfloat16;

constexpr int64_t kMostRows = 0x7FFFFF00;  // of either operand
constexpr int64_t kMostK = 131071;

struct S8Args {
  int M, N, K;
  const int8_t* A;
  long lda;
  const int8_t* B;
  long ldb;
  const float* sa;
  const float* sb;
  const void* bias;
  int bias_f32;
  void* C;
  long ldc;
  int c_vec4;  // four neighbouring values of any row of C can be stored at once
  int* err;
};

__device__ __forceinline__ float bias_at(const S8Args& a, int n) {
  if (a.bias == nullptr) return 0.f;
  return a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[n]
                    : __bfloat162float(reinterpret_cast<const bf16*>(a.bias)[n]);
}

// ---------------------------------------------------------------------------
// tcgen05 kind::i8: signed 8-bit operands, 32-bit integer accumulators.  One MMA
// covers K = 32 (32 bytes), so the K-major shared-memory layout and its
// descriptors are those of the bf16 kernels byte for byte.
// ---------------------------------------------------------------------------
// Instruction descriptor: [4,6) D format (2 = s32), [7,10) A format and [10,13) B
// format (1 = signed 8-bit), [17,23) N>>3, [24,29) M>>4; both operands K-major.
__host__ __device__ constexpr uint32_t make_idesc_s8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_s8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  HARP_CHECK_TMEM(d_tmem, (int)(((idesc >> 17) & 0x3Fu) << 3), 215);
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_s8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  HARP_CHECK_TMEM(d_tmem, (int)(((idesc >> 17) & 0x3Fu) << 3), 216);
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrive on the barrier at this offset in both CTAs of the pair once the MMAs issued so far are done
__device__ __forceinline__ void mma_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---------------------------------------------------------------------------
// CTA-pair kernel.  The same pipeline as the bf16 pair kernel (gemm_sm100.cu):
// each CTA stages its own 128 rows of A and BN/2 rows of B, the leader issues
// M = 256 MMAs, two accumulators let the epilogue of one tile run under the MMAs
// of the next.  A stage is 256 deep in K (two 128-byte swizzle atoms a row), the
// same bytes as the bf16 kernel's 128, at twice the arithmetic.  (Stages of 128 and
// a commit for four MMAs instead of eight: 17408 x 1152 x 4608 in 101 us, not 83.)
//
// What bounds it: a 256 x 256 tile of K = 1152 is 36 steps of 128 clocks, 4608 in all.
// The 2448 tiles of 17408 x 9216 x 1152 are 34 rounds of the 74 pairs that are resident
// (the last of 6 tiles).  A round takes 5160 clocks of the SMs and 0.81 us that do not
// shrink with their clock: fitted, within 1 %, to runs of a second and more at 1312 MHz
// (161.3 us, 991 W), 1417 MHz (operands of -1 .. 1: 152.4 us) and 1965 MHz (zeros:
// 116.9 us).  So in a long run power sets the clock, and at full clock a quarter of a
// round is time outside the SMs, whose operands arrive at 12.4 TB/s from L2.  In the same
// way 17408 x 1152 x 4608 takes 100400 clocks, 82900 of them MMAs of the busiest pair
// (four whole tiles and a narrow one), and 7.6 us.  Fewer operand bytes would help
// against both: a row band's A kept in shared memory over its column tiles, where K lets it
// fit, and half the B for a narrow band, which is loaded whole.
//
// Epilogue: each warp scales its 32 rows 128 bytes at a time, lays them out in
// shared memory and one lane stores the block with TMA (whole 128-byte lines;
// out of range rows and 16-byte groups are dropped by the map).  A C that TMA cannot
// address, or whose rows end inside a group, is written from the same buffer, a row of
// the block at a time.  Stored
// straight from registers, 32 bytes a lane, 17408 x 9216 x 1152 took 187 us, not 154;
// eight epilogue warps instead of four changed nothing (190 and 187 at that time).
// ---------------------------------------------------------------------------
constexpr int kThreads = 192;
constexpr int kStageK = 256;

template <int BN>
struct PairCfg {
  static constexpr int A_ATOM = 128 * 128;       // 128 rows x one 128-byte atom
  static constexpr int B_ATOM = (BN / 2) * 128;
  static constexpr int A_BYTES = A_ATOM * (kStageK / 128);
  static constexpr int B_BYTES = B_ATOM * (kStageK / 128);
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGING = 4 * 2 * 4096;   // 4 epilogue warps x 2 buffers x (32 rows x 128 bytes)
  static constexpr int VECS = 2 * BN * 4;        // the tile's channel scales and bias
  static constexpr int STAGES = (232448 - 256 - STAGING - VECS) / STAGE_BYTES;
  static constexpr int TMEM_COLS = (2 * BN <= 256) ? 256 : 512;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + STAGING + VECS + 256;
  static_assert(STAGES >= 3 && STAGES <= 8 && SMEM_BYTES <= 232448, "pair GEMM stages");
};

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// A wait of the whole warp with one answer (lanes that ran out of time a moment apart must not part ways).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int site) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, err, site)) != 0;
}
// Arrive on another CTA's barrier without ordering earlier stores: what the
// barrier hands over is tensor memory, which the tcgen05 fences order.  (With
// release.cluster the arrive waits for the stores of the epilogue: 1700 clocks a
// tile, and the accumulator is free that much later.)
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}
__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Order of the pair kernel's tiles: the whole ones first, those of a last column
// band narrower than the tile at the end, where they even out the last wave.
__device__ __forceinline__ void pair_tile(int t, int num_m, int num_n, bool narrow, int& mt, int& nt) {
  const int whole = narrow ? num_n - 1 : num_n;
  if (t < num_m * whole) {
    tile_coords(t, num_m, whole, mt, nt);
  } else {
    mt = t - num_m * whole;
    nt = whole;
  }
}

template <int BN, typename OUT>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_s8_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmC, const S8Args args, int c_tma) {
  using C_ = PairCfg<BN>;
  constexpr int CW = 128 / (int)sizeof(OUT);  // columns of one 128-byte block
  extern __shared__ __align__(1024) uint8_t smem[];  // swizzle atoms start on 1024-byte boundaries
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + C_::STAGES * C_::A_BYTES;
  uint8_t* staging = smem + C_::STAGES * C_::STAGE_BYTES;
  float* vecs = reinterpret_cast<float*>(staging + C_::STAGING);  // channel scales [BN], bias [BN]
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + C_::STAGING + C_::VECS);
  uint64_t* full_bar = bars;                         // [STAGES] (leader's are used)
  uint64_t* empty_bar = bars + C_::STAGES;           // [STAGES]
  uint64_t* tfull_bar = bars + 2 * C_::STAGES;       // [2]
  uint64_t* tempty_bar = bars + 2 * C_::STAGES + 2;  // [2] (leader's are used)
  uint64_t* drain_bar = bars + 2 * C_::STAGES + 4;   // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C_::STAGES + 5);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank();  // 0 = leader
  const int num_m = (args.M + 255) / 256;
  const int num_n = (args.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int num_kb = (args.K + kStageK - 1) / kStageK;
  const int pair = blockIdx.x / 2, npairs = gridDim.x / 2;
  int* err = args.err;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C_::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull_bar[i], 1);
      mbar_init(&tempty_bar[i], 8);
    }
    mbar_init(drain_bar, 1);
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (c_tma) tma_prefetch_desc(&tmC);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, C_::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers exist and the paired TMEM is allocated
  dependency_release();
  dependency_wait();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued[C_::STAGES] = {};
      bool ok = true;
      const uint32_t fb0 = peer_addr(smem_u32(&full_bar[0]), 0);  // the leader's barriers
      for (int t = pair; t < num_tiles && ok; t += npairs) {
        int mt, nt;
        pair_tile(t, num_m, num_n, args.N % BN != 0, mt, nt);
        // a narrow tile multiplies only the columns it has, half of them from each CTA
        const int half = min(BN / 2, ((args.N - nt * BN + 31) / 32) * 16);
        const int m0 = mt * 256 + (int)rank * 128, n0 = nt * BN + (int)rank * half;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, err, 61)) { ok = false; break; }
          const uint32_t fb = fb0 + stage * 8;
          const int atoms = min(kStageK / 128, (args.K - kb * kStageK + 127) / 128);  // the last stage may be half
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * C_::STAGE_BYTES / (kStageK / 128) * atoms);
          for (int h = 0; h < atoms; ++h) {
            const int k0 = kb * kStageK + h * 128;
            tma_load_2d_pair(smem_a + stage * C_::A_BYTES + h * C_::A_ATOM, &tmA, fb, k0, m0);
            tma_load_2d_pair(smem_b + stage * C_::B_BYTES + h * C_::B_ATOM, &tmB, fb, k0, n0);
          }
          issued[stage]++;
          if (++stage == C_::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // this CTA's copies land before it can pass the final cluster barrier:
      // the stage's empty barrier turns once the leader consumed it
      for (int s = 0; s < C_::STAGES; ++s)
        if (issued[s] > 0) mbar_wait_drain(&empty_bar[s], (uint32_t)((issued[s] - 1) & 1));
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader CTA) ----------------
    // The whole warp keeps the loop's state, so that it stays in uniform registers; one lane issues
    // (a lone thread moved each descriptor to uniform registers for each MMA: 169 us, not 156).
    if (rank == 0) {
      const bool issue = elect_one();
      const uint64_t a0 = make_sdesc(smem_u32(smem_a), 16, 1024, kLayoutSw128);
      const uint64_t b0 = make_sdesc(smem_u32(smem_b), 16, 1024, kLayoutSw128);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += npairs, ++local) {
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!warp_wait(&tempty_bar[acc], acc_phase ^ 1, err, 62)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        int mt, nt;
        pair_tile(t, num_m, num_n, args.N % BN != 0, mt, nt);
        const uint32_t idesc = make_idesc_s8(256, 2 * min(BN / 2, ((args.N - nt * BN + 31) / 32) * 16));
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!warp_wait(&full_bar[stage], phase, err, 63)) { ok = false; break; }
          tc_fence_after();
          const uint64_t ad = a0 + (uint64_t)(stage * (C_::A_BYTES >> 4));
          const uint64_t bd = b0 + (uint64_t)(stage * (C_::B_BYTES >> 4));
          const bool second = kb * kStageK + 128 < args.K;
          if (issue) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              mma_s8_pair(d_tmem, ad + r * 2, bd + r * 2, idesc, (kb > 0 || r > 0) ? 1u : 0u);
            if (second) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                mma_s8_pair(d_tmem, ad + (C_::A_ATOM >> 4) + r * 2, bd + (C_::B_ATOM >> 4) + r * 2, idesc, 1u);
            }
            mma_commit_both(&empty_bar[stage]);
          }
          __syncwarp();
          if (++stage == C_::STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (issue) mma_commit_both(&tfull_bar[acc]);
        __syncwarp();
      }
      if (issue) mma_commit_both(drain_bar);
      __syncwarp();
    }
    // both CTAs: the pair's MMAs are done before the paired TMEM goes away
    if (lane == 0) mbar_wait_drain(drain_bar, 0);
  } else {
    // ---------------- epilogue (warps 2..5, both CTAs) ----------------
    const int quarter = warp & 3;
    const int et = threadIdx.x - 64;
    uint8_t* const stage_out = staging + (warp - 2) * 8192;
    int local = 0, nbuf = 0;
    bool ok = true;  // after a failed wait the warp only keeps meeting the others at the barriers
    const uint32_t te_leader[2] = {peer_addr(smem_u32(&tempty_bar[0]), 0), peer_addr(smem_u32(&tempty_bar[1]), 0)};
    // a tile's scales and bias are fetched while the one before it is being stored
    constexpr int VPT = (BN + 127) / 128;
    float sa_next = 0.f, sb_next[VPT], bias_next[VPT];
    auto fetch = [&](int t) {
      int mt, nt;
      pair_tile(t, num_m, num_n, args.N % BN != 0, mt, nt);
      const int m = mt * 256 + (int)rank * 128 + quarter * 32 + lane;
      sa_next = m < args.M ? args.sa[m] : 0.f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = et + i * 128, n = nt * BN + j;
        const bool in = j < BN && n < args.N;
        sb_next[i] = in ? args.sb[n] : 0.f;
        bias_next[i] = in ? bias_at(args, n) : 0.f;
      }
    };
    if (pair < num_tiles) fetch(pair);
    for (int t = pair; t < num_tiles; t += npairs, ++local) {
      int mt, nt;
      pair_tile(t, num_m, num_n, args.N % BN != 0, mt, nt);
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      const int mw = mt * 256 + (int)rank * 128 + quarter * 32;  // the warp's first row
      const float sa = sa_next;
      if (local > 0) epilogue_barrier();  // every warp is done with the last tile's
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = et + i * 128;
        if (j < BN) {
          vecs[j] = sb_next[i];
          vecs[BN + j] = bias_next[i];
        }
      }
      epilogue_barrier();
      if (t + npairs < num_tiles) fetch(t + npairs);
      ok = ok && warp_wait(&tfull_bar[acc], acc_phase, err, 64);
      if (!ok) continue;
      tc_fence_after();
      const uint32_t tbase = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN;
#pragma unroll 1
      for (int c = 0; c < BN / CW; ++c) {
        const int n0 = nt * BN + c * CW;
        if (n0 >= args.N || mw >= args.M) break;
        uint8_t* const buf = stage_out + (nbuf & 1) * 4096;
        ++nbuf;
        if (lane == 0) bulk_wait_read<1>();  // the store that last read this buffer is done with it
        __syncwarp();
        uint8_t* const brow = buf + lane * 128;
#pragma unroll
        for (int g = 0; g < CW / 32; ++g) {
          uint32_t v[32];
          tmem_ld32(tbase + c * CW + g * 32, v);
          tmem_wait_ld();
#pragma unroll
          for (int j4 = 0; j4 < 8; ++j4) {
            const float4 s4 = *reinterpret_cast<const float4*>(vecs + c * CW + g * 32 + j4 * 4);
            float4 b4 = make_float4(0.f, 0.f, 0.f, 0.f);
            if (args.bias != nullptr) b4 = *reinterpret_cast<const float4*>(vecs + BN + c * CW + g * 32 + j4 * 4);
            const float x0 = fmaf((float)(int)v[4 * j4 + 0] * sa, s4.x, b4.x);
            const float x1 = fmaf((float)(int)v[4 * j4 + 1] * sa, s4.y, b4.y);
            const float x2 = fmaf((float)(int)v[4 * j4 + 2] * sa, s4.z, b4.z);
            const float x3 = fmaf((float)(int)v[4 * j4 + 3] * sa, s4.w, b4.w);
            if constexpr (sizeof(OUT) == 2) {
              v[2 * j4] = pack_bf16x2(x0, x1);
              v[2 * j4 + 1] = pack_bf16x2(x2, x3);
            } else {
              *reinterpret_cast<float4*>(brow + ((j4 ^ (lane & 7)) << 4)) = make_float4(x0, x1, x2, x3);
            }
          }
          if constexpr (sizeof(OUT) == 2) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint4*>(brow + (((g * 4 + q) ^ (lane & 7)) << 4)) =
                  make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          }
        }
        if (c_tma) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmC, buf, n0, mw);
            bulk_commit();
          }
        } else {
          __syncwarp();
          const int rows = min(32, args.M - mw), cols = min(CW, args.N - n0);
          for (int r = 0; r < rows; ++r) {
            OUT* crow = reinterpret_cast<OUT*>(args.C) + (long)(mw + r) * args.ldc + n0;
#pragma unroll
            for (int j = lane; j < CW; j += 32) {
              const int byte = j * (int)sizeof(OUT);
              if (j < cols)
                crow[j] = *reinterpret_cast<const OUT*>(buf + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15));
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(te_leader[acc]);
    }
    if (lane == 0) bulk_wait_read<0>();  // the staging buffers outlive the stores that read them
  }

  tc_fence_before();
  cluster_sync_all();  // neither CTA frees its half of the pair's TMEM while the other still works
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, C_::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// Few tokens or few channels.  A CTA multiplies 128 channels (the MMA's M) by NT
// tokens (its N) over its share of K; a cluster of `splits` CTAs along x covers
// K.  Each CTA of a split tile leaves its integer sums in its shared memory, the
// cluster meets, and rank r adds and stores the r-th part of the tokens, read from
// every rank's memory: one launch, no workspace, and the same sum in any order.
// ---------------------------------------------------------------------------
template <int NT>
struct RowsCfg {
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = NT * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = NT == 256 ? 4 : NT == 128 ? 6 : 8;
  static constexpr int SUMS = NT * 128 * 4;  // the tile's integer sums [NT][128], over the pipeline's buffers
  static constexpr int TMEM_COLS = NT < 32 ? 32 : NT;
  static constexpr int PIPE = STAGES * STAGE_BYTES;
  static constexpr int SMEM_BYTES = PIPE + NT * 4 + 256;
  static_assert(SUMS <= PIPE && SMEM_BYTES <= 232448, "rows GEMM stages");
};

__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// Four neighbouring channels of token m.
template <typename OUT>
__device__ __forceinline__ void store_out4(const S8Args& a, long m, int n, float v0, float v1, float v2, float v3) {
  OUT* c = reinterpret_cast<OUT*>(a.C) + m * a.ldc + n;
  if (a.c_vec4 && n + 4 <= a.N) {
    if constexpr (sizeof(OUT) == 2) *reinterpret_cast<uint2*>(c) = make_uint2(pack_bf16x2(v0, v1), pack_bf16x2(v2, v3));
    else *reinterpret_cast<float4*>(c) = make_float4(v0, v1, v2, v3);
    return;
  }
  const float v[4] = {v0, v1, v2, v3};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.N) continue;
    if constexpr (sizeof(OUT) == 2) c[i] = __float2bfloat16(v[i]);
    else c[i] = v[i];
  }
}

template <int NT, typename OUT>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_s8_rows(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const S8Args args,
                 int splits) {
  using C_ = RowsCfg<NT>;
  extern __shared__ __align__(1024) uint8_t smem[];  // swizzle atoms start on 1024-byte boundaries
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + C_::STAGES * C_::A_BYTES;
  float* tok_scale = reinterpret_cast<float*>(smem + C_::PIPE);  // [NT]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C_::PIPE + NT * 4);
  uint64_t* full_bar = bars;                    // [STAGES]
  uint64_t* empty_bar = bars + C_::STAGES;      // [STAGES]
  uint64_t* done_bar = bars + 2 * C_::STAGES;   // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C_::STAGES + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int rank = splits > 1 ? (int)cluster_rank() : 0;
  const int num_n = (args.N + 127) / 128;
  const int tile = blockIdx.x / splits;
  const int n0 = (tile % num_n) * 128;
  const int m0 = (tile / num_n) * NT;
  const int all_kb = (args.K + 127) / 128;
  const int kb0 = (int)((long)all_kb * rank / splits), kb1 = (int)((long)all_kb * (rank + 1) / splits);
  int* err = args.err;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C_::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C_::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  dependency_release();
  dependency_wait();
  const uint32_t tmem_base = *tmem_slot;
  bool have = false;  // epilogue warps: this CTA's sums are in tensor memory
  const int n = n0 + lane * 4;  // a lane's channels in the last step
  float sb[4] = {}, bias[4] = {};

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued[C_::STAGES] = {};
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1, err, 71)) break;
        mbar_arrive_expect_tx(&full_bar[stage], C_::STAGE_BYTES);
        tma_load_2d(smem_a + stage * C_::A_BYTES, &tmW, &full_bar[stage], kb * 128, n0);
        tma_load_2d(smem_b + stage * C_::B_BYTES, &tmX, &full_bar[stage], kb * 128, m0);
        issued[stage]++;
        if (++stage == C_::STAGES) { stage = 0; phase ^= 1; }
      }
      // every copy this thread issued has landed before the CTA can exit
      for (int s = 0; s < C_::STAGES; ++s)
        if (issued[s] > 0) mbar_wait_drain(&full_bar[s], (uint32_t)((issued[s] - 1) & 1));
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_s8(128, NT);
    const bool issue = elect_one();
    const uint64_t a0 = make_sdesc(smem_u32(smem_a), 16, 1024, kLayoutSw128);
    const uint64_t b0 = make_sdesc(smem_u32(smem_b), 16, 1024, kLayoutSw128);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait(&full_bar[stage], phase, err, 72)) break;
      tc_fence_after();
      if (issue) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          mma_s8(tmem_base, a0 + (uint64_t)(stage * (C_::A_BYTES >> 4) + r * 2),
                 b0 + (uint64_t)(stage * (C_::B_BYTES >> 4) + r * 2), idesc, (kb > kb0 || r > 0) ? 1u : 0u);
        mma_commit(&empty_bar[stage]);
      }
      __syncwarp();
      if (++stage == C_::STAGES) { stage = 0; phase ^= 1; }
    }
    // arrives once every MMA issued above has completed
    if (issue) mma_commit(done_bar);
    __syncwarp();
    if (lane == 0) mbar_wait_drain(done_bar, 0);
  } else {
    const int quarter = warp & 3;
    const int ch = quarter * 32 + lane;
    for (int j = threadIdx.x - 64; j < NT; j += 128) tok_scale[j] = m0 + j < args.M ? args.sa[m0 + j] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i < args.N) {
        sb[i] = args.sb[n + i];
        bias[i] = bias_at(args, n + i);
      }
    }
    have = warp_wait(done_bar, 0, err, 73);
    tc_fence_after();
    const uint32_t tbase = tmem_base + ((uint32_t)(quarter * 32) << 16);
    constexpr int W = NT < 32 ? NT : 32;  // tokens a step
    // the pipeline's buffers are free: every copy into them was consumed by an MMA that is done
    int* sums = reinterpret_cast<int*>(smem);
#pragma unroll 1
    for (int c = 0; c < NT && have && m0 + c < args.M; c += W) {
      uint32_t v[W];
      if constexpr (W == 32) tmem_ld32(tbase + c, v);
      else tmem_ld16(tbase + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < W; ++j) sums[(c + j) * 128 + ch] = (int)v[j];
    }
  }

  tc_fence_before();
  if (splits > 1) cluster_sync_all();  // every rank's sums are written
  else __syncthreads();
  if (warp >= 2 && have) {
    // a warp takes every fourth token of this rank's share, a lane four channels of it
    const int t0 = rank * NT / splits, t1 = (rank + 1) * NT / splits;
    const uint32_t mine = smem_u32(smem) + (uint32_t)lane * 16;
#pragma unroll 4
    for (int j = t0 + warp - 2; j < t1; j += 4) {
      if (m0 + j >= args.M) break;
      int4 sum = make_int4(0, 0, 0, 0);
      if (splits > 1) {
        for (int r = 0; r < splits; ++r) {
          const int4 v = ld_cluster_v4(peer_addr(mine + (uint32_t)j * 512, (uint32_t)r));
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
      } else {
        sum = *reinterpret_cast<const int4*>(smem + j * 512 + lane * 16);
      }
      const float sa = tok_scale[j];
      store_out4<OUT>(args, m0 + j, n, fmaf((float)sum.x * sa, sb[0], bias[0]), fmaf((float)sum.y * sa, sb[1], bias[1]),
                      fmaf((float)sum.z * sa, sb[2], bias[2]), fmaf((float)sum.w * sa, sb[3], bias[3]));
    }
  }
  if (splits > 1) cluster_sync_all();  // no rank's memory goes away while another reads it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C_::TMEM_COLS);
  }
}

// 2-D map over a row-major [rows, cols] matrix with row stride `ld_bytes`; box =
// 128 bytes x box_rows, 128-byte swizzle.
CUtensorMap make_map(const void* base, CUtensorMapDataType type, int esize, long rows, long cols, long ld_bytes,
                     int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld_bytes};
  cuuint32_t box[2] = {(cuuint32_t)(128 / esize), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = get_encode_fn()(&m, type, 2, const_cast<void*>(base), dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "harp gemm_s8: cuTensorMapEncodeTiled failed (", std::to_string((int)r), ")");
  return m;
}
CUtensorMap make_map_s8(const int8_t* base, long rows, long cols, long ld, int box_rows) {
  return make_map(base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, cols, ld, box_rows);
}

// Clusters of `cluster` blocks that the device keeps resident at once (GPC shapes leave
// SMs over), with the kernel set up for its shared memory.
template <typename... P>
int resident_clusters(void (*kern)(P...), int cluster, int smem) {
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(num_sms() / cluster * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  C10_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
  return std::max(1, n);
}

template <int BN, typename OUT>
void launch_pair(const S8Args& a, bool c_tma, int device, cudaStream_t stream) {
  using C_ = PairCfg<BN>;
  auto kern = gemm_s8_pair<BN, OUT>;
  static PerDevice<int> clusters;
  const int max_clusters = clusters.get(device, [&] { return resident_clusters(kern, 2, C_::SMEM_BYTES); });
  const CUtensorMap ta = make_map_s8(a.A, a.M, a.K, a.lda, 128), tb = make_map_s8(a.B, a.N, a.K, a.ldb, BN / 2);
  CUtensorMap tc = ta;
  if (c_tma)
    tc = make_map(a.C, sizeof(OUT) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                  sizeof(OUT), a.M, a.N, a.ldc * (long)sizeof(OUT), 32);
  const long tiles = (long)((a.M + 255) / 256) * ((a.N + BN - 1) / BN);
  TORCH_CHECK(tiles <= 0x3FFFFFFF, "harp gemm_s8: too many tiles");
  launch_dependent(kern, dim3(2 * (unsigned)std::min<long>(tiles, max_clusters)), dim3(kThreads), C_::SMEM_BYTES, stream,
                   2, ta, tb, tc, a, c_tma ? 1 : 0);
  count_launch();
}

template <int NT, typename OUT>
void launch_rows(const S8Args& a, int splits, int device, cudaStream_t stream) {
  using C_ = RowsCfg<NT>;
  auto kern = gemm_s8_rows<NT, OUT>;
  static PerDevice<bool> configured;
  configured.get(device, [&] {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C_::SMEM_BYTES));
    return true;
  });
  const CUtensorMap tw = make_map_s8(a.B, a.N, a.K, a.ldb, 128), tx = make_map_s8(a.A, a.M, a.K, a.lda, NT);
  const long ctas = (long)((a.N + 127) / 128) * ((a.M + NT - 1) / NT) * splits;
  TORCH_CHECK(ctas <= 0x7FFFFFFF, "harp gemm_s8: too many tiles");
  launch_dependent(kern, dim3((unsigned)ctas), dim3(kThreads), C_::SMEM_BYTES, stream, splits, tw, tx, a, splits);
  count_launch();
}

// CTAs of the rows kernel that run at once in clusters of `splits` (larger clusters
// leave SMs of a GPC over).
long cluster_slots(int splits, int device) {
  static PerDevice<long> slots[9];
  if (splits == 1) return num_sms();
  return slots[splits].get(device, [&] {
    return (long)splits * resident_clusters(gemm_s8_rows<16, bf16>, splits, RowsCfg<16>::SMEM_BYTES);
  });
}
// The kernel and its tile by estimated time.  The constants are microseconds
// measured on a B200: an SM takes in 135 KB a microsecond, all of them 14 MB; a pair
// multiplies 256 x BN x 128 in 0.0014 BN; the epilogues take time by the columns a
// CTA stores; a second wave of single-tile CTAs starts only when the first is done.
// Of 45 shapes (M = 1 .. 17408, N = 24 .. 9216, K = 32 .. 6144) timed with every tile
// and split, weights in L2 and not, the choice was within 8 % of the fastest at 42 and
// within 20 % at all: 4 x 1152 x 4608 takes 4.7 us with 8 splits and 9.5 with one; 4 x 6912 x
// 1152 4.3 with one split and 8.1 with 4; 128 x 9216 x 1152 6.0 in the rows kernel and 6.4 on
// CTA pairs; 1088 x 9216 x 1152 14.6 to 17.5 on CTA pairs and 30 in the rows kernel.  It does not
// know of outputs that TMA cannot store: 1061 x 1003 x 1155 into such rows of fp32 takes 12 us, 1061 x
// 1008 x 1155 7.7.
struct Plan {
  int pair_bn;  // 256 / 192 / 128, or 0: the rows kernel with
  int nt, splits;
};
Plan pick(const S8Args& a, int device) {
  const int sms = num_sms();
  const long chans = (a.N + 127) / 128;
  const int kb = (a.K + 127) / 128;
  auto load = [&](long ctas, double bytes) {
    return bytes * std::max(1.0 / 135e3, (double)std::min<long>(ctas, sms) / 14e6);
  };
  Plan best = {0, 16, 1};
  double best_t = 1e30;
  for (int nt : {16, 32, 64, 128, 256}) {
    const long tiles = chans * ((a.M + nt - 1) / nt);
    for (int sp = 1; sp <= 8 && sp <= kb; ++sp) {
      const long slots = cluster_slots(sp, device);
      const long waves = (tiles * sp + slots - 1) / slots;
      const double one = 4.0 + (kb + sp - 1) / sp * load(tiles * sp, 16384 + 128 * nt) + 0.016 * nt +
                         (sp == 1 ? 0.0 : sp <= 3 ? 1.0 : 0.5);
      const double t = 2.0 + waves * (one - 2.0);
      if (t < best_t) { best_t = t; best = {0, nt, sp}; }
    }
  }
  for (int bn : {128, 192, 256}) {
    const long tiles = (long)((a.M + 255) / 256) * ((a.N + bn - 1) / bn);
    const long waves = (tiles + sms / 2 - 1) / (sms / 2);
    const double stage = load(2 * tiles, (128 + bn / 2) * 128);
    const double t = 3.5 + 0.0125 * bn + kb * stage + (waves - 1) * (kb * std::max(stage, 0.0014 * bn) + 0.5);
    if (t < best_t) { best_t = t; best = {bn, 0, 0}; }
  }
  return best;
}

// pick(), with the plans of the sizes at hand kept: the estimate takes about a microsecond on the host.
Plan plan_of(const S8Args& a, int device) {
  struct Known {
    int device = -1, M = -1, N = -1, K = -1;
    Plan p = {};
  };
  static thread_local Known known[64];
  Known& k = known[((unsigned)a.M * 7u + (unsigned)a.N * 31u + (unsigned)a.K * 131u) % 64u];
  if (k.device != device || k.M != a.M || k.N != a.N || k.K != a.K) k = {device, a.M, a.N, a.K, pick(a, device)};
  return k.p;
}

template <typename OUT>
void dispatch(const S8Args& a, bool c_tma, int device, cudaStream_t stream) {
  const Plan p = plan_of(a, device);
  switch (p.pair_bn) {
    case 256: launch_pair<256, OUT>(a, c_tma, device, stream); return;
    case 192: launch_pair<192, OUT>(a, c_tma, device, stream); return;
    case 128: launch_pair<128, OUT>(a, c_tma, device, stream); return;
    default: break;
  }
  switch (p.nt) {
    case 16: launch_rows<16, OUT>(a, p.splits, device, stream); break;
    case 32: launch_rows<32, OUT>(a, p.splits, device, stream); break;
    case 64: launch_rows<64, OUT>(a, p.splits, device, stream); break;
    case 128: launch_rows<128, OUT>(a, p.splits, device, stream); break;
    default: launch_rows<256, OUT>(a, p.splits, device, stream); break;
  }
}

// Rows to 16-byte boundaries, `groups` groups of 16 bytes a row: a thread a group, read by words of W
// (four bytes if the source's address, stride and K are multiples of four, else one: a product of 8704 x
// 1008 x 4100 takes 47 us with the one, 64 with the other, 35 without copies).  What is past K is zero.
template <typename W>
__global__ void __launch_bounds__(256) copy_rows_kernel(const int8_t* src, long ld, long rows, int K, int groups,
                                                        uint4* dst) {
  dependency_wait();
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * groups) return;
  const long row = i / groups;
  const int k0 = (int)(i - row * groups) * 16;
  union {
    W w[16 / sizeof(W)];
    uint4 v;
  } u;
  u.v = make_uint4(0u, 0u, 0u, 0u);
  const int8_t* const p = src + row * ld + k0;
#pragma unroll
  for (int j = 0; j < 16; j += (int)sizeof(W))
    if (k0 + j < K) u.w[j / sizeof(W)] = *reinterpret_cast<const W*>(p + j);
  dst[i] = u.v;
}
// An empty sum: the epilogue of zeros.
template <typename OUT>
__global__ void __launch_bounds__(256) empty_sum_kernel(const S8Args a) {
  dependency_wait();
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)a.M * a.N) return;
  const long m = i / a.N;
  const int n = (int)(i - m * a.N);
  const float v = fmaf(0.f * a.sa[m], a.sb[n], bias_at(a, n));
  OUT* const c = reinterpret_cast<OUT*>(a.C) + m * a.ldc + n;
  if constexpr (sizeof(OUT) == 2) *c = __float2bfloat16(v);
  else *c = v;
}
unsigned blocks_of(long threads) {
  const long blocks = (threads + 255) / 256;
  TORCH_CHECK(blocks <= 0x7FFFFFFFL, "harp gemm_s8: too many rows");
  return (unsigned)blocks;
}

// t, or a copy (of whole 16-byte groups) whose rows TMA can address: starting on 16-byte boundaries, not overlapping.
at::Tensor addressable_rows(const at::Tensor& t, cudaStream_t stream) {
  const int64_t rows = t.size(0), K = t.size(1);
  if ((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 &&
      (rows == 1 || (t.stride(0) % 16 == 0 && t.stride(0) >= K)))
    return t;
  const int groups = (int)((K + 15) / 16);
  at::Tensor c(at::detail::empty_cuda({rows, groups * 16L}, at::kChar, t.device(), c10::nullopt));
  const int8_t* src = reinterpret_cast<const int8_t*>(t.data_ptr());
  uint4* dst = reinterpret_cast<uint4*>(c.data_ptr());
  const long ld = rows == 1 ? 0 : t.stride(0);
  auto kern = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)ld | (uintptr_t)K) & 3) == 0 ? copy_rows_kernel<uint32_t>
                                                                                             : copy_rows_kernel<uint8_t>;
  launch_dependent(kern, blocks_of(rows * groups), 256, 0, stream, 1, src, ld, (long)rows, (int)K, groups, dst);
  count_launch();
  return c;
}

void check_scales(const at::Tensor& s, const at::Tensor& rows, const char* name) {
  TORCH_CHECK(s.is_cuda() && s.device() == rows.device() && s.scalar_type() == at::kFloat && s.dim() == 1 &&
                  s.size(0) == rows.size(0) && (s.size(0) <= 1 || s.stride(0) == 1),
              "harp gemm_s8: ", name, " must be a dense fp32 vector with a scale for each row, on the operands' device");
}

}  // namespace

void gemm_s8_out(const at::Tensor& A, const at::Tensor& sa, const at::Tensor& B, const at::Tensor& sb,
                 const c10::optional<at::Tensor>& bias, at::Tensor C, at::Tensor err) {
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && C.is_cuda() && err.is_cuda(), "harp gemm_s8: CUDA tensors required");
  TORCH_CHECK(A.device() == B.device() && A.device() == C.device() && A.device() == err.device(),
              "harp gemm_s8: operands on one device");
  TORCH_CHECK(A.scalar_type() == at::kChar && B.scalar_type() == at::kChar, "harp gemm_s8: int8 operands");
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && C.dim() == 2, "harp gemm_s8: 2-D operands");
  const int64_t M = A.size(0), N = B.size(0), K = A.size(1);
  TORCH_CHECK(B.size(1) == K, "harp gemm_s8: A has ", std::to_string(K), " columns and B ", std::to_string(B.size(1)));
  TORCH_CHECK(C.size(0) == M && C.size(1) == N, "harp gemm_s8: C shape");
  TORCH_CHECK(K <= kMostK, "harp gemm_s8: K = ", std::to_string(K), " could overflow the 32-bit sums (at most 131071)");
  TORCH_CHECK(M <= kMostRows && N <= kMostRows, "harp gemm_s8: M and N below 2^31");
  TORCH_CHECK((A.stride(1) == 1 || K <= 1) && (B.stride(1) == 1 || K <= 1) && (C.stride(1) == 1 || N <= 1),
              "harp gemm_s8: unit inner stride");
  TORCH_CHECK(M <= 1 || C.stride(0) >= N, "harp gemm_s8: rows of C overlap");
  TORCH_CHECK(C.scalar_type() == at::kBFloat16 || C.scalar_type() == at::kFloat, "harp gemm_s8: bf16 or fp32 output");
  TORCH_CHECK(err.scalar_type() == at::kInt && err.numel() >= 4, "harp gemm_s8: error word");
  check_scales(sa, A, "a_scale");
  check_scales(sb, B, "b_scale");
  if (bias.has_value())
    TORCH_CHECK(bias->is_cuda() && bias->device() == A.device() && bias->dim() == 1 && bias->size(0) == N &&
                    (N <= 1 || bias->stride(0) == 1) &&
                    (bias->scalar_type() == at::kBFloat16 || bias->scalar_type() == at::kFloat),
                "harp gemm_s8: bias must be a dense bf16 or fp32 vector of ", std::to_string(N), " values on the operands' device");
  if (M == 0 || N == 0) return;
  const at::cuda::CUDAGuard guard(A.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  S8Args a = {};
  a.M = (int)M; a.N = (int)N; a.K = (int)K;
  a.sa = sa.data_ptr<float>();
  a.sb = sb.data_ptr<float>();
  a.bias = bias.has_value() ? bias->data_ptr() : nullptr;
  a.bias_f32 = bias.has_value() && bias->scalar_type() == at::kFloat;
  a.C = C.data_ptr();
  a.ldc = C.stride(0);
  a.err = err.data_ptr<int>();
  if (K == 0) {
    auto kern = C.scalar_type() == at::kFloat ? empty_sum_kernel<float> : empty_sum_kernel<bf16>;
    launch_dependent(kern, blocks_of(M * N), 256, 0, stream, 1, a);
    count_launch();
    return;
  }
  const at::Tensor Ar = addressable_rows(A, stream), Br = addressable_rows(B, stream);
  a.A = reinterpret_cast<const int8_t*>(Ar.data_ptr());
  a.B = reinterpret_cast<const int8_t*>(Br.data_ptr());
  const long pad = (K + 15) / 16 * 16;  // a single row's stride is never used, but has to be valid
  a.lda = M == 1 ? pad : Ar.stride(0);
  a.ldb = N == 1 ? pad : Br.stride(0);
  const uintptr_t where =
      reinterpret_cast<uintptr_t>(a.C) | (M == 1 ? 0 : (uintptr_t)(a.ldc * (long)C.element_size()));
  a.c_vec4 = where % (4 * C.element_size()) == 0;
  // TMA stores whole 16-byte groups: past a width that ends inside one it would overwrite what lies beside C
  const bool c_tma = where % 16 == 0 && N * C.element_size() % 16 == 0 && M > 1;
  if (C.scalar_type() == at::kFloat) dispatch<float>(a, c_tma, A.get_device(), stream);
  else dispatch<bf16>(a, c_tma, A.get_device(), stream);
}

at::Tensor gemm_s8(const at::Tensor& A, const at::Tensor& sa, const at::Tensor& B, const at::Tensor& sb,
                   const c10::optional<at::Tensor>& bias, bool f32, at::Tensor err) {
  TORCH_CHECK(A.is_cuda() && A.dim() == 2 && B.dim() == 2, "harp gemm_s8: 2-D CUDA operands");
  at::Tensor C(at::detail::empty_cuda({A.size(0), B.size(0)}, f32 ? at::kFloat : at::kBFloat16, A.device(), c10::nullopt));
  gemm_s8_out(A, sa, B, sb, bias, C, err);
  return C;
}

// The kernel that a product of these sizes runs on the current device: (pair tile's columns, 0, 0) or
// (0, tokens a CTA, splits of K).
std::tuple<int64_t, int64_t, int64_t> gemm_s8_plan(int64_t M, int64_t N, int64_t K) {
  TORCH_CHECK(M >= 1 && M <= kMostRows && N >= 1 && N <= kMostRows && K >= 1 && K <= kMostK,
              "harp gemm_s8: no plan for these sizes");
  S8Args a = {};
  a.M = (int)M; a.N = (int)N; a.K = (int)K;
  const Plan p = plan_of(a, at::cuda::current_device());
  if (p.pair_bn != 0) return {p.pair_bn, 0, 0};
  return {0, p.nt, p.splits};
}

}  // namespace harp
