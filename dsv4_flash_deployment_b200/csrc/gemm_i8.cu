// 8-bit integer matrix product with a scale per token and per output channel:
//
//   out[t][n] = (sum_k x[t][k] * w[n][k]) * xs[t] * ws[n]
//
// x, w int8, the sum exact in int32 (K <= 131071: no sum of int8 products can pass
// 2^31), converted to fp32 once and multiplied by the two scales, rounded once to
// the output type.  Integer sums do not depend on their order, so neither does the
// result, however K is split.
//
// tcgen05.mma kind::i8.  The weight's rows ride on the 128-row M side and tokens on
// the N side (32..256), as in gemm.cu: a decode batch of a few tokens then wastes
// the narrow side.  Both operands come by TMA in 128-byte k tiles whose out-of-range
// part reads as zero, so any T, N and K work without padded copies (rows have to
// start on 16-byte boundaries).
//
// Warp roles (192 threads): warp 0 TMA producer, warp 1 TMEM owner and MMA issuer,
// warps 2..5 epilogue.  Persistent over output tiles; two accumulators in TMEM, so
// the epilogue of a tile overlaps the products of the next.
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "gemm.h"

namespace dsv4 {

namespace {

// Instruction descriptor, kind::i8: int8 x int8 -> int32.
constexpr uint32_t idesc_i8(uint32_t m, uint32_t n) {
  return (2u << 4)            // D format s32
         | (1u << 7)          // A s8
         | (1u << 10)         // B s8
         | ((n >> 3) << 17) | ((m >> 4) << 24);
}

DSV4_DEV void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

template <typename TO>
DSV4_DEV TO out_of(float v);
template <>
DSV4_DEV float out_of<float>(float v) { return v; }
template <>
DSV4_DEV __nv_bfloat16 out_of<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
DSV4_DEV __half out_of<__half>(float v) { return __float2half_rn(v); }

template <int BN>
struct I8Smem {
  static constexpr int kA = 128 * 128;
  static constexpr int kB = BN * 128;
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int kBarriers = 256;
  static constexpr int kTotal = 1024 + kStages * kStage + kBarriers;
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr int kTmemCols = 2 * kAccCols;   // a power of two, 64 at least
  static_assert(kTotal <= 227 * 1024, "shared memory exceeds the per-CTA limit");
  static_assert(8 * (2 * kStages + 5) + 8 <= kBarriers, "barrier region too small");
};

}  // namespace

template <int BN, typename TO>
__global__ void __launch_bounds__(192, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, GemmI8Params p) {
  using L = I8Smem<BN>;
  constexpr int S = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S * L::kA;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sB + S * L::kB);
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* acc_full = bars + 2 * S;
  uint64_t* acc_empty = bars + 2 * S + 2;
  uint64_t* drain = bars + 2 * S + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  // tile -> (feature tile, token tile), token tiles of one feature tile next to each
  // other: CTAs that run together share the weight tile in L2
  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int w = blockIdx.x; w < p.n_tiles; w += gridDim.x) {
      const int m0 = w / p.t_tiles * 128, n0 = w % p.t_tiles * BN;
      for (int kt = 0; kt < p.k_tiles; ++kt) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.err, KID_GEMM, 11)) goto done;
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[stage], L::kStage);
          tma_load_2d(sA + stage * L::kA, &map_w, &full[stage], kt * 128, m0);
          tma_load_2d(sB + stage * L::kB, &map_x, &full[stage], kt * 128, n0);
        }
        __syncwarp();
        if (++stage == S) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    constexpr uint32_t idesc = idesc_i8(128, BN);
    for (int w = blockIdx.x; w < p.n_tiles; w += gridDim.x) {
      if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.err, KID_GEMM, 12)) goto done;
      tc_fence_after();
      const uint32_t d = tmem + acc * L::kAccCols;
      for (int kt = 0; kt < p.k_tiles; ++kt) {
        if (!mbar_wait(&full[stage], phase, abort_flag, p.err, KID_GEMM, 13)) goto done;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t a0 = smem_u32(sA + stage * L::kA), b0 = smem_u32(sB + stage * L::kB);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_i8(d, sdesc_kmajor_sw128(a0 + kk * 32), sdesc_kmajor_sw128(b0 + kk * 32), idesc,
                    (kt > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == S) stage = 0, phase ^= 1;
      }
      if (lane == 0) umma_commit(&acc_full[acc]);
      __syncwarp();
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
  } else {
    const int q = warp & 3;   // TMEM lane quadrant of this warp
    int acc = 0;
    uint32_t acc_phase = 0;
    TO* out = static_cast<TO*>(p.out);
    for (int w = blockIdx.x; w < p.n_tiles; w += gridDim.x) {
      const int n0 = w % p.t_tiles * BN, m = w / p.t_tiles * 128 + 32 * q + lane;
      const int nt = min(BN, p.T - n0);
      const float ws = m < p.N ? p.ws[m] : 0.f;
      if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.err, KID_GEMM, 14)) goto done;
      tc_fence_after();
      for (int c0 = 0; c0 < nt; c0 += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem + acc * L::kAccCols + ((uint32_t)(32 * q) << 16) + c0, r);
        tmem_ld_wait();
        if (m < p.N) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (c0 + j >= nt) break;
            const size_t t = (size_t)(n0 + c0 + j);
            out[t * p.ldo + m] = out_of<TO>((float)(int)r[j] * (ws * __ldg(p.xs + t)));
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
  }
done:
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) {   // no tensor-core op may still use the TMEM
      if (lane == 0) umma_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0, nullptr, p.err, KID_GEMM, 15);
    }
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// ------------------------------------------------------------------- host
namespace {

template <int BN, typename TO>
cudaError_t launch_i8(const CUtensorMap& mw, const CUtensorMap& mx, const GemmI8Params& p, int grid, cudaStream_t st) {
  using L = I8Smem<BN>;
  static std::atomic<uint64_t> configured{0};
  const cudaError_t e = smem_attr_once(gemm_i8_kernel<BN, TO>, L::kTotal, configured);
  if (e != cudaSuccess) return e;
  return launch_pdl(gemm_i8_kernel<BN, TO>, grid, 192, L::kTotal, st, mw, mx, p);
}

template <typename TO>
cudaError_t dispatch_i8(int bn, const CUtensorMap& mw, const CUtensorMap& mx, const GemmI8Params& p, int grid,
                        cudaStream_t st) {
  switch (bn) {
    case 32: return launch_i8<32, TO>(mw, mx, p, grid, st);
    case 64: return launch_i8<64, TO>(mw, mx, p, grid, st);
    case 128: return launch_i8<128, TO>(mw, mx, p, grid, st);
    default: return launch_i8<256, TO>(mw, mx, p, grid, st);
  }
}

}  // namespace

cudaError_t gemm_i8(const int8_t* x, size_t ldx, const int8_t* w, size_t ldw, GemmI8Params p, int otype, int sms,
                    cudaStream_t st) {
  if (p.T == 0 || p.N == 0) return cudaSuccess;
  const int bn = p.T <= 32 ? 32 : p.T <= 64 ? 64 : p.T <= 128 ? 128 : 256;
  p.t_tiles = (p.T + bn - 1) / bn;
  p.n_tiles = (p.N + 127) / 128 * p.t_tiles;
  p.k_tiles = (p.K + 127) / 128;
  CUtensorMap mw, mx;
  if (!make_tma_rows_u8(&mw, w, p.N, p.K, ldw, 128) || !make_tma_rows_u8(&mx, x, p.T, p.K, ldx, bn))
    return cudaErrorInvalidValue;
  const int grid = p.n_tiles < sms ? p.n_tiles : sms;
  switch (otype) {
    case F_BF16: return dispatch_i8<__nv_bfloat16>(bn, mw, mx, p, grid, st);
    case F_F16: return dispatch_i8<__half>(bn, mw, mx, p, grid, st);
    case F_F32: return dispatch_i8<float>(bn, mw, mx, p, grid, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace dsv4
