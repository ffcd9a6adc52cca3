// 8-bit integer matrix product with a scale per token and per output channel:
//
//   out[t][n] = (sum_k x[t][k] * w[n][k]) * xs[t] * ws[n]
//
// x, w int8, the sum exact in int32 (K <= 131071: no sum of int8 products can pass
// 2^31), converted to fp32 once and multiplied by the two scales, rounded once to
// the output type.  Integer sums do not depend on their order, so neither does the
// result, however K is split.
//
// Three kernels; gemm_i8() at the end chooses by the sizes:
//   rows   T <= 2: a warp per few weight rows, dp4a.  Bound by the weight's bytes.
//   tiles  tcgen05.mma kind::i8, one SM per 128 x BN tile, K split over a cluster
//          where the tiles are fewer than the SMs.
//   pairs  tcgen05.mma with cta_group::2, two SMs per 256 x 256 tile.
//
// In the tensor-core kernels the weight's rows ride on the 128-row M side and tokens
// on the N side (32..256), as in gemm.cu: a decode batch of a few tokens then wastes
// the narrow side.  Both operands come by TMA in 128-byte k tiles whose out-of-range
// part reads as zero, so any T, N and K work without padded copies (rows have to
// start on 16-byte boundaries).
//
// Warp roles (320 threads): warp 0 TMA producer, warp 1 TMEM owner and MMA issuer,
// warps 2..9 epilogue, two per TMEM lane quadrant, which take a tile's 32-token
// chunks in turn: a tile's epilogue has to fit beside the products of the next.
// Persistent over output tiles; two accumulators in TMEM, so the epilogue of a tile
// overlaps the products of the next.
#include <cuda_fp16.h>

#include <algorithm>
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

DSV4_DEV int dsmem_ld_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename TO>
DSV4_DEV TO out_of(float v);
template <>
DSV4_DEV float out_of<float>(float v) { return v; }
template <>
DSV4_DEV __nv_bfloat16 out_of<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
DSV4_DEV __half out_of<__half>(float v) { return __float2half_rn(v); }

// 16 weight bytes that no other warp will read
DSV4_DEV int4 ld_stream16(const int8_t* p) {
  int4 v;
  asm volatile("ld.global.L1::no_allocate.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
// the first n of 16 bytes, zeros behind them
DSV4_DEV int4 ld_tail16(const int8_t* p, int n) {
  if (n >= 16) return *reinterpret_cast<const int4*>(p);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < n) v[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
  return make_int4((int)v[0], (int)v[1], (int)v[2], (int)v[3]);
}
DSV4_DEV int dot16(int4 a, int4 b, int c) {
  return __dp4a(a.x, b.x, __dp4a(a.y, b.y, __dp4a(a.z, b.z, __dp4a(a.w, b.w, c))));
}

constexpr int kI8Threads = 320, kEpiWarps = 8;

template <int BN>
struct I8Smem {
  static constexpr int kA = 128 * 128;
  static constexpr int kB = BN * 128;
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int kBarriers = 256;
  static constexpr int kScales = kEpiWarps * 128 * 4;   // the tokens' scales of each epilogue warp
  static constexpr int kTotal = 1024 + kStages * kStage + kScales + kBarriers;
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr int kTmemCols = 2 * kAccCols;   // a power of two, 64 at least
  static_assert(kTotal <= 227 * 1024, "shared memory exceeds the per-CTA limit");
  static_assert(8 * (2 * kStages + 5) + 8 <= kBarriers, "barrier region too small");
  static_assert(kStages * kStage >= 128 * BN * 4, "a parked partial tile takes the stages' place");
};

// After an abort: waits, with mbar_wait's limit, for the copies into the stages last
// asked for, which nobody took.
template <int S>
DSV4_DEV void drain_copies(uint64_t* full, int issued, uint32_t* err, uint32_t detail) {
  for (int i = issued > S ? issued - S : 0; i < issued; ++i)
    if (!mbar_wait(&full[i % S], (uint32_t)(i / S) & 1, nullptr, err, KID_GEMM, detail)) return;
}

// Range of k tiles of one split.
DSV4_DEV int split_begin(int k_tiles, int splits, int i) { return (int)((long long)k_tiles * i / splits); }

// One 32-token column chunk of a tile: the integer sums of this lane's channel,
// scaled and stored (32 lanes write 32 neighbouring channels of a token).  The
// tokens' scales come from shared memory, four to a broadcast read (a shuffle per token
// instead: 12 k cycles a 256 x 256 fp32 tile against 11 k).  Whole chunks go without a
// test per store: with one a bf16 tile's epilogue took 13.5 k cycles, now 6.5 k.
template <typename TO>
DSV4_DEV void store_chunk(const uint32_t (&r)[32], int nt, const float4* xs, float ws, TO* out, size_t ldo, bool live) {
  float v[32];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 x = xs[j];
    v[4 * j] = (float)(int)r[4 * j] * (ws * x.x);
    v[4 * j + 1] = (float)(int)r[4 * j + 1] * (ws * x.y);
    v[4 * j + 2] = (float)(int)r[4 * j + 2] * (ws * x.z);
    v[4 * j + 3] = (float)(int)r[4 * j + 3] * (ws * x.w);
  }
  if (nt >= 32 && __all_sync(0xffffffffu, live)) {
#pragma unroll
    for (int j = 0; j < 32; ++j) out[j * ldo] = out_of<TO>(v[j]);
  } else if (live) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < nt) out[j * ldo] = out_of<TO>(v[j]);
  }
}

}  // namespace

template <int BN, typename TO>
__global__ void __launch_bounds__(kI8Threads, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, GemmI8Params p) {
  using L = I8Smem<BN>;
  constexpr int S = L::kStages;
  const int splits = p.splits;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S * L::kA;
  float* s_scale = reinterpret_cast<float*>(sB + S * L::kB);
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_scale + kEpiWarps * 128);
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* acc_full = bars + 2 * S;
  uint64_t* acc_empty = bars + 2 * S + 2;
  uint64_t* drain = bars + 2 * S + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int csyncs = 0, issued = 0;   // issued: k tiles the producer has asked for
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], kEpiWarps);
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
  pdl_trigger();   // only now: the next kernel's CTAs must not take the TMEM before this one
  pdl_wait();

  // Work unit -> (channel tile, token tile, split).  Token tiles of one channel tile
  // are next to each other: CTAs that run together share the weight tile in L2.  With
  // splits > 1 a unit is one CTA (no loop) and the splits of a tile are one cluster.
  // One lane alone runs the producer's and the issuer's loop: no warp barrier per k tile.
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < p.n_tiles * splits; u += gridDim.x) {
        const int w = u / splits, sp = u % splits;
        const int m0 = w / p.t_tiles * 128, n0 = w % p.t_tiles * BN;
        const int k1 = split_begin(p.k_tiles, splits, sp + 1);
        for (int kt = split_begin(p.k_tiles, splits, sp); kt < k1; ++kt) {
          if (!(ok = mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.err, KID_GEMM, 11))) break;
          mbar_arrive_expect_tx(&full[stage], L::kStage);
          tma_load_2d(sA + stage * L::kA, &map_w, &full[stage], kt * 128, m0);
          tma_load_2d(sB + stage * L::kB, &map_x, &full[stage], kt * 128, n0);
          ++issued;
          if (++stage == S) stage = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      constexpr uint32_t idesc = idesc_i8(128, BN);
      const uint64_t ad0 = sdesc_kmajor_sw128(smem_u32(sA)), bd0 = sdesc_kmajor_sw128(smem_u32(sB));
      bool ok = true;
      for (int u = blockIdx.x; ok && u < p.n_tiles * splits; u += gridDim.x) {
        const int sp = u % splits;
        const int nk = split_begin(p.k_tiles, splits, sp + 1) - split_begin(p.k_tiles, splits, sp);
        if (!(ok = mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.err, KID_GEMM, 12))) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * L::kAccCols;
        for (int kt = 0; kt < nk; ++kt) {
          if (!(ok = mbar_wait(&full[stage], phase, abort_flag, p.err, KID_GEMM, 13))) break;
          tc_fence_after();
          const uint64_t ad = ad0 + (uint64_t)(stage * (L::kA >> 4)), bd = bd0 + (uint64_t)(stage * (L::kB >> 4));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_i8(d, ad + 2 * kk, bd + 2 * kk, idesc, (kt | kk) != 0 ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == S) stage = 0, phase ^= 1;
        }
        if (!ok) break;
        umma_commit(&acc_full[acc]);
        if (++acc == 2) acc = 0, acc_phase ^= 1;
      }
    }
  } else {
    const int q = warp & 3;   // TMEM lane quadrant of this warp
    const int grp = (warp - 2) >> 2;
    const int row = 32 * q + lane;
    constexpr int kChunks = (BN / 32 + 1) / 2;   // 32-token chunks of a warp
    int acc = 0;
    uint32_t acc_phase = 0;
    TO* out = static_cast<TO*>(p.out);
    for (int u = blockIdx.x; u < p.n_tiles * splits; u += gridDim.x) {
      const int w = u / splits;
      const int n0 = w % p.t_tiles * BN, m = w / p.t_tiles * 128 + row;
      const int nt = min(BN, p.T - n0);
      const bool live = m < p.N;
      const float ws = live ? p.ws[m] : 0.f;
      float* xw = s_scale + (warp - 2) * 128;   // this warp's tokens, while the products run
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = 32 * (2 * i + grp) + lane;
        xw[32 * i + lane] = splits == 1 && c < nt ? p.xs[n0 + c] : 0.f;
      }
      __syncwarp();
      if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.err, KID_GEMM, 14)) goto done;
      tc_fence_after();
      const uint32_t d = tmem + acc * L::kAccCols + ((uint32_t)(32 * q) << 16);
      int* part = reinterpret_cast<int*>(smem);   // [token][128 channels], in the idle stages
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c0 = 32 * (2 * i + grp);
        if (c0 >= nt) break;
        uint32_t r[32];
        tmem_ld_32x32b_x32(d + c0, r);
        tmem_ld_wait();
        if (splits == 1) {
          store_chunk<TO>(r, nt - c0, reinterpret_cast<const float4*>(xw + 32 * i), ws,
                          out + (size_t)(n0 + c0) * p.ldo + m, p.ldo, live);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) part[(c0 + j) * 128 + row] = (int)r[j];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      if (splits > 1) {
        cluster_sync_all();   // every split's partial tile is parked
        ++csyncs;
        for (int c = (int)cluster_ctarank() * 2 + grp; c < nt; c += 2 * splits) {
          const float x = p.xs[n0 + c];
          const uint32_t local = smem_u32(part + c * 128 + row);
          int sum = 0;
#pragma unroll 8
          for (int r = 0; r < splits; ++r) sum += dsmem_ld_s32(dsmem_map(local, (uint32_t)r));
          if (live) out[(size_t)(n0 + c) * p.ldo + m] = out_of<TO>((float)sum * (ws * x));
        }
      }
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
  }
done:
  __syncwarp();
  // a cluster's threads take part in exactly two cluster barriers, also after an
  // abort, so that none waits for one that is gone or reads its shared memory then
  if (splits > 1)
    for (; csyncs < 2; ++csyncs) cluster_sync_all();
  tc_fence_before();
  __syncthreads();
  if (warp == 0 && lane == 0 && *abort_flag) drain_copies<S>(full, issued, p.err, 16);
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

// ------------------------------------------------------------- T <= 2: rows
// A warp takes R weight rows and all T tokens; lane l reads the 16-byte pieces l,
// l + 32, .. of a row, the tokens' pieces from L1/L2 beside it, four dp4a a piece
// and token, and the lanes' sums meet in one integer warp reduction.  Four rows a warp
// or one (launch_rows).
// One token, 129280 x 4096: 80 us (6.6 TB/s; the tensor-core tiles 83); 1280 x 5120:
// 2.9 us with the weight in the L2, 4.5 in turn over 39 MB of weights (the tiles 1.5 more, most
// of it getting started: barriers, TMEM, the first TMA).
template <int T, int R, typename TO>
__global__ void __launch_bounds__(256) gemm_i8_rows_kernel(const int8_t* x, size_t ldx, const int8_t* w, size_t ldw,
                                                           GemmI8Params p) {
  pdl_entry();
  const int lane = threadIdx.x & 31;
  const int n0 = (int)(blockIdx.x * 8 + (threadIdx.x >> 5)) * R;
  if (n0 >= p.N) return;
  const int8_t* wr[R];
#pragma unroll
  for (int r = 0; r < R; ++r) wr[r] = w + (size_t)min(n0 + r, p.N - 1) * ldw;   // past the end: the last row again
  int acc[R][T];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < T; ++t) acc[r][t] = 0;
  const int full = p.K / 512 * 512;
  constexpr int kUnroll = R == 1 ? 8 : 2;
#pragma unroll kUnroll
  for (int k = 16 * lane; k < full; k += 512) {
    int4 a[R], b[T];
#pragma unroll
    for (int r = 0; r < R; ++r) a[r] = ld_stream16(wr[r] + k);
#pragma unroll
    for (int t = 0; t < T; ++t) b[t] = *reinterpret_cast<const int4*>(x + t * ldx + k);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < T; ++t) acc[r][t] = dot16(a[r], b[t], acc[r][t]);
  }
  const int k = full + 16 * lane;   // the last pieces, the very last one byte by byte
  if (k < p.K) {
    int4 a[R], b[T];
#pragma unroll
    for (int r = 0; r < R; ++r) a[r] = ld_tail16(wr[r] + k, p.K - k);
#pragma unroll
    for (int t = 0; t < T; ++t) b[t] = ld_tail16(x + t * ldx + k, p.K - k);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < T; ++t) acc[r][t] = dot16(a[r], b[t], acc[r][t]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[r][t]);
      if (lane == r * T + t && n0 + r < p.N)
        static_cast<TO*>(p.out)[t * p.ldo + n0 + r] = out_of<TO>((float)sum * (p.ws[n0 + r] * p.xs[t]));
    }
}

// ----------------------------------------------------------- pairs: two SMs a tile
// The pair's tile is 256 channels x up to 256 tokens: each CTA loads its 128 channels
// and half the tokens (32 KB a k tile), the leader's tensor instruction reads both CTAs'
// shared memory, and each CTA's TMEM gets its 128 channels x all 256 tokens.  Per
// product that is a third less L2 -> SM traffic than a CTA of its own with a 128 x
// 256 tile moves, which is what bounds the latter.
// Measured in the kernel: 598 cycles a k tile (512 would be the tensor core's own; the
// reads of both operands and the TMA writes share the shared-memory path), 675 with
// fp32 stores beside it; a warp barrier in the issuing loop made the first 619.
// 8192^3: 380 us, 2.9 POP/s (tiles 430 us); 4096 x 5120 x 8192: 120 us (tiles 127 us,
// and 164 us before its epilogue).  Run for seconds the GPU is at its power cap, 1.3 to
// 1.5 GHz, and the same products take 10 to 25 % longer.
constexpr int kPairStages = 6;
constexpr int kPairA = 128 * 128, kPairB = 128 * 128, kPairStage = kPairA + kPairB;
constexpr int kPairSmem = 1024 + kPairStages * kPairStage + kEpiWarps * 128 * 4 + 256;

DSV4_DEV void umma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once the issued products are done.
DSV4_DEV void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// TMA load into this CTA, completion counted on a barrier of either CTA of the pair.
DSV4_DEV void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
DSV4_DEV void mbar_arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Unit u of a launch: whole tiles of p.width tokens first, then the tiles that would
// not fill a last wave of the GPU, in halves (p.n_whole and up; see launch_pairs).
struct PairUnit {
  int m0, n0, width;   // width tokens, a multiple of 32, from n0
};
DSV4_DEV PairUnit pair_unit(const GemmI8Params& p, int u) {
  const bool half = u >= p.n_whole;
  const int tile = half ? p.n_whole + ((u - p.n_whole) >> 1) : u;
  PairUnit r;
  r.m0 = tile / p.t_tiles * 256;
  r.n0 = tile % p.t_tiles * p.width;
  r.width = p.width;
  if (half) {
    r.width >>= 1;
    r.n0 += ((u - p.n_whole) & 1) * r.width;
  }
  return r;
}

template <typename TO>
__global__ void __launch_bounds__(kI8Threads, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_x64, GemmI8Params p) {
  constexpr int S = kPairStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S * kPairA;
  float* s_scale = reinterpret_cast<float*>(sB + S * kPairB);
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_scale + kEpiWarps * 128);
  uint64_t* full = bars;                    // leader's: both CTAs' four tiles of the stage
  uint64_t* empty = bars + S;               // each CTA's own, arrived at by the leader's commit
  uint64_t* acc_full = bars + 2 * S;        // each CTA's own, by the leader's commit
  uint64_t* acc_empty = bars + 2 * S + 2;   // leader's: the epilogue warps of both CTAs
  uint64_t* drain = bars + 2 * S + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  int issued = 0;   // k tiles this CTA's producer has asked for
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync_all();   // both CTAs' barriers are initialized, both have their TMEM
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full0 = dsmem_map(smem_u32(&full[0]), 0);   // the leader's barriers
      for (int u = pair; ok && u < p.n_units; u += n_pairs) {
        const PairUnit t = pair_unit(p, u);
        const int m0 = t.m0 + rank * 128, n0 = t.n0 + rank * (t.width >> 1);
        // up to 64 tokens a CTA come in a box of 64 rows; rows past the width are loaded but not used
        const bool narrow = t.width <= 128;
        const CUtensorMap* mx = narrow ? &map_x64 : &map_x;
        const uint32_t bytes = 2 * (kPairA + (narrow ? kPairB / 2 : kPairB));
        for (int kt = 0; kt < p.k_tiles; ++kt) {
          if (!(ok = mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.err, KID_GEMM, 21))) break;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          tma_load_2d_pair(sA + stage * kPairA, &map_w, full0 + 8 * stage, kt * 128, m0);
          tma_load_2d_pair(sB + stage * kPairB, mx, full0 + 8 * stage, kt * 128, n0);
          ++issued;
          if (++stage == S) stage = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      const uint64_t ad0 = sdesc_kmajor_sw128(smem_u32(sA)), bd0 = sdesc_kmajor_sw128(smem_u32(sB));
      bool ok = true;
      for (int u = pair; ok && u < p.n_units; u += n_pairs) {
        const uint32_t idesc = idesc_i8(256, (uint32_t)pair_unit(p, u).width);
        if (!(ok = mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.err, KID_GEMM, 22))) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * 256;
        bool ready = false;
        for (int kt = 0; kt < p.k_tiles; ++kt) {
          if (!ready && !(ok = mbar_wait(&full[stage], phase, abort_flag, p.err, KID_GEMM, 23))) break;
          tc_fence_after();
          const uint64_t ad = ad0 + (uint64_t)(stage * (kPairA >> 4)), bd = bd0 + (uint64_t)(stage * (kPairB >> 4));
          uint64_t* const done_bar = &empty[stage];
          if (++stage == S) stage = 0, phase ^= 1;
          // the next stage is asked for before this one's products, which hide the answer's latency
          ready = kt + 1 < p.k_tiles && mbar_try_wait(&full[stage], phase);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_i8_pair(d, ad + 2 * kk, bd + 2 * kk, idesc, (kt | kk) != 0 ? 1u : 0u);
          umma_commit_pair(done_bar);
        }
        if (!ok) break;
        umma_commit_pair(&acc_full[acc]);
        if (++acc == 2) acc = 0, acc_phase ^= 1;
      }
    }
  } else {
    const int q = warp & 3, grp = (warp - 2) >> 2;
    int acc = 0;
    uint32_t acc_phase = 0;
    TO* out = static_cast<TO*>(p.out);
    for (int u = pair; u < p.n_units; u += n_pairs) {
      const PairUnit t = pair_unit(p, u);
      const int m = t.m0 + rank * 128 + 32 * q + lane;
      const int nt = min(t.width, p.T - t.n0);
      const bool live = m < p.N;
      const float ws = live ? p.ws[m] : 0.f;
      float* xw = s_scale + (warp - 2) * 128;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 32 * (2 * i + grp) + lane;
        xw[32 * i + lane] = c < nt ? p.xs[t.n0 + c] : 0.f;
      }
      __syncwarp();
      if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.err, KID_GEMM, 24)) goto done;
      tc_fence_after();
      const uint32_t d = tmem + acc * 256 + ((uint32_t)(32 * q) << 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c0 = 32 * (2 * i + grp);
        if (c0 >= nt) break;
        uint32_t r[32];
        tmem_ld_32x32b_x32(d + c0, r);
        tmem_ld_wait();
        store_chunk<TO>(r, nt - c0, reinterpret_cast<const float4*>(xw + 32 * i), ws,
                        out + (size_t)(t.n0 + c0) * p.ldo + m, p.ldo, live);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(dsmem_map(smem_u32(&acc_empty[acc]), 0));
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
  }
done:
  __syncwarp();
  __syncthreads();   // every warp has finished or given up
  // the leader's barriers count both CTAs' copies; the other CTA waits for it below
  if (*abort_flag && warp == 0 && rank == 0 && lane == 0) drain_copies<S>(full, issued, p.err, 26);
  if (*abort_flag && warp == 1 && rank == 0) {   // no product may still use either CTA's TMEM
    if (lane == 0)
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(drain))
                   : "memory");
    __syncwarp();
    mbar_wait(drain, 0, nullptr, p.err, KID_GEMM, 25);
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();   // neither CTA's shared memory or TMEM is in use any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------------- host
namespace {

template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), int grid, int cluster, size_t smem, cudaStream_t st,
                           Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <int T, typename TO>
cudaError_t launch_rows(const int8_t* x, size_t ldx, const int8_t* w, size_t ldw, const GemmI8Params& p, int sms,
                        cudaStream_t st) {
  auto go = [&](auto kernel, int rows) {
    const unsigned grid = (unsigned)((p.N + 8 * rows - 1) / (8 * rows));
    return launch_pdl(kernel, grid, 256, 0, st, x, ldx, w, ldw, p);
  };
  // Four rows a warp share the tokens' pieces, one row has eight pieces of its own in flight
  // where K reaches 4096.  us with one and with four rows, one token: 5000 x 2048 4.2 and 5.1,
  // 9000 x 2048 6.6 and 5.9, 40000 x 2048 19.2 and 16.6; 19000 x 4096 14.5 and 18.7, 40000 x
  // 4096 27.7 and 30.6, 90000 x 4096 58.1 and 57.0; two tokens: 9000 x 2048 6.9 and 6.7, 40000 x
  // 4096 34.3 and 34.2, 65536 x 4096 55.1 and 47.7 (19000 rows of K below 4096 up to 13 % off).
  if (p.N >= (p.K < 4096 ? 56 : 440) * sms) return go(gemm_i8_rows_kernel<T, 4, TO>, 4);
  return go(gemm_i8_rows_kernel<T, 1, TO>, 1);
}

template <int BN, typename TO>
cudaError_t launch_tiles(const CUtensorMap& mw, const CUtensorMap& mx, const GemmI8Params& p, int sms,
                         cudaStream_t st) {
  using L = I8Smem<BN>;
  static std::atomic<uint64_t> configured{0};
  const cudaError_t e = smem_attr_once(gemm_i8_kernel<BN, TO>, L::kTotal, configured);
  if (e != cudaSuccess) return e;
  if (p.splits > 1)
    return launch_cluster(gemm_i8_kernel<BN, TO>, p.n_tiles * p.splits, p.splits, L::kTotal, st, mw, mx, p);
  return launch_pdl(gemm_i8_kernel<BN, TO>, p.n_tiles < sms ? p.n_tiles : sms, kI8Threads, L::kTotal, st, mw, mx, p);
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename TO>
cudaError_t launch_pairs(const int8_t* x, size_t ldx, const int8_t* w, size_t ldw, GemmI8Params p, int sms,
                         cudaStream_t st) {
  static std::atomic<uint64_t> configured{0};
  const cudaError_t e = smem_attr_once(gemm_i8_pair_kernel<TO>, kPairSmem, configured);
  if (e != cudaSuccess) return e;
  const int pairs = sms / 2;
  p.t_tiles = ceil_div(p.T, 256);
  p.width = ceil_div(ceil_div(p.T, p.t_tiles), 32) * 32;   // tiles of equal width
  p.n_tiles = ceil_div(p.N, 256) * p.t_tiles;
  // a last wave that under half the pairs would work in goes in tiles of half the width
  const int last = p.n_tiles % pairs;
  p.n_whole = p.width % 64 == 0 && 2 * last <= pairs ? p.n_tiles - last : p.n_tiles;
  p.n_units = p.n_whole + 2 * (p.n_tiles - p.n_whole);
  CUtensorMap mw, mx, mx64;
  if (!make_tma_rows_u8(&mw, w, p.N, p.K, ldw, 128) || !make_tma_rows_u8(&mx, x, p.T, p.K, ldx, 128) ||
      !make_tma_rows_u8(&mx64, x, p.T, p.K, ldx, 64))
    return cudaErrorInvalidValue;
  return launch_cluster(gemm_i8_pair_kernel<TO>, 2 * (p.n_units < pairs ? p.n_units : pairs), 2, kPairSmem, st, mw, mx,
                        mx64, p);
}

// Clusters of `splits` CTAs of the tiles kernel that can be resident at once (a
// cluster lives inside one GPC, so this is below SMs / splits).  Cached per device.
template <int BN, typename TO>
int cluster_room(int splits) {
  constexpr int kDevs = 64;
  static std::atomic<int> cache[kDevs][9] = {};
  int dev = 0;
  if (splits < 2 || splits > 8 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevs) return 0;
  int n = cache[dev][splits].load(std::memory_order_relaxed);
  if (n) return n - 1;
  using L = I8Smem<BN>;
  if (cudaFuncSetAttribute(gemm_i8_kernel<BN, TO>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) == cudaSuccess) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3(kI8Threads);
    cfg.dynamicSmemBytes = L::kTotal;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, gemm_i8_kernel<BN, TO>, &cfg) != cudaSuccess) n = 0;
  }
  (void)cudaGetLastError();
  cache[dev][splits].store(n + 1, std::memory_order_relaxed);
  return n;
}
template <typename TO>
int cluster_room_bn(int bn, int splits) {
  return bn == 32 ? cluster_room<32, TO>(splits) : bn == 64 ? cluster_room<64, TO>(splits)
       : bn == 128 ? cluster_room<128, TO>(splits) : cluster_room<256, TO>(splits);
}

// Widths and split of the tiles kernel, or the pairs kernel.  An SM takes in about
// 80 KB/us from L2, which bounds every tile shape but the pairs' (those run at the
// tensor core's 0.35 us a k tile), so a choice costs, in 128-byte rows loaded by the
// busiest SM (640 to a microsecond): the rows of its k tiles, 6 a token column for
// the epilogue, and with K split 768 for the cluster's barriers and 7 a column to
// park and add the partial tiles.  Against every width and split timed at 17 shapes
// from 3 x 2560 x 5120 to 2048 x 2048 x 4096 the choice was the fastest or within 4 %
// of it at 15 (64 x 2304 x 1280: 5.6 us, the widest tile with K in 4 parts 18.5), 13 %
// off at 1500 x 700 x 7000 and a third at 256 x 1280 x 5120 (14.9 us; 256-token tiles
// with K in 8 parts 11.1).
struct I8Plan {
  int path, bn, splits;
};
template <typename TO>
I8Plan plan_i8(const GemmI8Params& p, int sms) {
  I8Plan best{I8_TILES, 32, 1};
  long long least = -1;
  auto offer = [&](int path, int bn, int splits, long long cost) {
    if (least < 0 || cost < least) least = cost, best = I8Plan{path, bn, splits};
  };
  for (int bn = 32; bn <= 256 && (bn == 32 || bn / 2 < p.T); bn *= 2) {
    const long long tiles = (long long)ceil_div(p.N, 128) * ceil_div(p.T, bn);
    offer(I8_TILES, bn, 1, (tiles + sms - 1) / sms * p.k_tiles * (128 + bn) + 6 * bn);
    for (int s = 2; s <= 8 && tiles * s <= sms && 2 * s <= p.k_tiles; ++s)
      if (cluster_room_bn<TO>(bn, s) >= tiles)
        offer(I8_TILES, bn, s, (long long)ceil_div(p.k_tiles, s) * (128 + bn) + 13 * bn + 768);
  }
  if (p.T > 64) {
    const int t_tiles = ceil_div(p.T, 256), width = ceil_div(ceil_div(p.T, t_tiles), 32) * 32;
    const long long tiles = (long long)ceil_div(p.N, 256) * t_tiles;
    const long long pairs = sms / 2, last = tiles % pairs;
    const long long halves = width % 64 == 0 && 2 * last <= pairs ? last : 0;
    const long long waves2 = 2 * ((tiles - halves + pairs - 1) / pairs) + (halves ? 1 : 0);
    offer(I8_PAIRS, 0, 0, waves2 * p.k_tiles * (128 + width / 2) / 2 + 6 * width + 640);
  }
  return best;
}

template <typename TO>
cudaError_t run_i8(const int8_t* x, size_t ldx, const int8_t* w, size_t ldw, GemmI8Params p, I8Plan how, int sms,
                   cudaStream_t st) {
  p.k_tiles = ceil_div(p.K, 128);
  if (how.path == I8_AUTO) {
    how.path = p.T <= 2 ? I8_ROWS : I8_AUTO;
    if (how.path == I8_AUTO) how = plan_i8<TO>(p, sms);
  }
  if (how.path == I8_ROWS) {
    switch (p.T) {
      case 1: return launch_rows<1, TO>(x, ldx, w, ldw, p, sms, st);
      case 2: return launch_rows<2, TO>(x, ldx, w, ldw, p, sms, st);
      default: return cudaErrorInvalidValue;
    }
  }
  if (how.path == I8_PAIRS) return launch_pairs<TO>(x, ldx, w, ldw, p, sms, st);
  if (how.bn == 0) how.bn = p.T <= 32 ? 32 : p.T <= 64 ? 64 : p.T <= 128 ? 128 : 256;
  const int bn = how.bn;
  p.splits = std::max(1, std::min({8, how.splits, p.k_tiles}));
  p.t_tiles = ceil_div(p.T, bn);
  p.n_tiles = ceil_div(p.N, 128) * p.t_tiles;
  CUtensorMap mw, mx;
  if (!make_tma_rows_u8(&mw, w, p.N, p.K, ldw, 128) || !make_tma_rows_u8(&mx, x, p.T, p.K, ldx, bn))
    return cudaErrorInvalidValue;
  switch (bn) {
    case 32: return launch_tiles<32, TO>(mw, mx, p, sms, st);
    case 64: return launch_tiles<64, TO>(mw, mx, p, sms, st);
    case 128: return launch_tiles<128, TO>(mw, mx, p, sms, st);
    case 256: return launch_tiles<256, TO>(mw, mx, p, sms, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t gemm_i8(const int8_t* x, size_t ldx, const int8_t* w, size_t ldw, const GemmI8Params& p, int otype,
                    int path, int bn, int splits, int sms, cudaStream_t st) {
  if (p.T == 0 || p.N == 0) return cudaSuccess;
  const I8Plan how{path, bn, splits};
  switch (otype) {
    case F_BF16: return run_i8<__nv_bfloat16>(x, ldx, w, ldw, p, how, sms, st);
    case F_F16: return run_i8<__half>(x, ldx, w, ldw, p, how, sms, st);
    case F_F32: return run_i8<float>(x, ldx, w, ldw, p, how, sms, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace dsv4
