// RMS norm with the residual's addition and an 8-bit output, per-row 8-bit
// quantization without the norm, and the way back to bf16.
//
//   s = x + residual                          (fp32; residual_out = s rounded once)
//   y = s * rsqrt(mean(s^2) + eps) * w        (fp32, never rounded before the codes)
//   I8:   scale = max|y| / 127,  q = rne(y / scale)            one scale per row
//   E4M3: scale = max|y| / 448,  q = e4m3(y / scale)           one scale per row
//   MX8:  scale = 2^ceil(log2(max(max|y|, 1e-4) / 448)) per 32 columns, in the
//         GEMM's 512-byte chunks (common.cuh), the operand form of gemm_mx
//
// With r = rsqrt(..) > 0 the same for the whole row, max|y| = r * max|s w|: the
// scale of the per-row formats is r * max|s w| / 127.  So the sum of squares and
// the maximum come out of one pass and one block reduction, and the row stays in registers (as s w) between the two halves.
//
// Rows that hold an infinity or NaN come out as NaN: NaN scale, codes 0 (MX8:
// scale byte 0xFF, which the tensor core reads as NaN).  Finite rows whose squares
// pass fp32's range are scaled by 2^-96 and summed again (the eps is lost there:
// it is under 2^-60 of the mean).
#include "common.cuh"
#include "kernels.h"

#include <cuda_fp16.h>

#include <algorithm>

namespace dsv4 {

namespace {

DSV4_DEV float to_f(float v) { return v; }
DSV4_DEV float to_f(__half v) { return __half2float(v); }
DSV4_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
DSV4_DEV T from_f(float v);
template <>
DSV4_DEV float from_f<float>(float v) { return v; }
template <>
DSV4_DEV __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
DSV4_DEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// 8 consecutive elements with 16-byte accesses
template <typename T>
struct alignas(16) Vec8 {
  T v[8];
};
template <typename T>
DSV4_DEV void ld_vec8(const T* p, float (&o)[8]) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(r) / 16; ++i)
    reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = to_f(r.v[i]);
}
template <typename T>
DSV4_DEV void st_vec8(T* p, const float (&x)[8]) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = from_f<T>(x[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(r) / 16; ++i)
    reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&r)[i];
}

DSV4_DEV uint8_t code_of(float y, int fmt) {
  if (fmt == Q8_I8) return (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
  return f32_to_e4m3(fminf(fmaxf(y, -448.f), 448.f));
}

// Sum and maximum over the block, in a fixed order: the result does not depend on
// which warp arrives first.
DSV4_DEV void block_sum_max(float& sum, float& mx, float (*red)[32]) {
  sum = warp_sum(sum);
  mx = warp_max(mx);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (nw == 1) return;
  if (lane == 0) {
    red[0][warp] = sum;
    red[1][warp] = mx;
  }
  __syncthreads();
  sum = warp_sum(lane < nw ? red[0][lane] : 0.f);
  mx = warp_max(lane < nw ? red[1][lane] : 0.f);
}

}  // namespace

constexpr int kNormThreads = 512;

// One CTA per row.  VEC: thread i owns the 8-column groups i, i + blockDim, ..
// (16-byte accesses); otherwise element j of a thread is column (k * 8 + j) *
// blockDim + i, so a warp still touches consecutive columns (and 32 columns of an
// MX8 block are one warp's).  PER groups of 8 per thread.
template <typename TX, typename TW, int FMT, bool VEC, int PER>
__global__ void __launch_bounds__(kNormThreads) norm_quant_kernel(NormQuantParams p) {
  pdl_entry();
  const int tid = threadIdx.x, nt = blockDim.x;
  const size_t t = blockIdx.x;
  const int D = p.D;
  const TX* x = static_cast<const TX*>(p.x) + t * p.ldx;
  const TX* res = p.res ? static_cast<const TX*>(p.res) + t * p.ldr : nullptr;
  TX* ro = p.res_out ? static_cast<TX*>(p.res_out) + t * p.ldro : nullptr;
  const TW* w = static_cast<const TW*>(p.w);
  auto col = [&](int k, int j) { return VEC ? 8 * (tid + k * nt) + j : (k * 8 + j) * nt + tid; };

  float v[PER][8];
  float ss = 0.f, mx = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    float wv[8];
    if constexpr (VEC) {
      const int c = col(k, 0);
      if (c < D) {
        ld_vec8(x + c, v[k]);
        if (res) {
          float r[8];
          ld_vec8(res + c, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] += r[j];
          if (ro) st_vec8(ro + c, v[k]);
        }
        if (w) ld_vec8(w + c, wv);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = 0.f, wv[j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = col(k, j);
        v[k][j] = 0.f;
        wv[j] = 0.f;
        if (c < D) {
          v[k][j] = to_f(x[c]);
          if (res) {
            v[k][j] += to_f(res[c]);
            if (ro) ro[c] = from_f<TX>(v[k][j]);
          }
          if (w) wv[j] = to_f(w[c]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss += v[k][j] * v[k][j];
      if (w) v[k][j] *= wv[j];
      mx = fmaxf(mx, fabsf(v[k][j]));
    }
  }
  __shared__ float red[2][2][32];
  block_sum_max(ss, mx, red[0]);
  bool bad = false;
  float r = 1.f;
  if (w) {
    if (!(ss < INFINITY) || !(mx < INFINITY)) {   // the whole block alike: the row again, scaled by 2^-96
      constexpr float kDown = 1.2621774483536189e-29f;   // 2^-96
      ss = 0.f;
      mx = 0.f;
#pragma unroll
      for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = col(k, j);
          float s = 0.f, wc = 0.f;
          if (c < D) {
            // residual_out may be the residual itself and then holds the rounded sum:
            // the ratio of two such rows differs by that rounding only
            s = ro ? to_f(ro[c]) : to_f(x[c]) + (res ? to_f(res[c]) : 0.f);
            wc = to_f(w[c]);
          }
          s *= kDown;
          ss += s * s;
          v[k][j] = s * wc;
          mx = fmaxf(mx, fabsf(v[k][j]));
        }
      block_sum_max(ss, mx, red[1]);
      bad = !(ss < INFINITY) || !(mx < INFINITY);
      r = rsqrtf(ss / (float)D);
    } else {
      r = rsqrtf(ss / (float)D + p.eps);
    }
  } else {
    bad = ss != ss || !(mx < INFINITY);   // no norm: squares may overflow, infinities and NaN may not pass
  }
  const float nan = __uint_as_float(0x7fffffffu);
  uint8_t* q = p.q + t * p.ldq;
  if constexpr (FMT == Q8_MX8) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      float am[8];
      if constexpr (VEC) {   // 4 lanes hold a block of 32 columns
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] *= r, a = fmaxf(a, fabsf(v[k][j]));
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
        const int c = col(k, 0);
        if (c < D) {
          const uint32_t e = bad ? 255u : pow2_ceil_exp(fmaxf(a, 1e-4f), 1.f / 448.f);
          const float s = exp_to_f32(e);
          uint32_t pk[2] = {0, 0};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            pk[j >> 2] |= (uint32_t)(bad ? 0 : code_of(v[k][j] / s, FMT)) << (8 * (j & 3));
          *reinterpret_cast<uint2*>(q + c) = make_uint2(pk[0], pk[1]);
          if ((tid & 3) == 0) p.sf[sf_chunk_offset((int)t, c >> 5, D / 128)] = (uint8_t)e;
        }
      } else {               // a warp's 32 lanes hold a block
#pragma unroll
        for (int j = 0; j < 8; ++j) am[j] = warp_max(fabsf(v[k][j] * r));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = col(k, j);
          if (c >= D) continue;
          const uint32_t e = bad ? 255u : pow2_ceil_exp(fmaxf(am[j], 1e-4f), 1.f / 448.f);
          q[c] = bad ? 0 : code_of(v[k][j] * r / exp_to_f32(e), FMT);
          if ((tid & 31) == 0) p.sf[sf_chunk_offset((int)t, c >> 5, D / 128)] = (uint8_t)e;
        }
      }
    }
  } else {
    const float top = FMT == Q8_I8 ? 127.f : 448.f;
    const float amax = fmaxf(r * mx, 1e-30f);
    if (tid == 0) p.scale[t] = bad ? nan : amax / top;
    const float inv = top / amax;   // at most 4.5e32: y is scaled by r first, so no product overflows
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if constexpr (VEC) {
        const int c = col(k, 0);
        if (c < D) {
          uint32_t pk[2] = {0, 0};
#pragma unroll
          for (int j = 0; j < 8; ++j) pk[j >> 2] |= (uint32_t)(bad ? 0 : code_of(v[k][j] * r * inv, FMT)) << (8 * (j & 3));
          *reinterpret_cast<uint2*>(q + c) = make_uint2(pk[0], pk[1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = col(k, j);
          if (c < D) q[c] = bad ? 0 : code_of(v[k][j] * r * inv, FMT);
        }
      }
    }
  }
}

// y[t, c] = code * scale, rounded to bf16 (8 columns a thread, plain accesses).
template <int FMT>
__global__ void dequant_kernel(const uint8_t* q, int ldq, const float* scale, const uint8_t* sf, int T, int D,
                               __nv_bfloat16* y, int ldy,
                               int vec) {
  pdl_entry();
  const int groups = (D + 7) / 8;
  const long long gid = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (gid >= (long long)T * groups) return;
  const int t = (int)(gid / groups), c0 = (int)(gid % groups) * 8;
  uint8_t b[8];
  const uint8_t* src = q + (size_t)t * ldq + c0;
  const int n = min(8, D - c0);
  if (vec) {
    *reinterpret_cast<uint2*>(b) = *reinterpret_cast<const uint2*>(src);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = j < n ? src[j] : 0;
  }
  float s;
  if constexpr (FMT == Q8_MX8) {
    const uint32_t e = sf[sf_chunk_offset(t, c0 >> 5, D / 128)];
    s = e == 255 ? __uint_as_float(0x7fffffffu) : e == 0 ? 5.8774717541114375e-39f : exp_to_f32(e);   // e 0: 2^-127
  } else {
    s = scale[t];
  }
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (FMT == Q8_I8 ? (float)(int8_t)b[j] : e4m3_to_f32(b[j])) * s;
  __nv_bfloat16* dst = y + (size_t)t * ldy + c0;
  if (vec) {
    st_vec8(dst, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) dst[j] = __float2bfloat16(v[j]);
  }
}

// ------------------------------------------------------------------- host
template <typename TX, typename TW, int FMT>
static cudaError_t launch_norm(const NormQuantParams& p, bool vec, cudaStream_t st) {
  // one group of 8 columns per thread up to 512 threads, then 2, 4 and 8
  const int groups = (p.D + 7) / 8;
  const int per = groups <= kNormThreads ? 1 : groups <= 2 * kNormThreads ? 2 : groups <= 4 * kNormThreads ? 4 : 8;
  const int nt = std::max(32, ((groups + per - 1) / per + 31) / 32 * 32);
#define DSV4_NQ(V, P) launch_pdl(norm_quant_kernel<TX, TW, FMT, V, P>, (unsigned)p.T, (unsigned)nt, 0, st, p)
  if (vec)
    per == 1 ? DSV4_NQ(true, 1) : per == 2 ? DSV4_NQ(true, 2) : per == 4 ? DSV4_NQ(true, 4) : DSV4_NQ(true, 8);
  else
    per == 1 ? DSV4_NQ(false, 1) : per == 2 ? DSV4_NQ(false, 2) : per == 4 ? DSV4_NQ(false, 4) : DSV4_NQ(false, 8);
#undef DSV4_NQ
  return cudaGetLastError();
}

template <typename TX, typename TW>
static cudaError_t norm_fmt(const NormQuantParams& p, int fmt, bool vec, cudaStream_t st) {
  switch (fmt) {
    case Q8_I8: return launch_norm<TX, TW, Q8_I8>(p, vec, st);
    case Q8_E4M3: return launch_norm<TX, TW, Q8_E4M3>(p, vec, st);
    case Q8_MX8: return launch_norm<TX, TW, Q8_MX8>(p, vec, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t norm_quant(const NormQuantParams& p, int xtype, int wtype, int fmt, cudaStream_t st) {
  if (p.T == 0 || p.D == 0) return cudaSuccess;
  static_assert(kNormMaxD == 8 * 8 * kNormThreads, "the widest row fills 8 groups a thread");
  if (p.D > kNormMaxD) return cudaErrorInvalidValue;
  const size_t ex = xtype == F_F32 ? 4 : 2, ew = wtype == F_F32 ? 4 : 2;
  auto al = [](const void* q, size_t ld_bytes) {
    return q == nullptr || (reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld_bytes % 16 == 0);
  };
  const bool vec = p.D % 8 == 0 && al(p.x, p.ldx * ex) && al(p.res, p.ldr * ex) && al(p.res_out, p.ldro * ex) &&
                   al(p.w, ew * 8) && reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && p.ldq % 8 == 0;
  if (xtype == F_BF16 && wtype == F_BF16) return norm_fmt<__nv_bfloat16, __nv_bfloat16>(p, fmt, vec, st);
  if (xtype == F_BF16 && wtype == F_F32) return norm_fmt<__nv_bfloat16, float>(p, fmt, vec, st);
  if (xtype == F_F16 && wtype == F_F16) return norm_fmt<__half, __half>(p, fmt, vec, st);
  if (xtype == F_F16 && wtype == F_F32) return norm_fmt<__half, float>(p, fmt, vec, st);
  if (xtype == F_F32 && wtype == F_F32) return norm_fmt<float, float>(p, fmt, vec, st);
  return cudaErrorInvalidValue;
}

cudaError_t dequant_rows(const uint8_t* q, int ldq, const float* scale, const uint8_t* sf, int T, int D, int fmt,
                         __nv_bfloat16* y, int ldy, cudaStream_t st) {
  const long long n = (long long)T * ((D + 7) / 8);
  if (n == 0) return cudaSuccess;
  const int vec = D % 8 == 0 && ldq % 8 == 0 && ldy % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(y) % 16 == 0;
  const unsigned grid = (unsigned)((n + 255) / 256);
  switch (fmt) {
    case Q8_I8: launch_pdl(dequant_kernel<Q8_I8>, grid, 256, 0, st, q, ldq, scale, sf, T, D, y, ldy, vec); break;
    case Q8_E4M3: launch_pdl(dequant_kernel<Q8_E4M3>, grid, 256, 0, st, q, ldq, scale, sf, T, D, y, ldy, vec); break;
    case Q8_MX8: launch_pdl(dequant_kernel<Q8_MX8>, grid, 256, 0, st, q, ldq, scale, sf, T, D, y, ldy, vec); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace dsv4
