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
// the maximum come out of one pass and one reduction, and the row stays in registers
// between the two halves.
//
// Rows that hold an infinity or NaN come out as NaN: NaN scale, codes 0 (MX8:
// scale byte 0xFF, which the tensor core reads as NaN), and so do rows whose y passes
// fp32's range.  A row where only a partial result passes it is worked out again
// (far_row): squares are those of s scaled by 2^-96 (the eps is lost there: it is under
// 2^-60 of the mean), and where s w passes the range the root comes first, y = (s r) w.
#include "common.cuh"
#include "kernels.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace dsv4 {

constexpr int kNormThreads = 512, kNormWide = 768;

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

// Two fp32 operations in one instruction (sm_100); the kernel for aligned rows is close to
// the issue limit, so it works on pairs.
struct F2 {
  float x, y;
};
DSV4_DEV unsigned long long bits2(F2 a) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
DSV4_DEV F2 pair2(unsigned long long r) {
  F2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
  return a;
}
DSV4_DEV F2 add2(F2 a, F2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(r);
}
DSV4_DEV F2 mul2(F2 a, F2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(r);
}
DSV4_DEV F2 fma2(F2 a, F2 b, F2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(r);
}

// 8 consecutive elements as loaded, in 16-byte registers: taken apart only where they
// are used, so that a load stays in flight until then (as an array of 16-bit elements
// they were taken apart, and waited for, right behind the load).
template <typename T>
struct Vec8 {
  uint4 raw[sizeof(T) / 2];
};
template <typename T>
DSV4_DEV Vec8<T> ld_vec8(const T* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.raw[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
DSV4_DEV void floats_of(const Vec8<T>& r, F2 (&o)[4]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      o[2 * i] = {__uint_as_float(r.raw[i].x), __uint_as_float(r.raw[i].y)};
      o[2 * i + 1] = {__uint_as_float(r.raw[i].z), __uint_as_float(r.raw[i].w)};
    }
  } else {
    const uint32_t w[4] = {r.raw[0].x, r.raw[0].y, r.raw[0].z, r.raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        o[i] = {__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)};
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        o[i] = {f.x, f.y};
      }
    }
  }
}
DSV4_DEV uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
DSV4_DEV uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
DSV4_DEV void st_vec8(T* p, const F2 (&x)[4]) {
  uint4* d = reinterpret_cast<uint4*>(p);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      d[i] = make_uint4(__float_as_uint(x[2 * i].x), __float_as_uint(x[2 * i].y), __float_as_uint(x[2 * i + 1].x),
                        __float_as_uint(x[2 * i + 1].y));
  } else {
    d[0] = make_uint4(pack2(x[0].x, x[0].y, T()), pack2(x[1].x, x[1].y, T()), pack2(x[2].x, x[2].y, T()),
                      pack2(x[3].x, x[3].y, T()));
  }
}

// x + residual of one column after residual_out was written: its rounded value where that
// took the place of an input
template <typename TX>
DSV4_DEV float row_again(const NormQuantParams& p, int t, int c) {
  if (p.in_place) return to_f(static_cast<const TX*>(p.res_out)[(size_t)t * p.ldro + c]);
  const float a = to_f(static_cast<const TX*>(p.x)[(size_t)t * p.ldx + c]);
  return p.res ? a + to_f(static_cast<const TX*>(p.res)[(size_t)t * p.ldr + c]) : a;
}

// Codes of v * k, which is at most 127 (I8; a few roundings above it still round to 127)
// or 448 (the others; the conversion saturates).  I8: adding 1.5 * 2^23 leaves the
// integer nearest to the product, ties to even, in the low bits of the sum.
template <int FMT>
DSV4_DEV uint32_t codes4(F2 a, F2 b, float k) {
  a = mul2(a, {k, k});
  b = mul2(b, {k, k});
  if constexpr (FMT == Q8_I8) {
    a = add2(a, {12582912.f, 12582912.f});
    b = add2(b, {12582912.f, 12582912.f});
    const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a.x, a.y), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(b.x, b.y), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
}
// NaN wins, so that a NaN weight shows in the maximum as a NaN in the row does in the sum.
DSV4_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
DSV4_DEV float abs_max(float m, F2 a) { return max_nan(m, max_nan(fabsf(a.x), fabsf(a.y))); }
// Largest of the warp's values, none negative: their bits order as they do (NaN on top).
DSV4_DEV float warp_max_abs(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }

// What takes s w to its code: r * top / max|y|, with max|y| = r * max|s w| kept above
// 1e-30.  Where max|s w| is so small that this would overflow, *up (2^100) has to scale
// s w first.
DSV4_DEV float code_scale(float r, float mx, float top, float* up) {
  const float amax = fmaxf(r * mx, 1e-30f), inv = top / amax;
  *up = 1.f;
  if (mx < 1e-30f) {
    *up = 1.2676506002282294e30f;
    r *= 7.888609052210118e-31f;   // 2^-100
  }
  return r * inv;
}

// Sum and maximum over the threads of a row (at most MAXT), in a fixed order: the result
// does not depend on which warp arrives first.  One barrier; the caller alternates `red`.
// MXFP8 sums in 64 bits (see norm_once).
template <typename Sum>
struct RowRed {
  Sum sum[32];
  float mx[32];
};
DSV4_DEV double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <bool WARP, int MAXT, typename Sum>
DSV4_DEV void row_sum_max(Sum& sum, float& mx, RowRed<Sum>& red) {
  sum = warp_sum(sum);
  mx = warp_max_abs(mx);
  if constexpr (WARP) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (nw == 1) return;
  if (lane == 0) {
    red.sum[warp] = sum;
    red.mx[warp] = mx;
  }
  __syncthreads();
  sum = lane < nw ? red.sum[lane] : Sum(0);
#pragma unroll
  for (int o = MAXT / 32 > 16 ? 16 : 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  sum = __shfl_sync(0xffffffffu, sum, 0);
  mx = warp_max_abs(lane < nw ? red.mx[lane] : 0.f);
}

// 1 / sqrt(sum / D + eps); from a sum in 64 bits as the sum of two floats: rsqrtf and one
// Newton step whose residual is formed in 64 bits.
struct Root {
  float hi, lo;
};
DSV4_DEV Root inv_root(float sum, const NormQuantParams& p, float eps) {
  return {rsqrtf(fmaf(sum, (float)p.inv_d, eps)), 0.f};
}
DSV4_DEV Root inv_root(double sum, const NormQuantParams& p, float eps) {
  const double m = sum * p.inv_d + (double)eps;
  const float r0 = rsqrtf((float)m);
  const double e = fma(-m * (double)r0, (double)r0, 1.0);
  const float c = 0.5f * r0 * (float)e;
  Root r;
  r.hi = r0 + c;
  r.lo = c - (r.hi - r0);
  return r;
}
DSV4_DEV void add_squares(F2 a, double& x, double& y) {
  x = fma((double)a.x, (double)a.x, x);
  y = fma((double)a.y, (double)a.y, y);
}

// y = s * w * r rounded once, for MXFP8: its scales are powers of two, so y's own rounding
// errors are all that moves a code to its neighbour (one code in a million with three
// roundings in a row and the sum in 32 bits).  Rounded once, y can only mislead the code
// where it lies exactly between two codes, and so has its low 19 bits zero; there it is
// rounded to odd instead (to the neighbour with an odd last bit where it is not exact),
// and rounding that to a code is rounding the product itself.
DSV4_DEV F2 norm_once(F2 s, F2 w, Root r) {
  const F2 v = mul2(s, w), ev{fmaf(s.x, w.x, -v.x), fmaf(s.y, w.y, -v.y)};   // s w = v + ev
  return fma2(v, {r.hi, r.hi}, fma2(ev, {r.hi, r.hi}, mul2(v, {r.lo, r.lo})));
}
DSV4_DEV bool between_codes(F2 y) {
  return (__float_as_uint(y.x) & 0x7ffffu) == 0 || (__float_as_uint(y.y) & 0x7ffffu) == 0;
}
// a b + c to odd; c is small beside a b
DSV4_DEV float fma_odd(float a, float b, float c) {
  const float y0 = a * b, e0 = fmaf(a, b, -y0);      // a b = y0 + e0
  c += e0;
  const float y = y0 + c, rest = c - (y - y0);
  uint32_t bits = __float_as_uint(y);
  if (rest != 0.f && !(bits & 1u)) bits += (__float_as_uint(rest) ^ bits) >> 31 ? 0xffffffffu : 1u;
  return __uint_as_float(bits);
}
DSV4_DEV float norm_odd(float s, float w, Root r) {
  const float v = s * w, ev = fmaf(s, w, -v);
  return fma_odd(v, r.hi, fmaf(ev, r.hi, v * r.lo));
}
// y of a row that passes the range on the way: where s w does, the root comes first
template <int FMT>
DSV4_DEV float norm_far(float s, float w, Root r) {
  if (fabsf(s * w) < INFINITY) return FMT == Q8_MX8 ? norm_odd(s, w, r) : s * w * r.hi;
  const float v = s * r.hi;
  return FMT == Q8_MX8 ? fma_odd(v, w, fmaf(s, r.lo, fmaf(s, r.hi, -v)) * w) : v * w;
}

}  // namespace

constexpr float kDown = 1.2621774483536189e-29f;   // 2^-96

DSV4_DEV uint32_t mx_exp(float amax, bool bad) { return bad ? 255u : pow2_ceil_exp(fmaxf(amax, 1e-4f), 1.f / 448.f); }
// 1 / 2^(e - 127), exact: e is under 248 for finite rows
DSV4_DEV float mx_inv(uint32_t e, bool bad) { return bad ? 0.f : exp_to_f32(254 - e); }

// A row (with weights) whose sum of squares ss or whose y by way of s w is not finite, by
// all its threads: from memory again, an element at a time, since such rows are rare.
// Three passes: the sum of the squares scaled down, the largest y, the codes.
template <typename TX, typename TW, int FMT, bool WARP, int MAXT, typename Sum>
DSV4_DEV void far_row(const NormQuantParams& p, int t, int tid, int nt, Sum ss, RowRed<Sum>& red) {
  constexpr bool kMx = FMT == Q8_MX8;
  constexpr float top = FMT == Q8_I8 ? 127.f : 448.f;
  const TW* w = static_cast<const TW*>(p.w);
  const int D = p.D;
  // also: the row's residual_out is written, and `red` has been read
  auto sync = [] {
    if constexpr (WARP)
      __syncwarp();
    else
      __syncthreads();
  };
  sync();
  float mx = 0.f, down = 1.f;
  Root r;
  if ((float)ss < INFINITY) {
    r = inv_root(ss, p, p.eps);
  } else {
    down = kDown;
    ss = 0;
#pragma unroll 1
    for (int c = tid; c < D; c += nt) {
      const float s = row_again<TX>(p, t, c) * kDown;
      ss += (Sum)s * (Sum)s;
    }
    row_sum_max<WARP, MAXT>(ss, mx, red);
    sync();
    r = inv_root(ss, p, 0.f);
  }
  auto y_at = [&](int c) { return norm_far<FMT>(row_again<TX>(p, t, c) * down, to_f(w[c]), r); };
  mx = 0.f;
#pragma unroll 1
  for (int c = tid; c < D; c += nt) mx = max_nan(mx, fabsf(y_at(c)));
  Sum unused = ss;
  row_sum_max<WARP, MAXT>(unused, mx, red);
  const bool bad = !((float)ss < INFINITY) || !(mx < INFINITY);
  float k8 = 0.f, up = 1.f;
  if constexpr (!kMx) {
    if (tid == 0) p.scale[t] = bad ? __uint_as_float(0x7fffffffu) : fmaxf(mx, 1e-30f) / top;
    k8 = code_scale(1.f, mx, top, &up);
  }
  uint8_t* q = p.q + (size_t)t * p.ldq;
#pragma unroll 1
  for (int c = 4 * tid; c < D; c += 4 * nt) {   // MX8: D % 128 == 0, so a warp's lanes stay together
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = c + j < D ? y_at(c + j) : 0.f;
    if constexpr (kMx) {                        // 8 lanes hold a block of 32 columns
      float am = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
      const uint32_t e = mx_exp(am, bad);
      k8 = mx_inv(e, bad);
      if ((tid & 7) == 0) p.sf[sf_chunk_offset(t, c >> 5, D / 128)] = (uint8_t)e;
    }
    const uint32_t pk = bad ? 0u : codes4<FMT>({y[0] * up, y[1] * up}, {y[2] * up, y[3] * up}, k8);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < D) q[c + j] = (uint8_t)(pk >> (8 * j));
  }
}

// Rows of up to 8192 columns, all on 16-byte boundaries, 8 columns to a group.
//
// A row is a block's (WARP: a warp's, four rows to a block; no barrier then), and a
// block takes rows blockIdx.x, + gridDim.x, ..: it asks for the next row before it
// works on this one, and its weights stay in registers.  Thread i of the row owns the
// groups i, i + threads, .. (PER of them).
//
// Bound by its bytes once many rows are in flight: 16384 x 4096 bf16 with residual to
// int8, 470 MB: 118 us with a block per row (load, reduce and store in turn, 2 blocks
// an SM), 88 us with single fp32 operations (273 instructions for a lane's 8 columns:
// issue slots), 82 us so (5.7 TB/s).
template <typename TX, typename TW, int FMT, bool WARP, int PER, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) norm_quant_kernel(NormQuantParams p) {
  pdl_entry();
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, nt = WARP ? 32 : blockDim.x;
  const int row0 = WARP ? (int)(blockIdx.x * 4 + (threadIdx.x >> 5)) : (int)blockIdx.x;
  const int rows = WARP ? (int)gridDim.x * 4 : (int)gridDim.x;
  const int D = p.D;
  const bool has_res = p.res != nullptr, has_w = p.w != nullptr;
  constexpr bool kMx = FMT == Q8_MX8;   // keeps s in registers, the others s w
  using Sum = typename std::conditional<kMx, double, float>::type;
  __shared__ RowRed<Sum> red[2];
  auto col = [&](int k) { return 8 * (tid + k * nt); };

  Vec8<TW> wv[PER];
  Vec8<TX> nx[PER], nr[PER];
  auto fetch = [&](int t) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (col(k) >= D) continue;
      nx[k] = ld_vec8(static_cast<const TX*>(p.x) + (size_t)t * p.ldx + col(k));
      if (has_res) nr[k] = ld_vec8(static_cast<const TX*>(p.res) + (size_t)t * p.ldr + col(k));
    }
  };
  if (row0 < p.T) fetch(row0);
  if (has_w)
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (col(k) < D) wv[k] = ld_vec8(static_cast<const TW*>(p.w) + col(k));
  int turn = 0;
  for (int t = row0; t < p.T; t += rows, turn ^= 1) {
    TX* ro = p.res_out ? static_cast<TX*>(p.res_out) + (size_t)t * p.ldro : nullptr;
    F2 v[PER][4], sq{0.f, 0.f};
    double dx = 0.0, dy = 0.0;
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const bool live = col(k) < D;
      floats_of(nx[k], v[k]);
      if (has_res) {
        F2 a[4];
        floats_of(nr[k], a);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = add2(v[k][j], a[j]);
      }
      if (!live)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = {0.f, 0.f};
      if (ro && live) st_vec8(ro + col(k), v[k]);
    }
    if (t + rows < p.T) fetch(t + rows);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if constexpr (kMx) {
#pragma unroll
        for (int j = 0; j < 4; ++j) add_squares(v[k][j], dx, dy);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) sq = fma2(v[k][j], v[k][j], sq);
      }
      if (!kMx && has_w && col(k) < D) {
        F2 f[4];
        floats_of(wv[k], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = mul2(v[k][j], f[j]);
      }
      if (kMx && has_w && col(k) < D) {   // only to see whether every s w is finite
        F2 f[4];
        floats_of(wv[k], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = abs_max(mx, mul2(v[k][j], f[j]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = abs_max(mx, v[k][j]);
      }
    }
    Sum ss = kMx ? Sum(dx + dy) : Sum(sq.x + sq.y);
    row_sum_max<WARP, MAXT>(ss, mx, red[turn]);
    bool bad = false;
    Root r{1.f, 0.f};
    if (!has_w) {
      bad = ss != ss || !(mx < INFINITY);   // no norm: squares may overflow, infinities and NaN may not pass
    } else {
      r = inv_root(ss, p, p.eps);
      if (!((float)ss < INFINITY) || !(r.hi * mx < INFINITY)) {   // all threads of the row alike
        far_row<TX, TW, FMT, WARP, MAXT>(p, t, tid, nt, ss, red[turn]);
        continue;
      }
    }
    uint8_t* q = p.q + (size_t)t * p.ldq;
    constexpr float top = FMT == Q8_I8 ? 127.f : 448.f;
    float k8 = 0.f;
    if constexpr (!kMx) {
      if (tid == 0) p.scale[t] = bad ? __uint_as_float(0x7fffffffu) : fmaxf(r.hi * mx, 1e-30f) / top;
      float up;
      k8 = code_scale(r.hi, mx, top, &up);
      if (up != 1.f)   // the row's threads alike
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[k][j] = mul2(v[k][j], {up, up});
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int c = col(k);
      if constexpr (kMx) {   // 4 lanes hold a block of 32 columns
        if (has_w) {
          F2 f[4];
          floats_of(wv[k], f);   // past the row's end: not used, v is 0 there
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c < D) {
              const F2 y = norm_once(v[k][j], f[j], r);
              v[k][j] = between_codes(y) ? F2{norm_odd(v[k][j].x, f[j].x, r), norm_odd(v[k][j].y, f[j].y, r)} : y;
            }
        }
        float am = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) am = abs_max(am, v[k][j]);
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
        const uint32_t e = mx_exp(am, bad);
        k8 = mx_inv(e, bad);
        if (c < D && (tid & 3) == 0) p.sf[sf_chunk_offset(t, c >> 5, D / 128)] = (uint8_t)e;
      }
      if (c >= D) continue;
      const uint2 pk = make_uint2(codes4<FMT>(v[k][0], v[k][1], k8), codes4<FMT>(v[k][2], v[k][3], k8));
      *reinterpret_cast<uint2*>(q + c) = bad ? make_uint2(0, 0) : pk;
    }
  }
}

// Every other row: any alignment, any width up to 32768.  A block per row, which waits in
// shared memory (as s w in fp32; MX8: as s) between the two halves; off 16-byte
// boundaries element accesses, neighbours in a warp, eight in flight a thread (777 x 5003
// fp32: 9.8 us then, with four 11.0; in 16-byte pieces from the boundary before the row
// 13.2, since a lane's columns then lie apart in the weights and in shared memory).  WARP: a
// warp per row, 8 rows a block.
constexpr int kStagedWarps = 8;
template <typename TX, typename TW, int FMT, bool ALIGNED, bool WARP>
__global__ void __launch_bounds__(kNormThreads, 2) norm_quant_staged_kernel(NormQuantParams p) {
  pdl_entry();
  extern __shared__ __align__(16) float s_rows[];   // a row: D, rounded up to 4
  constexpr bool kMx = FMT == Q8_MX8;
  using Sum = typename std::conditional<kMx, double, float>::type;
  __shared__ RowRed<Sum> red;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, nt = WARP ? 32 : blockDim.x, D = p.D;
  const int t = WARP ? (int)blockIdx.x * kStagedWarps + (int)(threadIdx.x >> 5) : (int)blockIdx.x;
  if (WARP && t >= p.T) return;   // a warp alike; no barrier of the block follows
  float* s_row = s_rows + (WARP ? (size_t)(threadIdx.x >> 5) * ((D + 3) / 4 * 4) : 0);
  const TX* x = static_cast<const TX*>(p.x) + (size_t)t * p.ldx;
  const TX* res = p.res ? static_cast<const TX*>(p.res) + (size_t)t * p.ldr : nullptr;
  TX* ro = p.res_out ? static_cast<TX*>(p.res_out) + (size_t)t * p.ldro : nullptr;
  const TW* w = static_cast<const TW*>(p.w);
  Sum ss = 0;
  float mx = 0.f;
  if constexpr (ALIGNED) {   // wide rows on 16-byte boundaries: two groups of 8 columns in flight
    for (int g0 = tid; g0 < D / 8; g0 += 2 * nt) {
      Vec8<TX> a[2], b[2];
      Vec8<TW> wc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 8 * min(g0 + i * nt, D / 8 - 1);   // past the end: not used
        a[i] = ld_vec8(x + c);
        if (res) b[i] = ld_vec8(res + c);
        if (w) wc[i] = ld_vec8(w + c);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (g0 + i * nt >= D / 8) break;
        const int c = 8 * (g0 + i * nt);
        F2 v[4], f[4];
        floats_of(a[i], v);
        if (res) {
          floats_of(b[i], f);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = add2(v[j], f[j]);
        }
        if (ro) st_vec8(ro + c, v);
        if constexpr (kMx) {
          double dx = 0.0, dy = 0.0;
#pragma unroll
          for (int j = 0; j < 4; ++j) add_squares(v[j], dx, dy);
          ss += dx + dy;
        } else {
          F2 sq{0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; ++j) sq = fma2(v[j], v[j], sq);
          ss += sq.x + sq.y;
        }
        if (w && !kMx) {
          floats_of(wc[i], f);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], f[j]);
        }
        if (w && kMx) {
          floats_of(wc[i], f);
#pragma unroll
          for (int j = 0; j < 4; ++j) mx = abs_max(mx, mul2(v[j], f[j]));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) mx = abs_max(mx, v[j]);
        }
        *reinterpret_cast<float4*>(s_row + c) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        *reinterpret_cast<float4*>(s_row + c + 4) = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
      }
    }
  } else {
    constexpr int U = 8;
    for (int c0 = tid; c0 < D; c0 += U * nt) {
      TX a[U], b[U];
      TW wc[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = min(c0 + i * nt, D - 1);   // past the end: not used
        a[i] = x[c];
        if (res) b[i] = res[c];
        if (w) wc[i] = w[c];
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = c0 + i * nt;
        if (c >= D) break;
        float s = to_f(a[i]);
        if (res) s += to_f(b[i]);
        if (ro) ro[c] = from_f<TX>(s);
        ss += (Sum)s * (Sum)s;
        const float sw = w ? s * to_f(wc[i]) : s;
        mx = max_nan(mx, fabsf(sw));
        s_row[c] = kMx ? s : sw;
      }
    }
  }
  if (tid < (4 - D % 4) % 4) s_row[D + tid] = 0.f;
  row_sum_max<WARP, kNormThreads>(ss, mx, red);
  bool bad = false;
  Root r{1.f, 0.f};
  if (!w) {
    bad = ss != ss || !(mx < INFINITY);
  } else {
    r = inv_root(ss, p, p.eps);
    if (!((float)ss < INFINITY) || !(r.hi * mx < INFINITY)) {
      far_row<TX, TW, FMT, WARP, kNormThreads>(p, t, tid, nt, ss, red);
      return;
    }
  }
  if constexpr (WARP)   // the row is complete
    __syncwarp();
  else
    __syncthreads();   // (a block of one warp has met no barrier yet)
  uint8_t* q = p.q + (size_t)t * p.ldq;
  const bool words = reinterpret_cast<uintptr_t>(q) % 4 == 0;
  constexpr float top = FMT == Q8_I8 ? 127.f : 448.f;
  float k8 = 0.f, up = 1.f;
  if constexpr (!kMx) {
    if (tid == 0) p.scale[t] = bad ? __uint_as_float(0x7fffffffu) : fmaxf(r.hi * mx, 1e-30f) / top;
    k8 = code_scale(r.hi, mx, top, &up);
  }
  for (int c = 4 * tid; c < D; c += 4 * nt) {   // MX8: D % 128 == 0, so a warp's lanes stay together
    const float4 f = *reinterpret_cast<const float4*>(s_row + c);
    float y[4] = {f.x, f.y, f.z, f.w};
    if constexpr (kMx) {                        // 8 lanes hold a block of 32 columns
      if (w)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = norm_odd(y[j], to_f(w[c + j]), r);
      float am = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
      const uint32_t e = mx_exp(am, bad);
      k8 = mx_inv(e, bad);
      if ((tid & 7) == 0) p.sf[sf_chunk_offset(t, c >> 5, D / 128)] = (uint8_t)e;
    }
    const uint32_t pk = bad ? 0u : codes4<FMT>({y[0] * up, y[1] * up}, {y[2] * up, y[3] * up}, k8);
    if (words && c + 4 <= D) {
      *reinterpret_cast<uint32_t*>(q + c) = pk;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < D) q[c + j] = (uint8_t)(pk >> (8 * j));
    }
  }
}

// y[t, c] = code * scale, rounded to bf16.  A thread has 16 columns of a row next to each
// other (16-byte accesses), or 8 elements that are 256 apart, of a row or of all rows in
// order.
template <int FMT>
DSV4_DEV float dequant_scale(const float* scale, const uint8_t* sf, int t, int c, int k_tiles) {
  if constexpr (FMT == Q8_MX8) {
    const uint32_t e = sf[sf_chunk_offset(t, c >> 5, k_tiles)];
    return e == 255 ? __uint_as_float(0x7fffffffu) : e == 0 ? 5.8774717541114375e-39f : exp_to_f32(e);   // 0: 2^-127
  } else {
    return scale[t];
  }
}
template <int FMT>
DSV4_DEV float code_value(uint8_t b) {
  return FMT == Q8_I8 ? (float)(int8_t)b : e4m3_to_f32(b);
}

enum DequantWalk { DQ_VEC, DQ_ROW, DQ_FLAT };
template <int FMT, DequantWalk WALK>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t* q, size_t ldq, const float* scale, const uint8_t* sf,
                                                      int T, int D, __nv_bfloat16* y, size_t ldy, unsigned per_row) {
  pdl_entry();
  if constexpr (WALK == DQ_VEC) {
    const unsigned long long gid = (unsigned long long)blockIdx.x * 256 + threadIdx.x;   // per_row = D / 16
    const unsigned hi = (unsigned)(gid >> 32);
    const int t = hi ? (int)(gid / per_row) : (int)((unsigned)gid / per_row);
    if (t >= T) return;
    const int c = (int)(gid - (unsigned long long)t * per_row) * 16;
    const uint4 raw = *reinterpret_cast<const uint4*>(q + (size_t)t * ldq + c);
    const float s = dequant_scale<FMT>(scale, sf, t, c, D / 128);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    F2 v[2][4];
#pragma unroll
    for (int j = 0; j < 16; j += 2)
      v[j >> 3][(j & 7) >> 1] = {code_value<FMT>((uint8_t)(w[j >> 2] >> (8 * (j & 3)))) * s,
                                 code_value<FMT>((uint8_t)(w[j >> 2] >> (8 * (j & 3) + 8))) * s};
    st_vec8(y + (size_t)t * ldy + c, v[0]);
    st_vec8(y + (size_t)t * ldy + c + 8, v[1]);
  } else if constexpr (WALK == DQ_FLAT) {
    const unsigned long long n = (unsigned long long)T * D, i0 = (unsigned long long)blockIdx.x * 2048 + threadIdx.x;
    int t[8], c[8];
    uint8_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned long long i = i0 + 256 * j < n ? i0 + 256 * j : n - 1;   // past the end: not used
      t[j] = (int)(i >> 32 ? i / (unsigned)D : (unsigned)i / (unsigned)D);
      c[j] = (int)(i - (unsigned long long)t[j] * D);
      b[j] = q[(size_t)t[j] * ldq + c[j]];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + 256 * j < n)
        y[(size_t)t[j] * ldy + c[j]] =
            __float2bfloat16(code_value<FMT>(b[j]) * dequant_scale<FMT>(scale, sf, t[j], c[j], D / 128));
  } else {
    const int t = (int)(blockIdx.x / per_row), c0 = (int)(blockIdx.x % per_row) * 2048 + (int)threadIdx.x;
    const uint8_t* src = q + (size_t)t * ldq;
    uint8_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = src[min(c0 + 256 * j, D - 1)];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = c0 + 256 * j;
      if (c < D) y[(size_t)t * ldy + c] = __float2bfloat16(code_value<FMT>(b[j]) * dequant_scale<FMT>(scale, sf, t, c, D / 128));
    }
  }
}

// ------------------------------------------------------------------- host
template <typename TX, typename TW, int FMT>
static cudaError_t launch_norm(const NormQuantParams& p, bool vec, int sms, cudaStream_t st) {
  if (!vec || p.D > 2 * 8 * kNormThreads) {
    // 8 to 32 columns a thread, as many as it takes for the rows to be resident together (1024
    // threads an SM), and 256 threads, four blocks an SM, rather than two of up to 384 (fp32
    // 777 x 5003 9.9 us with 16, 8.2 so; 9598 x 6177 166 and 144; 4096 x 8200 59 and 44; bf16
    // 2000 x 12001 54.6 and 49.0; 777 x 1001 5.2 and 4.2).
    auto warps = [](int n) { return std::max(32, (n + 31) / 32 * 32); };
    const int fit = 1024 / std::min(32, (p.T + sms - 1) / sms) / 32 * 32;
    int nt = std::max(warps(p.D / 32), std::min(warps(p.D / 8), fit));
    if (p.T > 4 * sms && nt > 256 && nt <= 384) nt = 256;
    nt = std::min(kNormThreads, nt);
    const size_t row_bytes = (size_t)(p.D + 3) / 4 * 16;
    // very many narrow rows: a warp each (9135 x 37 fp16: 9.9 us with a block a row, 5.2 so;
    // 1200 x 1001 bf16: 5.4 and 6.6)
    if (!vec && p.D <= 1024 && p.T >= 16 * sms)
      return launch_pdl(norm_quant_staged_kernel<TX, TW, FMT, false, true>, (unsigned)((p.T + kStagedWarps - 1) / kStagedWarps),
                        32 * kStagedWarps, kStagedWarps * row_bytes, st, p);
    auto go = [&](auto kernel, std::atomic<uint64_t>& configured) {
      const cudaError_t e = smem_attr_once(kernel, 4 * kNormMaxD, configured);
      if (e != cudaSuccess) return e;
      return launch_pdl(kernel, (unsigned)p.T, (unsigned)nt, row_bytes, st, p);
    };
    static std::atomic<uint64_t> aligned{0}, any{0};
    return vec ? go(norm_quant_staged_kernel<TX, TW, FMT, true, false>, aligned)
               : go(norm_quant_staged_kernel<TX, TW, FMT, false, false>, any);
  }
  // as many blocks as are resident at once, each with its share of the rows
  auto go = [&](auto kernel, int nt, int rows_per_block, std::atomic<int>* room) {
    int per_sm = room[nt / 32].load(std::memory_order_relaxed);
    if (per_sm == 0) {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, nt, 0) != cudaSuccess || per_sm < 1) {
        (void)cudaGetLastError();
        per_sm = 1;
      }
      room[nt / 32].store(per_sm, std::memory_order_relaxed);
    }
    const int want = (p.T + rows_per_block - 1) / rows_per_block;
    const int turns = (want + per_sm * sms - 1) / (per_sm * sms);
    return launch_pdl(kernel, (unsigned)((want + turns - 1) / turns), (unsigned)nt, 0, st, p);
  };
#define DSV4_NQ(W, P, NT, ROWS, MAXT, MINB)                                    \
  do {                                                                         \
    static std::atomic<int> room[kNormWide / 32 + 1] = {};                     \
    return go(norm_quant_kernel<TX, TW, FMT, W, P, MAXT, MINB>, NT, ROWS, room); \
  } while (0)
  const int groups = p.D / 8;
  // many narrow rows: a warp each (4096 x 1280 bf16: 8.5 us with a block a row, 6.8 us so)
  constexpr int kWarpGroups = sizeof(TX) == 2 ? 192 : 64;   // what a lane's registers hold
  if (groups <= kWarpGroups && p.T >= 8 * sms) {
    if (groups <= 32) DSV4_NQ(true, 1, 128, 4, 128, 1);
    if (groups <= 64) DSV4_NQ(true, 2, 128, 4, 128, 1);
    if constexpr (sizeof(TX) == 2) {
      if (groups <= 128) DSV4_NQ(true, 4, 128, 4, 128, 1);
      DSV4_NQ(true, 6, 128, 4, 128, 1);
    }
  }
  // 16-bit rows: two blocks of 512 threads an SM (64 registers; 16384 x 4096 bf16 to MXFP8
  // 111 us, with one block an SM 139), and one group a thread up to 6144 columns (512 x 5120
  // to MXFP8 8.0 us, with two groups a thread 8.8; to int8 5.9 and 6.1)
  const int nt1 = (groups + 31) / 32 * 32;
  if constexpr (sizeof(TX) == 2) {
    if (groups <= kNormThreads) DSV4_NQ(false, 1, nt1, 1, kNormThreads, 2);
    if (groups <= kNormWide) DSV4_NQ(false, 1, nt1, 1, kNormWide, 1);
  } else {
    if (groups <= kNormThreads) DSV4_NQ(false, 1, nt1, 1, kNormThreads, 1);
  }
  DSV4_NQ(false, 2, ((groups + 1) / 2 + 31) / 32 * 32, 1, kNormThreads, 1);
#undef DSV4_NQ
}

template <typename TX, typename TW>
static cudaError_t norm_fmt(const NormQuantParams& p, int fmt, bool vec, int sms, cudaStream_t st) {
  switch (fmt) {
    case Q8_I8: return launch_norm<TX, TW, Q8_I8>(p, vec, sms, st);
    case Q8_E4M3: return launch_norm<TX, TW, Q8_E4M3>(p, vec, sms, st);
    case Q8_MX8: return launch_norm<TX, TW, Q8_MX8>(p, vec, sms, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t norm_quant(NormQuantParams p, int xtype, int wtype, int fmt, int sms, cudaStream_t st) {
  if (p.T == 0 || p.D == 0) return cudaSuccess;
  static_assert(4 * kNormMaxD <= 200 * 1024, "the widest row fits shared memory");
  if (p.D > kNormMaxD) return cudaErrorInvalidValue;
  p.inv_d = 1.0 / p.D;
  p.in_place = p.res_out && (p.res_out == p.x || p.res_out == p.res);
  const size_t ex = xtype == F_F32 ? 4 : 2, ew = wtype == F_F32 ? 4 : 2;
  auto al = [](const void* q, size_t ld_bytes) {
    return q == nullptr || (reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld_bytes % 16 == 0);
  };
  const bool vec = p.D % 8 == 0 && al(p.x, p.ldx * ex) && al(p.res, p.ldr * ex) && al(p.res_out, p.ldro * ex) &&
                   al(p.w, ew * 8) && reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && p.ldq % 8 == 0;
  if (xtype == F_BF16 && wtype == F_BF16) return norm_fmt<__nv_bfloat16, __nv_bfloat16>(p, fmt, vec, sms, st);
  if (xtype == F_BF16 && wtype == F_F32) return norm_fmt<__nv_bfloat16, float>(p, fmt, vec, sms, st);
  if (xtype == F_F16 && wtype == F_F16) return norm_fmt<__half, __half>(p, fmt, vec, sms, st);
  if (xtype == F_F16 && wtype == F_F32) return norm_fmt<__half, float>(p, fmt, vec, sms, st);
  if (xtype == F_F32 && wtype == F_F32) return norm_fmt<float, float>(p, fmt, vec, sms, st);
  return cudaErrorInvalidValue;
}

template <int FMT>
static cudaError_t launch_dequant(const uint8_t* q, size_t ldq, const float* scale, const uint8_t* sf, int T, int D,
                                  __nv_bfloat16* y, size_t ldy, cudaStream_t st) {
  const bool vec = D % 16 == 0 && ldq % 16 == 0 && ldy % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(y) % 16 == 0;
  // A block for 2048 columns of a row, or for 2048 elements of many narrow rows, where a
  // division each costs less than idle threads (4095 x 37 by rows 5.8 us, 4096 x 37 flat
  // 3.4; x 401: 6.1 and 5.4; x 509: 6.2 and 6.1)
  const bool flat = D <= 512 && T >= 4096;
  const unsigned per_row = vec ? (unsigned)(D / 16) : flat ? 0u : (unsigned)((D + 2047) / 2048);
  const unsigned long long blocks = vec    ? ((unsigned long long)T * per_row + 255) / 256
                                    : flat ? ((unsigned long long)T * D + 2047) / 2048
                                           : (unsigned long long)T * per_row;
  if (blocks >= (1ull << 31)) return cudaErrorInvalidValue;
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, (unsigned)blocks, 256, 0, st, q, ldq, scale, sf, T, D, y, ldy, per_row);
  };
  if (vec) return go(dequant_kernel<FMT, DQ_VEC>);
  return flat ? go(dequant_kernel<FMT, DQ_FLAT>) : go(dequant_kernel<FMT, DQ_ROW>);
}

cudaError_t dequant_rows(const uint8_t* q, size_t ldq, const float* scale, const uint8_t* sf, int T, int D, int fmt,
                         __nv_bfloat16* y, size_t ldy, cudaStream_t st) {
  if (T == 0 || D == 0) return cudaSuccess;
  switch (fmt) {
    case Q8_I8: return launch_dequant<Q8_I8>(q, ldq, scale, sf, T, D, y, ldy, st);
    case Q8_E4M3: return launch_dequant<Q8_E4M3>(q, ldq, scale, sf, T, D, y, ldy, st);
    case Q8_MX8: return launch_dequant<Q8_MX8>(q, ldq, scale, sf, T, D, y, ldy, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace dsv4
