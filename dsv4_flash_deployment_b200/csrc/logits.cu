// Rules on logits between the output head and the sampler: penalties for repeated
// tokens, per-token biases and grammar masks, with the token history they read.
//
//   z = l / rho if l > 0 else l * rho      tokens of the prompt or the output
//   z -= frequency * count + presence      tokens of the output (count > 0)
//   z += bias                              bias -inf: banned whatever l is
//   z = -inf                               tokens the row's mask does not allow
//
// in fp32, rounded once to the logits' type.  What a mask or a -inf bias takes away
// is -inf even where l is NaN or infinite; a row whose mask leaves nothing is all
// -inf (its argmax is then token 0, as torch's).
//
// A row's history is a bit per vocabulary entry (prompt or output) and a count per
// entry (output).  Few of the 129K entries have their bit set, so the counts are
// read only there: per entry the kernel reads the logit, two bits, and writes the
// result.  In place nothing is read or written where no rule acts.
#include "common.cuh"
#include "kernels.h"

#include <cuda_fp16.h>

#include <algorithm>

namespace dsv4 {

namespace {
DSV4_DEV float lg_f(float v) { return v; }
DSV4_DEV float lg_f(__half v) { return __half2float(v); }
DSV4_DEV float lg_f(__nv_bfloat16 v) { return __bfloat162float(v); }
DSV4_DEV void lg_set(float& d, float v) { d = v; }
DSV4_DEV void lg_set(__half& d, float v) { d = __float2half_rn(v); }
DSV4_DEV void lg_set(__nv_bfloat16& d, float v) { d = __float2bfloat16(v); }

template <typename T>
struct alignas(4 * sizeof(T)) Quad {
  T v[4];
};

// first index in [lo, hi) whose id is >= v
DSV4_DEV int lower_bound(const int* ids, int lo, int hi, int v) {
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (ids[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}
}  // namespace

constexpr int kRulesThreads = 256;
constexpr int kRulesMaxChunk = 4096;   // columns of one CTA (its bias column sums take 16 KB)

// Grid (chunks of a row, rows).  Thread i owns 4 consecutive columns (one 16- or
// 8-byte access), 4 * blockDim apart from its next ones.  VEC false: rows that do
// not start on such a boundary, plain accesses.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRulesThreads) logits_rules_kernel(LogitsRules p, int chunk, bool in_place) {
  pdl_entry();
  __shared__ float s_bias[kRulesMaxChunk];
  const int s = blockIdx.y, tid = threadIdx.x;
  const int v0 = blockIdx.x * chunk, v1 = min(p.V, v0 + chunk);
  const T* in = static_cast<const T*>(p.in) + (size_t)s * p.ld_in;
  T* out = static_cast<T*>(p.out) + (size_t)s * p.ld_out;
  // the row's rules; an index outside its table counts as none and is reported
  const int* seen = nullptr;
  const int* counts = nullptr;
  float rho = 1.f, freq = 0.f, pres = 0.f;
  if (p.slots) {
    const int slot = p.slots[s];
    if (slot >= p.n_slots) {
      if (tid == 0) report_error(p.err, ERR_BAD_ARG, KID_LOGITS, 1);
    } else if (slot >= 0) {
      rho = p.repetition[s];
      freq = p.frequency[s];
      pres = p.presence[s];
      if (rho != 1.f || freq != 0.f || pres != 0.f) {
        seen = p.seen + (size_t)slot * p.words;
        counts = p.counts + (size_t)slot * p.V;
      }
    }
  }
  const int* mask = nullptr;
  if (p.mask) {
    const int m = p.mask_row[s];
    if (m >= p.n_masks) {
      if (tid == 0) report_error(p.err, ERR_BAD_ARG, KID_LOGITS, 2);
    } else if (m >= 0) {
      mask = p.mask + (size_t)m * p.ld_mask;
    }
  }
  bool biased = false;
  if (p.bias_off) {
    const int b0 = max(0, p.bias_off[s]), b1 = min(p.n_bias, p.bias_off[s + 1]);
    const int lo = lower_bound(p.bias_id, b0, b1, v0), hi = lower_bound(p.bias_id, lo, max(lo, b1), v1);
    biased = lo < hi;
    if (biased) {   // the whole CTA alike
      for (int i = tid; i < v1 - v0; i += kRulesThreads) s_bias[i] = 0.f;
      __syncthreads();
      // an id given more than once: its first entry adds the run in order
      for (int i = lo + tid; i < hi; i += kRulesThreads) {
        const int id = p.bias_id[i];
        if (id < v0 || id >= v1 || (i > lo && p.bias_id[i - 1] == id)) continue;
        float b = 0.f;
        for (int j = i; j < hi && p.bias_id[j] == id; ++j) b += p.bias_val[j];
        s_bias[id - v0] = b;
      }
      __syncthreads();
    }
  }
  for (int v = v0 + 4 * tid; v < v1; v += 4 * kRulesThreads) {
    const int n = min(4, v1 - v);
    const uint32_t all = (1u << n) - 1;
    const uint32_t sb = seen ? ((uint32_t)seen[v >> 5] >> (v & 31)) & all : 0u;
    const uint32_t mb = mask ? ((uint32_t)mask[v >> 5] >> (v & 31)) & all : all;
    if (in_place && sb == 0 && mb == all && !biased) continue;
    float l[4];
    if (VEC && n == 4) {
      const Quad<T> q = *reinterpret_cast<const Quad<T>*>(in + v);
#pragma unroll
      for (int j = 0; j < 4; ++j) l[j] = lg_f(q.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) l[j] = j < n ? lg_f(in[v + j]) : 0.f;
    }
    if (sb) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!(sb >> j & 1)) continue;
        l[j] = l[j] > 0.f ? l[j] / rho : l[j] * rho;
        const int c = counts[v + j];
        if (c > 0) l[j] -= freq * (float)c + pres;
      }
    }
    if (biased) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float b = j < n ? s_bias[v - v0 + j] : 0.f;
        l[j] = b == -INFINITY ? b : l[j] + b;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(mb >> j & 1)) l[j] = -INFINITY;
    if (VEC && n == 4) {
      Quad<T> q;
#pragma unroll
      for (int j = 0; j < 4; ++j) lg_set(q.v[j], l[j]);
      *reinterpret_cast<Quad<T>*>(out + v) = q;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) lg_set(out[v + j], l[j]);
    }
  }
}

__global__ void history_add_kernel(const int* ids, const int* slots, const int* generated, int n, int* seen, int* counts, int n_slots,
                                   int V, int words, uint32_t* err) {
  pdl_entry();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int g = generated[i], slot = slots[i], id = ids[i];
  if (g < 0 || slot < 0) return;
  if (slot >= n_slots || id < 0 || id >= V) {
    report_error(err, ERR_BAD_ARG, KID_LOGITS, 3);
    return;
  }
  // integer updates: the result does not depend on their order
  atomicOr(seen + (size_t)slot * words + (id >> 5), 1 << (id & 31));
  if (g > 0) atomicAdd(counts + (size_t)slot * V + id, 1);
}

// ------------------------------------------------------------------- host
template <typename T>
static cudaError_t rules_type(const LogitsRules& p, cudaStream_t st) {
  const size_t a = 4 * sizeof(T);
  const bool vec = reinterpret_cast<uintptr_t>(p.in) % a == 0 && reinterpret_cast<uintptr_t>(p.out) % a == 0 &&
                   p.ld_in % 4 == 0 && p.ld_out % 4 == 0;
  const int chunk = kRulesMaxChunk;
  const dim3 grid((unsigned)((p.V + chunk - 1) / chunk), (unsigned)p.S);
  if (vec)
    launch_pdl(logits_rules_kernel<T, true>, grid, kRulesThreads, 0, st, p, chunk, p.in == p.out);
  else
    launch_pdl(logits_rules_kernel<T, false>, grid, kRulesThreads, 0, st, p, chunk, p.in == p.out);
  return cudaGetLastError();
}

cudaError_t logits_rules(const LogitsRules& p, int type, cudaStream_t st) {
  if (p.S == 0 || p.V == 0) return cudaSuccess;
  switch (type) {
    case F_BF16: return rules_type<__nv_bfloat16>(p, st);
    case F_F16: return rules_type<__half>(p, st);
    case F_F32: return rules_type<float>(p, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t history_add(const int* ids, const int* slots, const int* generated, int n, int* seen, int* counts,
                        int n_slots, int V, int words, uint32_t* err, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  launch_pdl(history_add_kernel, (unsigned)((n + 255) / 256), 256, 0, st, ids, slots, generated, n, seen, counts,
             n_slots, V, words, err);
  return cudaGetLastError();
}

}  // namespace dsv4
