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

// 16 bytes of logits
template <typename T>
struct alignas(16) Vec {
  T v[16 / sizeof(T)];
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

constexpr int kRulesThreads = 128;
constexpr int kRulesCols = 768;                   // columns of a warp
constexpr int kRulesWords = kRulesCols / 32 + 1;  // bit words that they touch
constexpr int kRulesChunk = kRulesCols * kRulesThreads / 32;

// Grid (chunks of a row, rows); a warp has 768 columns and works by itself.  Few columns
// are special (seen before, or biased): they are worked out one lane each, and the pass
// over all columns knows nothing of them.
//   1  lane i has word i of the seen bits and of the mask; the logits are asked for
//   2  the seen columns become a list; a lane per entry reads logit and count and
//      leaves the penalized value
//   3  a lane per bias entry adds it to that value, or to the logit and lists the column
//   4  lane i takes the 16-byte pieces i, i + 32, ..: the mask, store
//   5  a lane per listed column that the mask allows stores its value over it
// In place step 4 only touches the pieces that the mask takes something of.
//
// 512 x 129280 fp32 with every rule: 174 us with the counts read in step 4 (four
// dependent reads in a row a piece), 132 us with the steps shared by a block (its
// barriers), 117 us with the special values picked up by a bit in step 4 (750
// instructions a warp), 107 us so (547 MB: 5.1 TB/s).  A copy takes 78 us; the rest are
// the dependent reads slot -> bits -> counts.
//
// A piece starts on a 16-byte boundary whatever the row does, so a row's first and last
// pieces may be partial; rows of `in` and `out` that start at different offsets from
// such a boundary take plain accesses.
template <typename T, bool IN_PLACE>
__global__ void __launch_bounds__(kRulesThreads) logits_rules_kernel(LogitsRules p) {
  pdl_entry();
  constexpr int NV = 16 / sizeof(T);              // columns of a piece
  constexpr int P = kRulesCols / (32 * NV);       // pieces of a lane
  constexpr uint32_t kAll = (1u << NV) - 1, kFull = 0xffffffffu;
  __shared__ float s_val[kRulesThreads / 32][kRulesCols];       // values of the special columns
  __shared__ uint16_t s_list[kRulesThreads / 32][kRulesCols];   // the special columns
  __shared__ uint32_t s_bits[kRulesThreads / 32][32];           // which they are
  __shared__ uint32_t s_mask[kRulesThreads / 32][32];
  __shared__ int s_n[kRulesThreads / 32];
  const int s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* in = static_cast<const T*>(p.in) + (size_t)s * p.ld_in;
  T* out = static_cast<T*>(p.out) + (size_t)s * p.ld_out;
  const int shift = (int)(reinterpret_cast<uintptr_t>(in) / sizeof(T) % NV);
  const bool vec = IN_PLACE || reinterpret_cast<uintptr_t>(out) / sizeof(T) % NV == (uintptr_t)shift;
  const int c0 = ((int)blockIdx.x * (kRulesThreads / 32) + warp) * kRulesCols - shift;   // first column
  if (c0 >= p.V) return;
  const bool inner = vec && c0 >= 0 && c0 + kRulesCols <= p.V;   // every piece is whole
  // the row's rules; an index outside its table counts as none and is reported
  const int slot = p.slots ? p.slots[s] : -1;
  const int mrow = p.mask ? p.mask_row[s] : -1;
  int b0 = 0, b1 = 0;
  if (p.bias_off) {
    b0 = max(0, p.bias_off[s]);
    b1 = min(p.n_bias, p.bias_off[s + 1]);
  }
  Vec<T> l[P];
  if constexpr (!IN_PLACE) {
    if (inner) {
#pragma unroll
      for (int k = 0; k < P; ++k) l[k] = *reinterpret_cast<const Vec<T>*>(in + c0 + (lane + k * 32) * NV);
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int v = c0 + (lane + k * 32) * NV;
        if (vec && v >= 0 && v + NV <= p.V) {
          l[k] = *reinterpret_cast<const Vec<T>*>(in + v);
        } else {
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (v + j >= 0 && v + j < p.V) l[k].v[j] = in[v + j];
        }
      }
    }
  }
  bool pen = slot >= 0, masked = mrow >= 0;
  if (slot >= p.n_slots && p.slots) {
    if (lane == 0) report_error(p.err, ERR_BAD_ARG, KID_LOGITS, 1);
    pen = false;
  }
  if (mrow >= p.n_masks && p.mask) {
    if (lane == 0) report_error(p.err, ERR_BAD_ARG, KID_LOGITS, 2);
    masked = false;
  }
  const int wb = c0 >> 5, bit0 = c0 & 31;         // the first column's word (-1 where c0 < 0) and bit
  const int w = wb + lane;
  const bool have = lane < kRulesWords && w >= 0 && w < p.words;
  uint32_t sw = 0, mw = 0;                        // this lane's words: special, allowed
  int n = 0;                                      // listed columns
  if (masked && have) mw = (uint32_t)p.mask[(size_t)mrow * p.ld_mask + w];
  if (pen) {
    const float rho = p.repetition[s], freq = p.frequency[s], pres = p.presence[s];
    if (have) sw = (uint32_t)p.seen[(size_t)slot * p.words + w];
    // only the warp's own columns, and none past the vocabulary
    if (lane == 0) sw &= kFull << bit0;
    if (lane == kRulesCols / 32) sw &= (1u << bit0) - 1;
    if (w == p.V >> 5) sw &= (1u << (p.V & 31)) - 1;
    if (rho == 1.f && freq == 0.f && pres == 0.f) sw = 0;
    if (__any_sync(kFull, sw != 0)) {
      int at = __popc(sw);                        // this lane's place in the list
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int below = __shfl_up_sync(kFull, at, o);
        if (lane >= o) at += below;
      }
      n = __shfl_sync(kFull, at, 31);
      at -= __popc(sw);
      for (uint32_t x = sw; x; x &= x - 1) s_list[warp][at++] = (uint16_t)(32 * lane + __ffs(x) - 1 - bit0);
      __syncwarp();
      const int* counts = p.counts + (size_t)slot * p.V + c0;
      for (int i = lane; i < n; i += 32) {
        const int c = s_list[warp][i];
        const float z = lg_f(in[c0 + c]);
        const int cnt = counts[c];
        const float r = z > 0.f ? z / rho : z * rho;
        s_val[warp][c] = cnt > 0 ? r - (freq * (float)cnt + pres) : r;
      }
      __syncwarp();
    }
  }
  if (b0 < b1) {                                  // the warp's lanes alike
    // A long list: only the warp's part of it.  us with all of it and with the search, 512 x
    // 129280: 64 entries 78.9 and 82.7, 256 116 and 105, 1000 260 and 129; one row: 256 4.1 and
    // 4.3, 500 5.9 and 4.9; 64 x 32003 bf16: 256 6.0 and 6.1, 500 7.8 and 6.6.
    if (b1 - b0 > 256) {
      b0 = lower_bound(p.bias_id, b0, b1, c0);
      b1 = lower_bound(p.bias_id, b0, b1, c0 + kRulesCols);
    }
    s_bits[warp][lane] = sw;
    if (lane == 0) s_n[warp] = n;
    __syncwarp();
    for (int i = b0 + lane; i < b1; i += 32) {
      const int id = p.bias_id[i], c = id - c0;
      if ((unsigned)c >= (unsigned)kRulesCols || (unsigned)id >= (unsigned)p.V) continue;
      if (i > b0 && p.bias_id[i - 1] == id) continue;   // given more than once: the first entry adds the run in order
      float b = 0.f;
      for (int j = i; j < b1 && p.bias_id[j] == id; ++j) b += p.bias_val[j];
      const int at = bit0 + c;
      // the column's bit is asked for and set at once: an id out of its order, and so seen
      // as another run, adds to what is listed already
      const bool had = atomicOr(&s_bits[warp][at >> 5], 1u << (at & 31)) >> (at & 31) & 1;
      const float z = had ? s_val[warp][c] : lg_f(in[id]);
      s_val[warp][c] = b == -INFINITY ? b : z + b;
      if (!had) s_list[warp][atomicAdd(&s_n[warp], 1)] = (uint16_t)c;   // once a column: the list holds them all
    }
    __syncwarp();
    n = s_n[warp];
  }
  if constexpr (IN_PLACE) {
    if (masked) {
      T ninf;
      lg_set(ninf, -INFINITY);
      uint32_t ok[P];
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int c = (lane + k * 32) * NV, v = c0 + c;
        const int i = (bit0 + c) >> 5, sh = (bit0 + c) & 31;
        ok[k] = __funnelshift_r(__shfl_sync(kFull, mw, i), __shfl_sync(kFull, mw, i + 1), sh) & kAll;
        // nothing of a piece that stays or goes whole is read
        if (ok[k] != 0 && ok[k] != kAll && v >= 0 && v + NV <= p.V) l[k] = *reinterpret_cast<const Vec<T>*>(in + v);
      }
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int v = c0 + (lane + k * 32) * NV;
        if (ok[k] == kAll) continue;
        if (v >= 0 && v + NV <= p.V) {
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (!(ok[k] >> j & 1)) l[k].v[j] = ninf;
          *reinterpret_cast<Vec<T>*>(out + v) = l[k];
        } else {
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (!(ok[k] >> j & 1) && v + j >= 0 && v + j < p.V) out[v + j] = ninf;
        }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int c = (lane + k * 32) * NV, v = c0 + c;
      if (masked) {
        const int i = (bit0 + c) >> 5, sh = (bit0 + c) & 31;
        uint32_t ok = __shfl_sync(kFull, mw, i) >> sh;
        if (bit0 != 0) ok = __funnelshift_r(__shfl_sync(kFull, mw, i), __shfl_sync(kFull, mw, i + 1), sh);   // a piece may straddle words
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (!(ok >> j & 1)) lg_set(l[k].v[j], -INFINITY);
      }
      if (inner || (vec && v >= 0 && v + NV <= p.V)) {
        *reinterpret_cast<Vec<T>*>(out + v) = l[k];
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (v + j >= 0 && v + j < p.V) out[v + j] = l[k].v[j];
      }
    }
  }
  if (n > 0) {
    if (masked) s_mask[warp][lane] = mw;
    __syncwarp();   // also: these stores come after the lanes' stores to the same places
    for (int i = lane; i < n; i += 32) {
      const int c = s_list[warp][i], at = bit0 + c;
      if (!masked || (s_mask[warp][at >> 5] >> (at & 31) & 1)) lg_set(out[c0 + c], s_val[warp][c]);
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
  // a row's first piece may begin up to a piece before the row
  const int chunks = (p.V + 16 / (int)sizeof(T) - 1 + kRulesChunk - 1) / kRulesChunk;
  const dim3 grid((unsigned)chunks, (unsigned)p.S);
  if (p.in == p.out)
    launch_pdl(logits_rules_kernel<T, true>, grid, kRulesThreads, 0, st, p);
  else
    launch_pdl(logits_rules_kernel<T, false>, grid, kRulesThreads, 0, st, p);
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
