// Processing of a step's logits before sampling (sm_100a): penalties for repeated tokens, a bias
// and a grammar mask, in one pass. For row (b, s) and token v, with n the times v occurs in the
// first hist_len[b] entries of history[b]:
//   x = logits[b, s, v]
//   if n > 0:  x = (x > 0 ? x / r_b : x * r_b) - (f_b * n + p_b)
//   x += bias[v] (or bias[b, v]);  x = -inf where the mask's bit v is 0
// in fp32, each product, quotient and sum rounded to fp32, the result rounded once to the
// logits' type. The S rows of a sequence (a block of a denoising step) share its history.
//
// DRAM-bound: every logit is read and written once. A CTA takes a slice of the vocabulary for some
// rows of one sequence: it counts the history's tokens of its slice in shared memory (integer
// atomics: the order does not matter) with a bitmap of the tokens seen, stages the bias of the
// slice, and streams the rows through. A thread takes 8 consecutive logits with 16-byte
// accesses; rows of an odd vocabulary start at any alignment, so its chunks begin `a` logits
// before the multiples of 8, a being the row's misalignment. Eight tokens that the mask
// forbids are not read.
#pragma once

#include "kv_rope.cuh"

namespace bd3 {

constexpr int kLogitThreads = 256;
constexpr int kLogitSlice = 8192;  // tokens per CTA at most

struct LogitParams {
  const void* logits;          // (B, S, V), vocabulary contiguous
  void* out;                   // (B, S, V), may be `logits`
  long long l_sb, l_ss, o_sb, o_ss;
  const void* history;         // (B, cap) int64 (int32: hist32), or null
  long long h_sb;
  const int* hist_len;         // (B)
  int hist32, hist_cap;
  const float* repetition;     // (B) or null: 1
  const float* presence;       // (B) or null: 0
  const float* frequency;      // (B) or null: 0
  const float* bias;           // (V) with bias_sb = 0 or (B, V), or null
  long long bias_sb;
  const uint32_t* allowed;     // bit v % 32 of word v / 32; strides 0 where shared; or null
  long long a_sb, a_ss;
  int B, S, V;
  int slice;                   // tokens per CTA, a multiple of 8
  int n_slices, rows;          // rows per CTA
};

// Where value x of the slice's bias sits: 8 values and a gap, so that lanes reading value c of
// consecutive groups of 8 hit different banks.
__device__ __forceinline__ int bias_at(int x) { return x + (x >> 3); }

__host__ __device__ constexpr int logit_smem_words(int slice) {
  // counts, bitmap (one word more for the funnel shift), bias: of slice + 8 tokens each
  return (slice + 8) + ((slice + 8) / 32 + 2) + ((slice + 8) / 8 * 9 + 1);
}

template <int kDtype>
__device__ __forceinline__ void store_logit(void* row, long long v, float x) {
  if constexpr (kDtype == 2) reinterpret_cast<float*>(row)[v] = x;
  else reinterpret_cast<uint16_t*>(row)[v] = static_cast<uint16_t>(pack2<kDtype == 0>(x, x));
}
template <int kDtype>
__device__ __forceinline__ float load_logit(const void* row, long long v) {
  if constexpr (kDtype == 0) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[v]);
  else if constexpr (kDtype == 1) return __half2float(reinterpret_cast<const __half*>(row)[v]);
  else return reinterpret_cast<const float*>(row)[v];
}

template <int kDtype>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const LogitParams p) {
  extern __shared__ uint32_t lsm[];
  constexpr int kBytes = kDtype == 2 ? 4 : 2;
  constexpr int kVec = 16 / kBytes;  // logits of a 16-byte access
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y, sl = blockIdx.x;
  // tokens [base, base + slice + 8): the slice's chunks start up to 7 tokens early
  const int k0 = sl * (p.slice / 8), base = 8 * k0 - 8, span = p.slice + 8;
  uint32_t* count = lsm;
  uint32_t* seen = count + span;
  float* s_bias = reinterpret_cast<float*>(seen + span / 32 + 2);
  const int n_hist = p.history == nullptr ? 0 : max(0, min(p.hist_len[b], p.hist_cap));
  if (n_hist > 0) {
    for (int i = threadIdx.x; i < span + span / 32 + 2; i += kLogitThreads) lsm[i] = 0;
  }
  if (p.bias != nullptr) {
    const float* src = p.bias + b * p.bias_sb;
    for (int i = threadIdx.x; i < span; i += kLogitThreads) {
      const int v = base + i;
      s_bias[bias_at(i)] = v >= 0 && v < p.V ? src[v] : 0.f;
    }
  }
  if (n_hist > 0) {
    __syncthreads();
    const long long h0 = b * p.h_sb;
    for (int i = threadIdx.x; i < n_hist; i += kLogitThreads) {
      const long long v = p.hist32 ? reinterpret_cast<const int*>(p.history)[h0 + i]
                                   : reinterpret_cast<const long long*>(p.history)[h0 + i];
      const long long x = v - base;
      if (v >= 0 && v < p.V && x >= 0 && x < span) {
        if (atomicAdd(&count[x], 1u) == 0) atomicOr(&seen[x >> 5], 1u << (x & 31));
      }
    }
  }
  __syncthreads();
  const float rep = p.repetition ? p.repetition[b] : 1.f;
  const float pres = p.presence ? p.presence[b] : 0.f;
  const float freq = p.frequency ? p.frequency[b] : 0.f;
  const int s0 = blockIdx.z * p.rows, s1 = min(s0 + p.rows, p.S);
  for (int s = s0; s < s1; ++s) {
    const uint8_t* in = reinterpret_cast<const uint8_t*>(p.logits) + (b * p.l_sb + s * p.l_ss) * kBytes;
    uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + (b * p.o_sb + s * p.o_ss) * kBytes;
    const uint32_t* mask = p.allowed ? p.allowed + b * p.a_sb + s * p.a_ss : nullptr;
    const int a = static_cast<int>(reinterpret_cast<uintptr_t>(in) / kBytes) & (kVec - 1);
    const bool vec_out = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int k_end = min(k0 + p.slice / 8, (p.V + a + 7) / 8);
    for (int k = k0 + static_cast<int>(threadIdx.x); k < k_end; k += kLogitThreads) {
      const int v0 = 8 * k - a;
      const int x0 = v0 - base;
      const bool whole = v0 >= 0 && v0 + 8 <= p.V;
      uint32_t ok = 0xFFu, hit = 0;
      if (mask != nullptr) {
        if (whole) {
          ok = __funnelshift_r(mask[v0 >> 5], mask[(v0 + 7) >> 5], v0 & 31) & 0xFFu;
        } else {
          ok = 0;
          for (int e = 0; e < 8; ++e) {
            const int v = v0 + e;
            if (v >= 0 && v < p.V) ok |= (mask[v >> 5] >> (v & 31) & 1u) << e;
          }
        }
      }
      if (n_hist > 0) hit = __funnelshift_r(seen[x0 >> 5], seen[(x0 >> 5) + 1], x0 & 31) & 0xFFu;
      float x[8];
      if (ok != 0) {
        if (whole) {
          load8<kDtype>(in, v0, x);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = v0 + e >= 0 && v0 + e < p.V ? load_logit<kDtype>(in, v0 + e) : 0.f;
        }
        if (hit != 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (hit >> e & 1u) {
              const float n = static_cast<float>(count[x0 + e]);
              const float y = x[e] > 0.f ? __fdiv_rn(x[e], rep) : __fmul_rn(x[e], rep);
              x[e] = __fsub_rn(y, __fadd_rn(__fmul_rn(freq, n), pres));
            }
        }
        if (p.bias != nullptr) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(x[e], s_bias[bias_at(x0 + e)]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(ok >> e & 1u)) x[e] = -INFINITY;
      if (whole && vec_out) {
        store8<kDtype>(out, v0, x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v0 + e >= 0 && v0 + e < p.V) store_logit<kDtype>(out, v0 + e, x[e]);
      }
    }
  }
}

}  // namespace bd3
