// Processing of a step's logits before sampling (sm_100a): penalties for repeated tokens, a bias
// and a grammar mask, in one pass. For row (b, s) and token v, with n the times v occurs in the
// first hist_len[b] entries of history[b]:
//   x = logits[b, s, v]
//   if n > 0:  x = (x > 0 ? x / r_b : x * r_b) - (f_b * n + p_b)
//   x += bias[v] (or bias[b, v]);  x = -inf where the mask's bit v is 0
// in fp32, each product, quotient and sum rounded to fp32, the result rounded once to the
// logits' type. The S rows of a sequence (a block of a denoising step) share its history.
//
// DRAM-bound: every logit is read and written once, 16 bytes an access; a chunk of eight (four in
// fp32) tokens that the mask forbids is not read. At that rate a warp has about 170 issue slots
// for 32 chunks, so what is the same for several rows is worked out once. A CTA takes a slice of
// the vocabulary, kU chunks a thread, for some rows of one sequence. Rows of an odd vocabulary
// start at any alignment, so a row's chunks begin `a` logits before the multiples of the chunk,
// a being its misalignment, which repeats every `period` rows: the CTA takes the rows of one
// alignment together, with their mask and bias in registers, kR rows' loads at a time. (The two
// ends of a row go one logit a thread.)
// The history's tokens of the slice are counted in shared memory (integer atomics: their order
// does not matter) and listed. The streaming leaves the listed tokens as they were; then the CTA's
// threads go over the list, all lanes at work. (Penalising them while streaming has one or two
// lanes of a warp divide at a time: two thirds of all instructions with several rows; single fp32
// rows do it all the same, see kInline.)
// Measured: 64 x 16 rows of 50258 bf16 logits with bias, mask and histories of 64 to 1024 tokens
// 50 us (42 us with histories up to 64, where a copy takes 35; the scattered pass over the listed
// tokens is the rest); 96 fp32 rows of 128001 44 us with histories of up to 16384 (1296 in the
// mean), 40 with 64 each, 84 with 16384 each: every slice's CTA scans all of its sequence's
// history, from L2. Before, with the counting behind the logits' loads at four CTAs an SM and four
// rows at a time, those took 53, 46, 55, 40 and 129 us. Slices of 8192 tokens, CTAs of 128, 512 and
// 1024 threads, eight or more history loads in flight, the next batch loaded ahead (70 against 55),
// a list made by ballots over the counts, and histories read by eighths in clusters of 8 CTAs
// (adding through distributed shared memory) were all slower over these lengths.
#pragma once

#include <type_traits>

#include "kv_rope.cuh"

namespace bd3 {

constexpr int kLogitThreads = 256;

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
  int S, V;
  int rows;                    // rows per CTA
};

template <int kDtype, int kU>
struct LogitTile {
  static constexpr int kBytes = kDtype == 2 ? 4 : 2;
  static constexpr int kE = 16 / kBytes;                     // logits of a chunk
  static constexpr int kSlice = kLogitThreads * kU * kE;     // tokens of a CTA
  static constexpr int kSpan = kSlice + kE;                  // its chunks start up to kE - 1 early
  // shared words: counts, then the bitmap (one word more for the funnel shift)
  static constexpr int kSeen = kSpan, kWords = kSeen + kSpan / 32 + 2;
  static_assert(kSpan <= 65536, "the list holds 16-bit positions");
};

template <int kDtype>
__device__ __forceinline__ float load_logit(const void* row, long long v) {
  if constexpr (kDtype == 0) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[v]);
  else if constexpr (kDtype == 1) return __half2float(reinterpret_cast<const __half*>(row)[v]);
  else return reinterpret_cast<const float*>(row)[v];
}
template <int kDtype>
__device__ __forceinline__ void store_logit(void* row, long long v, float x) {
  if constexpr (kDtype == 2) reinterpret_cast<float*>(row)[v] = x;
  else reinterpret_cast<uint16_t*>(row)[v] = static_cast<uint16_t>(pack2<kDtype == 0>(x, x));
}

__device__ __forceinline__ float penalise(float x, float n, float rep, float freq, float pres) {
  const float y = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
  return __fsub_rn(y, __fadd_rn(__fmul_rn(freq, n), pres));
}

// CTAs an SM: six (40 registers) hide the latency of a CTA's own phases; not where four chunks a
// thread need the registers, nor for one row of one chunk (50258 bf16 logits: 3.1 us at four CTAs
// an SM, 3.4 at six).
constexpr int logit_ctas(int dtype, int u, int r) { return r == 1 && (u == 1 || dtype == 2) ? 4 : 6; }

template <int kDtype, int kU, int kR>
__global__ void __launch_bounds__(kLogitThreads, logit_ctas(kDtype, kU, kR))
    logits_kernel(const LogitParams p) {
  using T = LogitTile<kDtype, kU>;
  constexpr int kE = T::kE;
  // Listed tokens are penalised as they stream by: single fp32 rows, whose chunks are four tokens
  // (96 rows of 128001: histories of 1024 tokens 43 us against 45 by the list, of 16384 84 against
  // 111; 256 bf16 rows of 32000 with 1024, eight tokens a chunk, 25.6 against 23.4).
  constexpr bool kInline = kR == 1 && kU > 1 && kDtype == 2;
  // The history comes before the loads of the logits, so that its counting has their registers;
  // behind them where a CTA has one chunk a thread and nothing else hides its latency.
  constexpr bool kFirst = kR > 1 || kU > 1;
  constexpr uint32_t kAll = (1u << kE) - 1u;
  __shared__ uint32_t lsm[T::kWords];
  __shared__ uint16_t list[kInline ? 1 : T::kSpan];  // the slice's tokens that the history holds
  __shared__ int n_list;
  uint32_t* const count = lsm;
  uint32_t* const seen = lsm + T::kSeen;
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y, k0 = blockIdx.x * (T::kSlice / kE);
  const int base = (k0 - 1) * kE;  // token of the span's first count
  const int s0 = blockIdx.z * p.rows, s1 = min(s0 + p.rows, p.S);
  const uint8_t* const in0 = reinterpret_cast<const uint8_t*>(p.logits) + b * p.l_sb * T::kBytes;
  uint8_t* const out0 = reinterpret_cast<uint8_t*>(p.out) + b * p.o_sb * T::kBytes;
  const uint32_t* const mask0 = p.allowed ? p.allowed + b * p.a_sb : nullptr;
  const bool row_mask = kR > 1 && mask0 != nullptr && p.a_ss != 0;  // (kR = 1: one row)
  const float* const bias = p.bias ? p.bias + b * p.bias_sb : nullptr;
  const int n_hist = p.history == nullptr ? 0 : max(0, min(p.hist_len[b], p.hist_cap));
  const float rep = p.repetition ? p.repetition[b] : 1.f;
  const float pres = p.presence ? p.presence[b] : 0.f;
  const float freq = p.frequency ? p.frequency[b] : 0.f;

  // counts of the slice's tokens in the history (whole CTA)
  auto count_history = [&]() {
    for (int i = threadIdx.x; i < T::kWords; i += kLogitThreads) lsm[i] = 0;
    if (threadIdx.x == 0) n_list = 0;
    __syncthreads();
    const long long h0 = b * p.h_sb;
    // tokens [lo, lo + n_in) are counted here: one unsigned comparison a token
    const int lo = max(base, 0), off = lo - base;
    const uint32_t n_in = max(min(base + T::kSpan, p.V) - lo, 0);
    auto add = [&](auto d) {
      if (d < n_in) {
        const uint32_t x = static_cast<uint32_t>(d) + off;
        if (atomicAdd(&count[x], 1u) == 0) {
          atomicOr(&seen[x >> 5], 1u << (x & 31));
          if constexpr (!kInline) list[atomicAdd(&n_list, 1)] = static_cast<uint16_t>(x);
        }
      }
    };
    auto scan = [&](const auto* h) {  // unsigned: a token below lo is far above lo + n_in, as ~0 is
      using U = std::remove_cv_t<std::remove_reference_t<decltype(*h)>>;
      const U low = static_cast<U>(lo);
      U v[4];  // 4 loads of a thread in flight
      int i = threadIdx.x;
      if constexpr (kFirst) {
        for (; i + 3 * kLogitThreads < n_hist; i += 4 * kLogitThreads) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = h[i + j * kLogitThreads];
#pragma unroll
          for (int j = 0; j < 4; ++j) add(v[j] - low);
        }
      }
      for (; i < n_hist; i += 4 * kLogitThreads) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j * kLogitThreads < n_hist ? h[i + j * kLogitThreads] : ~U(0);
#pragma unroll
        for (int j = 0; j < 4; ++j) add(v[j] - low);
      }
    };
    if (p.hist32) scan(reinterpret_cast<const uint32_t*>(p.history) + h0);
    else scan(reinterpret_cast<const unsigned long long*>(p.history) + h0);
    __syncthreads();
  };
  // the mask's bits of the tokens [v0, v0 + kE)
  auto bits_of = [&](const uint32_t* m, int v0) {
    return __funnelshift_r(m[v0 >> 5], m[(v0 + kE - 1) >> 5], v0 & 31) & kAll;
  };

  // which bits of a chunk's four words the mask keeps
  auto keep_of = [&](uint32_t ok, uint32_t (&keep)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kDtype == 2) {
        keep[j] = ok >> j & 1u ? 0xFFFFFFFFu : 0u;
      } else {
        const uint32_t two = ok >> (2 * j);
        keep[j] = (two & 1u) * 0xFFFFu + (two & 2u) * 0x7FFF8000u;
      }
    }
  };

  if (kFirst && n_hist > 0) count_history();
  // rows of one alignment: s0 + c, s0 + c + period, ...
  const int step = static_cast<int>(p.l_ss & (kE - 1));
  const int period = step == 0 ? 1 : kE / (step & -step);
  const long long step_in = period * p.l_ss * T::kBytes, step_out = period * p.o_ss * T::kBytes;
  const bool same_step = ((step_in ^ step_out) & 15) == 0;  // in and out keep their distance mod 16
  bool counted = n_hist == 0;
  for (int c = 0; c < period && s0 + c < s1; ++c) {
    const int a = static_cast<int>(reinterpret_cast<uintptr_t>(in0 + (s0 + c) * p.l_ss * T::kBytes) / T::kBytes) & (kE - 1);
    // of this thread's chunks in the rows of this alignment: first token, where the first row has
    // it, its mask (0 at an end of the row or past it) and, as a 16-bit mask per logit, what to keep
    int v0[kU];
    const uint8_t* pin[kU];
    uint8_t* pout[kU];
    uint32_t ok_all[kU], keep[kU][4];
    float bv[kU][kE];
    const uint8_t* const in_c = in0 + (s0 + c) * p.l_ss * T::kBytes;
    uint8_t* const out_c = out0 + (s0 + c) * p.o_ss * T::kBytes;
    const bool vec = ((reinterpret_cast<uintptr_t>(in_c) ^ reinterpret_cast<uintptr_t>(out_c)) & 15) == 0 && same_step;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      v0[u] = (k0 + u * kLogitThreads + static_cast<int>(threadIdx.x)) * kE - a;
      pin[u] = in_c + static_cast<long long>(v0[u]) * T::kBytes;
      pout[u] = out_c + static_cast<long long>(v0[u]) * T::kBytes;
      ok_all[u] = v0[u] >= 0 && v0[u] + kE <= p.V ? kAll : 0u;
      if (ok_all[u] != 0 && mask0 != nullptr && !row_mask) ok_all[u] = bits_of(mask0 + s0 * p.a_ss, v0[u]);
      keep_of(ok_all[u], keep[u]);
    }
    for (int sb = s0 + c; sb < s1; sb += period * kR) {
      uint32_t ok[kR][kU];
      uint4 raw[kR][kU];
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const int s = sb + r * period;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          ok[r][u] = s < s1 ? ok_all[u] : 0u;
          if (row_mask && ok[r][u] != 0) ok[r][u] = bits_of(mask0 + s * p.a_ss, v0[u]);
        }
      }
#pragma unroll
      for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (ok[r][u] != 0) raw[r][u] = *reinterpret_cast<const uint4*>(pin[u] + r * step_in);
      if (sb == s0 + c) {  // once for the rows of this alignment, behind the first loads
        if (bias != nullptr) {
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            const float* src = bias + v0[u];
            if (ok_all[u] == 0) continue;
            if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
#pragma unroll
              for (int e = 0; e < kE; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(src + e);
                bv[u][e] = f.x, bv[u][e + 1] = f.y, bv[u][e + 2] = f.z, bv[u][e + 3] = f.w;
              }
            } else {
#pragma unroll
              for (int e = 0; e < kE; ++e) bv[u][e] = src[e];
            }
          }
        }
        if (!kFirst && !counted) {
          count_history();
          counted = true;
        }
        if (!kInline && bias != nullptr && n_hist > 0) {  // listed tokens stay as they are for now
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            if (ok_all[u] == 0) continue;
            const int x0 = v0[u] - base;
            const uint32_t hit = __funnelshift_r(seen[x0 >> 5], seen[(x0 >> 5) + 1], x0 & 31) & kAll;
            if (hit == 0) continue;
#pragma unroll
            for (int e = 0; e < kE; ++e)
              if (hit >> e & 1u) bv[u][e] = 0.f;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        if (sb + r * period >= s1) break;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          if (v0[u] < 0 || v0[u] + kE > p.V) continue;  // an end of the row, below, or past it
          uint32_t w[4] = {raw[r][u].x, raw[r][u].y, raw[r][u].z, raw[r][u].w};
          uint32_t hit = 0;  // one row: what the history holds of the chunk
          if (kInline && n_hist > 0) {
            const int x0 = v0[u] - base;
            hit = __funnelshift_r(seen[x0 >> 5], seen[(x0 >> 5) + 1], x0 & 31) & ok[r][u];
          }
          if (bias != nullptr || hit != 0) {
            auto value = [&](float x, int e) {
              if (kInline && (hit >> e & 1u)) x = penalise(x, static_cast<float>(count[v0[u] - base + e]), rep, freq, pres);
              return bias != nullptr ? __fadd_rn(x, bv[u][e]) : x;
            };
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if constexpr (kDtype == 2) {
                w[j] = __float_as_uint(value(__uint_as_float(w[j]), j));
              } else {
                const float2 f = unpack2<kDtype == 0>(w[j]);
                w[j] = pack2<kDtype == 0>(value(f.x, 2 * j), value(f.y, 2 * j + 1));
              }
            }
          }
          if (mask0 != nullptr) {  // forbidden tokens
            constexpr uint32_t kInf = kDtype == 0 ? 0xFF80FF80u : kDtype == 1 ? 0xFC00FC00u : 0xFF800000u;
            if (row_mask) keep_of(ok[r][u], keep[u]);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (w[j] & keep[u][j]) | (kInf & ~keep[u][j]);
          }
          uint8_t* const out = pout[u] + r * step_out;
          if (vec) {
            *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              if constexpr (kDtype == 2) reinterpret_cast<uint32_t*>(out)[e] = w[e];
              else reinterpret_cast<uint16_t*>(out)[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        pin[u] += kR * step_in;
        pout[u] += kR * step_out;
      }
    }
  }
  // ---- the ends of the rows: tokens before the first whole chunk and after the last ----
  for (int i = threadIdx.x; i < (s1 - s0) * 2 * kE; i += kLogitThreads) {
    const int s = s0 + i / (2 * kE), e = i % (2 * kE);
    const uint8_t* in = in0 + s * p.l_ss * T::kBytes;
    const int a = static_cast<int>(reinterpret_cast<uintptr_t>(in) / T::kBytes) & (kE - 1);
    const int head = a == 0 ? 0 : min(kE - a, p.V);  // tokens [0, head) of chunk 0
    const int last = (p.V + a) / kE;                 // chunk of the tokens after the last whole one
    const int v = e < kE ? e : last * kE - a + e - kE;
    const bool mine = e < kE ? k0 == 0 && v < head
                             : last >= k0 && last < k0 + T::kSlice / kE && v >= head && v < p.V;
    if (!mine) continue;
    const uint32_t* m = mask0 ? mask0 + s * p.a_ss : nullptr;
    float y = -INFINITY;
    if (m == nullptr || (m[v >> 5] >> (v & 31) & 1u)) {
      y = load_logit<kDtype>(in, v);
      const uint32_t n = n_hist > 0 ? count[v - base] : 0;
      if (kInline && n != 0) y = penalise(y, static_cast<float>(n), rep, freq, pres);
      if (bias != nullptr && (kInline || n == 0)) y = __fadd_rn(y, bias[v]);
    }
    store_logit<kDtype>(out0 + s * p.o_ss * T::kBytes, v, y);
  }
  if (kInline || n_hist == 0) return;
  // ---- the listed tokens ----
  __syncthreads();  // the rows are in `out`
  if constexpr (kR == 1) {
    // one row: a thread takes every kLogitThreads-th token, four loads at a time
    for (int i0 = threadIdx.x; i0 < n_list; i0 += 4 * kLogitThreads) {
      float y[4];
      int px[4];
      bool live[4];
      const int a = static_cast<int>(reinterpret_cast<uintptr_t>(in0 + s0 * p.l_ss * T::kBytes) / T::kBytes) & (kE - 1);
      uint8_t* const out = out0 + s0 * p.o_ss * T::kBytes;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kLogitThreads;
        live[j] = i < n_list;
        if (!live[j]) continue;
        px[j] = list[i];
        const int v = base + px[j];
        // not the neighbour's (the span's ends are, for some alignments), nor forbidden
        live[j] = v >= k0 * kE - a && v < k0 * kE - a + T::kSlice &&
                  (mask0 == nullptr || (mask0[s0 * p.a_ss + (v >> 5)] >> (v & 31) & 1u));
        if (live[j]) y[j] = load_logit<kDtype>(out, v);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!live[j]) continue;
        const int v = base + px[j];
        y[j] = penalise(y[j], static_cast<float>(count[px[j]]), rep, freq, pres);
        if (bias != nullptr) y[j] = __fadd_rn(y[j], bias[v]);
        store_logit<kDtype>(out, v, y[j]);
      }
    }
    return;
  }
  // a thread takes a token and every `groups`-th row: its count, bias and shared mask once
  const int rows = s1 - s0, listed = n_list;
  const int groups = listed == 0 ? 1 : min(rows, max(1, kLogitThreads / listed));
  for (int i = threadIdx.x; i < listed * groups; i += kLogitThreads) {
    const int g = i / listed, x = list[i - g * listed], v = base + x;
    const float n = static_cast<float>(count[x]), bias_v = bias != nullptr ? bias[v] : 0.f;
    if (mask0 != nullptr && !row_mask && !(mask0[s0 * p.a_ss + (v >> 5)] >> (v & 31) & 1u)) continue;
    for (int r = g; r < rows; r += 4 * groups) {
      float y[4];
      bool live[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = s0 + r + j * groups;
        live[j] = s < s1;
        if (!live[j]) continue;
        // not the neighbour's (the span's ends are, for some alignments), nor forbidden
        const int a = static_cast<int>(reinterpret_cast<uintptr_t>(in0 + s * p.l_ss * T::kBytes) / T::kBytes) & (kE - 1);
        live[j] = v >= k0 * kE - a && v < k0 * kE - a + T::kSlice &&
                  (!row_mask || (mask0[s * p.a_ss + (v >> 5)] >> (v & 31) & 1u));
        if (live[j]) y[j] = load_logit<kDtype>(out0 + s * p.o_ss * T::kBytes, v);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!live[j]) continue;
        y[j] = penalise(y[j], n, rep, freq, pres);
        if (bias != nullptr) y[j] = __fadd_rn(y[j], bias_v);
        store_logit<kDtype>(out0 + (s0 + r + j * groups) * p.o_ss * T::kBytes, v, y[j]);
      }
    }
  }
}

}  // namespace bd3
