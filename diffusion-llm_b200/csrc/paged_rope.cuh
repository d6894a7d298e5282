// Fused QKV split + rotary embedding + write into a paged KV cache (sm_100a).
//
// For each packed new token (paged_sched.cuh has the layout): q and k are rotated by the angle of
// the token's position p,
//   out_1 = x_1 cos - x_2 sin,  out_2 = x_1 sin + x_2 cos   for the pair (x_k, x_{k + D/2}),
// in fp32 from the fp32 tables and rounded once to the tensors' type; q goes to its own tensor,
// k and v to row p % page_size of page page_table[b, p / page_size]. (qkv_rope_cache_kernel
// repeats the reference's rounding of every product and sum; this one rounds the result only.)
//
// DRAM-bound: the projection is read once and q, k, v are written once, 16 bytes an access. A
// CTA takes `tpb` tokens; one thread per token finds its sequence, page and row, then the
// threads share the (token, head, 8 pairs) units. Measured: 5753 tokens of 32 + 2 x 8 f16 heads
// 16.6 us (4.5 TB/s, 0.69 of the copy rate), 16384 fp32 tokens of 12 + 2 x 12 heads 52.3 us
// (5.8 TB/s, 0.88); 1024 tokens of a denoising step 5.1 us, latency.
#pragma once

#include "kv_rope.cuh"

namespace bd3 {

constexpr int kRopeMaxTokens = 64;  // tokens per CTA at most

struct PagedRopeParams {
  const void* qkv;             // (T, (Hq + 2 Hkv) * D) rows of q, k, v heads
  long long qkv_st;
  const float* cos_table;      // (max_pos, D/2) fp32
  const float* sin_table;
  long long max_pos;
  void* q_out;                 // (T, Hq, D)
  long long q_st, q_sh;
  void* k_pages;               // (num_pages, Hkv, page_size, D)
  long long k_sp, k_sh, k_sr;
  void* v_pages;
  long long v_sp, v_sh, v_sr;
  const int* page_table;       // (B, max_pages)
  long long pt_stride;
  const int* kv_lens;          // (B)
  const int* cu_q;             // (B + 1)
  int B, T, Hq, Hkv, D, tpb;
  int num_pages, page_size, max_pages;
};

template <int kDtype>
__global__ void __launch_bounds__(256) qkv_rope_paged_kernel(const PagedRopeParams p) {
  __shared__ int s_pos[kRopeMaxTokens];   // position, or -1: the token is left alone
  __shared__ int s_page[kRopeMaxTokens], s_row[kRopeMaxTokens];
  griddep_wait();
  griddep_launch_dependents();
  const int t0 = blockIdx.x * p.tpb;
  const int n = p.T - t0 < p.tpb ? p.T - t0 : p.tpb;
  // the sequence of the first token: the number of sequences that end at or before it
  int b0 = 0;
  for (int j = 0; j < p.B; j += 256) {
    const int e = j + static_cast<int>(threadIdx.x);
    b0 += __syncthreads_count(e < p.B && p.cu_q[e + 1] <= t0);
  }
  if (static_cast<int>(threadIdx.x) < n) {
    const int t = t0 + static_cast<int>(threadIdx.x);
    int b = b0;
    while (b < p.B && p.cu_q[b + 1] <= t) ++b;
    int pos = -1, page = 0, row = 0;
    if (b < p.B && t >= p.cu_q[b]) {  // tokens before cu_q[0] or past cu_q[B] are in no sequence
      const long long at = static_cast<long long>(p.kv_lens[b]) - p.cu_q[b + 1] + t;
      const long long pg = at / p.page_size;
      bool ok = at >= 0 && at < p.max_pos && pg < p.max_pages;
      if (ok) {
        page = p.page_table[b * p.pt_stride + pg];
        ok = page >= 0 && page < p.num_pages;
      }
      if (ok) {
        pos = static_cast<int>(at);
        row = static_cast<int>(at - pg * p.page_size);
      } else {
        atomicOr(&g_bd3_status, kStatusBadPosition);
      }
    }
    s_pos[threadIdx.x] = pos;
    s_page[threadIdx.x] = page;
    s_row[threadIdx.x] = row;
  }
  __syncthreads();
  const int groups = p.D / 16, half = p.D / 2;
  const int slots = p.Hq + 2 * p.Hkv;
  const int units = n * slots * groups;
  for (int u = threadIdx.x; u < units; u += 256) {
    const int k = 8 * (u % groups);
    const int v = u / groups;
    const int hs = v % slots, tl = v / slots;
    const int pos = s_pos[tl];
    if (pos < 0) continue;
    const long long src = (t0 + tl) * p.qkv_st + static_cast<long long>(hs) * p.D + k;
    float x1[8], x2[8];
    load8<kDtype>(p.qkv, src, x1);
    load8<kDtype>(p.qkv, src + half, x2);
    void* dst;
    long long off;
    if (hs < p.Hq) {
      dst = p.q_out;
      off = (t0 + tl) * p.q_st + hs * p.q_sh;
    } else if (hs < p.Hq + p.Hkv) {
      dst = p.k_pages;
      off = s_page[tl] * p.k_sp + (hs - p.Hq) * p.k_sh + s_row[tl] * p.k_sr;
    } else {
      dst = p.v_pages;
      off = s_page[tl] * p.v_sp + (hs - p.Hq - p.Hkv) * p.v_sh + s_row[tl] * p.v_sr;
    }
    if (hs < p.Hq + p.Hkv) {
      const float4* ct = reinterpret_cast<const float4*>(p.cos_table + static_cast<long long>(pos) * half + k);
      const float4* st = reinterpret_cast<const float4*>(p.sin_table + static_cast<long long>(pos) * half + k);
      const float4 c0 = __ldg(ct), c1 = __ldg(ct + 1), s0 = __ldg(st), s1 = __ldg(st + 1);
      const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = x1[e], b = x2[e];
        x1[e] = a * c[e] - b * sn[e];
        x2[e] = a * sn[e] + b * c[e];
      }
    }
    store8<kDtype>(dst, off + k, x1);
    store8<kDtype>(dst, off + k + half, x2);
  }
}

}  // namespace bd3
