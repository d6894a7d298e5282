// Attention of many new rows per sequence over a paged KV cache on tcgen05 tensor cores
// (sm_100a): prompt chunks, blocks of grouped heads, and batches that mix them with short
// sequences. paged_sched.cuh has the layout, the visible keys and the distribution of work,
// paged_attn.cuh the mathematics (the same, on 128-row tiles).
//
// One CTA per SM steps through its share of the work list, 128 x 128 score tiles, with TMEM,
// barriers, the K/V ring and the double-buffered Q tile kept across items. The tensor cores
// need 512 cycles a tile at D = 64 and the exponentials 1024 (16 a cycle and SM), so the
// softmax bounds it: two warpgroups share a tile by key columns, each with its own running
// max, sum and O accumulator in TMEM (no exchange per tile), merged once per item. S is
// double-buffered, so the tensor cores work on tile j + 1 during the softmax of tile j.
// Roles (320 threads):
//   warps 0-3  softmax, key columns [0, 64) of every tile: thread t owns row t (TMEM lane t); at
//              an item's end they merge the halves and write O, or the share's partial
//   warps 4-7  softmax, key columns [64, 128)
//   warp 8     producer: Q rows (token, head) by cp.async into the swizzled tile, K and V pieces
//              page by page by TMA
//   warp 9     TMEM owner and UMMA issuer: S = Q K^T (SS), then O_g += P_g V_g (P from TMEM)
// TMEM columns: S0 [0,128), S1 [128,256), O_0 [256,320), O_1 [320,384); P_g (16-bit pairs)
// overwrites the S columns that warpgroup g has read. O_g is rescaled only when a row's max
// grows by more than 2^8 (log2 domain), voted per warp.
#pragma once

#include "attn_fwd.cuh"
#include "paged_attn.cuh"

namespace bd3 {

constexpr int kPtBM = 128, kPtBN = 128;
constexpr int kPtStages = 4;
constexpr int kPtThreads = 320;
constexpr int kPtSlot = 128 * 66;  // floats of a partial: m[128], l[128], O[16][128] float4

struct PtSmem {
  static constexpr uint32_t kQ = 0;                             // [item parity]
  static constexpr uint32_t kK = kQ + 2 * kTile16;
  static constexpr uint32_t kV = kK + kPtStages * kTile16;
  static constexpr uint32_t kBar = kV + kPtStages * kTile16;
  // q_full[2], q_empty[2], k_full[S], v_full[S], kv_empty[S], s_full[2], p_full[2], o_done[2],
  // o_free
  static constexpr uint32_t kNumBars = 4 + 3 * kPtStages + 7;
  static constexpr uint32_t kMerge = kBar + kNumBars * 8;       // [item parity] warpgroup 1's m, l
  static constexpr uint32_t kScan = kMerge + 2 * 2 * 128 * 4;
  static constexpr uint32_t kTmemSlot = kScan + ((sizeof(PagedScan) + 15) / 16) * 16;
  static constexpr uint32_t kLast = kTmemSlot + 8;
  static constexpr uint32_t kBytes = kTmemSlot + 16;
  static constexpr uint32_t kAlloc = kBytes + 1024;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 16u : 0u)
               : "memory");
}

template <bool kBF16>
__global__ void __launch_bounds__(kPtThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v,
                         const __grid_constant__ PagedParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PtSmem::kBar);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 2;
  uint64_t* k_full = bars + 4;
  uint64_t* v_full = k_full + kPtStages;
  uint64_t* kv_empty = v_full + kPtStages;
  uint64_t* s_full = kv_empty + kPtStages;  // [buffer]
  uint64_t* p_full = s_full + 2;            // [warpgroup]
  uint64_t* o_done = s_full + 4;            // [warpgroup]
  uint64_t* o_free = s_full + 6;            // O_0 and O_1 of the item have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + PtSmem::kTmemSlot);
  int* last_flag = reinterpret_cast<int*>(smem + PtSmem::kLast);
  const int warp = static_cast<int>(warp_id());
  const int lane = static_cast<int>(lane_id());

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
    }
    for (int s = 0; s < kPtStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    mbar_init(o_free, 128);
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before();
  griddep_wait();
  griddep_launch_dependents();
  PagedCursor cur = paged_chunk<kPtThreads, kPtBM, kPtBN>(p, reinterpret_cast<PagedScan*>(smem + PtSmem::kScan));
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  PagedItem it;

  if (warp == 8) {
    // ---------------- producer ----------------
    bool ok = true;
    int J = 0;  // key tiles loaded so far
    for (int n = 0; ok && paged_next<kPtBM, kPtBN>(p, cur, it); ++n) {
      const int qb = n & 1;
      if (n >= 2) ok = mbar_wait_warp(&q_empty[qb], ((n >> 1) - 1) & 1);
      if (!ok) break;
      const int rows = it.s.qn * p.G, r0 = it.i * kPtBM;
      const uint32_t sq = sbase + PtSmem::kQ + qb * kTile16;
#pragma unroll 4
      for (int i = 0; i < 32; ++i) {
        const int row = i * 4 + (lane >> 3), c = lane & 7;
        const int r = r0 + row;
        const bool live = r < rows;
        const int t = live ? r / p.G : 0;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + (it.s.q0 + t) * p.q_st +
                              (it.h * p.G + (live ? r - t * p.G : 0)) * p.q_sh + c * 8;
        cp_async16(sq + sw128_offset(row, c), src, live);
      }
      bool q_sent = false;
      auto send_q = [&]() {  // the rows are in shared memory: hand them to the tensor cores
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[qb]);
        q_sent = true;
      };
      const int J0 = J;
      ok = paged_stream<kPtBN>(
          p, it, J,
          [&](int j) {
            if (j == J0 + 1 && !q_sent) send_q();  // with the first K and V tile on their way
            const int st = j % kPtStages;
            if (j >= kPtStages && !mbar_wait_warp(&kv_empty[st], ((j / kPtStages) - 1) & 1))
              return false;
            if (lane == 0) {
              mbar_expect_tx(&k_full[st], kTile16);
              mbar_expect_tx(&v_full[st], kTile16);
            }
            return true;
          },
          [&](int j, int piece, int page, int row) {
            const int st = j % kPtStages;
            const uint32_t off = st * kTile16 + piece * p.box * 128;
            tma_load_4d(&tm_k, &k_full[st], smem + PtSmem::kK + off, 0, row, it.h, page);
            tma_load_4d(&tm_v, &v_full[st], smem + PtSmem::kV + off, 0, row, it.h, page);
          });
      if (!q_sent) send_q();
    }
    __syncwarp();
  } else if (warp == 9) {
    // ---------------- UMMA issuer ----------------
    if (elect_one()) {
      constexpr uint32_t idesc_qk = idesc_f16(128, 128, false, false, kBF16);
      constexpr uint32_t idesc_pv = idesc_f16(128, 64, false, true, kBF16);
      bool ok = true;
      // O_g += P_g V[64g, 64g+64) of key tile Jg, then release its K/V stage; the first one of
      // item n overwrites O, after the previous item's epilogue has read it
      auto issue_pv = [&](int Jg, bool first, int n) {
        const int st = Jg % kPtStages;
        ok = ok && mbar_wait(&v_full[st], (Jg / kPtStages) & 1);
        if (ok && first && n > 0) ok = mbar_wait(o_free, (n - 1) & 1);
        for (int g = 0; g < 2 && ok; ++g) {
          ok = mbar_wait(&p_full[g], Jg & 1);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vdesc =
              sw128_desc(sbase + PtSmem::kV + st * kTile16 + g * (kTile16 / 2), kTile16, 1024);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ts(tmem + 256 + g * 64, tmem + (Jg & 1) * 128 + g * 64 + kk * 8,
                    vdesc + ((kk * 2048) >> 4), idesc_pv, (!first || kk > 0) ? 1u : 0u);
          umma_commit(&o_done[g]);
        }
        if (ok) umma_commit(&kv_empty[st]);
      };
      // S of a tile is issued before O += P V of the one before it, across items too
      int J = 0, prev_J = -1, prev_n = 0;
      bool prev_first = false;
      for (int n = 0; ok && paged_next<kPtBM, kPtBN>(p, cur, it); ++n) {
        const int qb = n & 1;
        ok = mbar_wait(&q_full[qb], (n >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t qdesc = sw128_desc(sbase + PtSmem::kQ + qb * kTile16, 16, 1024);
        for (int t = it.t0; ok && t < it.t1; ++t, ++J) {
          const int st = J % kPtStages;
          ok = mbar_wait(&k_full[st], (J / kPtStages) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint64_t kdesc = sw128_desc(sbase + PtSmem::kK + st * kTile16, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ss(tmem + (J & 1) * 128, qdesc + ((kk * 32) >> 4), kdesc + ((kk * 32) >> 4),
                    idesc_qk, kk > 0 ? 1u : 0u);
          umma_commit(&s_full[J & 1]);
          if (t == it.t1 - 1) umma_commit(&q_empty[qb]);
          if (prev_J >= 0) issue_pv(prev_J, prev_first, prev_n);
          prev_J = J;
          prev_first = t == it.t0;
          prev_n = n;
        }
      }
      if (ok && prev_J >= 0) issue_pv(prev_J, prev_first, prev_n);
    }
    __syncwarp();
  } else {
    // ---------------- softmax: warpgroup g owns key columns [64g, 64g+64) ----------------
    const int g = warp >> 2;
    const int row = threadIdx.x & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_base + 256 + g * 64;
    bool ok = true;
    int J = 0;  // key tiles consumed so far
    for (int n = 0; paged_next<kPtBM, kPtBN>(p, cur, it); ++n) {
      const int rows = it.s.qn * p.G, r = it.i * kPtBM + row;
      const bool live = r < rows;
      const int tok = live ? r / p.G : 0;
      const int row_hi = live ? paged_hi(p, it.s, tok) : 0;
      const int full_all = paged_hi(p, it.s, it.i * kPtBM / p.G);  // seen by every row
      const bool dead = !__any_sync(0xffffffffu, live);  // a warp without rows computes nothing
      float m_run = -INFINITY, l_run = 0.f;
      int Jg = J;
      for (int t = it.t0; t < it.t1; ++t, ++Jg) {
        const int s = t * kPtBN, b = Jg & 1;
        ok = mbar_wait_warp(&s_full[b], (Jg >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tS = tmem + lane_base + b * 128 + g * 64;
        const bool masked = s + kPtBN > full_all;
        const int hi = row_hi - s - g * 64;  // this row's visible columns of the 64: [0, hi)
        const bool skip = dead || (masked && __all_sync(0xffffffffu, hi <= 0));
        float alpha = 1.f, sum = 0.f;
        bool rescale = false;
        if (skip) {
          uint32_t zero[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) zero[i] = 0u;
          if (!dead) tmem_st32(tS, zero);  // (the O rows of a dead warp are not read)
        } else {
          float x[64];
          {
            uint32_t u[2][32];
            tmem_ld32_async(tS, u[0]);
            tmem_ld32_async(tS + 32, u[1]);
            tmem_ld_wait();
#pragma unroll
            for (int c2 = 0; c2 < 2; ++c2) {
              reg_fence(u[c2]);
#pragma unroll
              for (int i = 0; i < 32; ++i) x[c2 * 32 + i] = __uint_as_float(u[c2][i]);
            }
          }
          if (masked) {
#pragma unroll
            for (int c = 0; c < 64; ++c)
              if (c >= hi) x[c] = -INFINITY;
          }
          const float m_new = fmaxf(m_run, max64(x) * p.scale_log2);
          if (m_new - m_run > kRescaleLog2) {  // false for NaN (-inf - -inf)
            alpha = ex2(m_run - m_new);        // 0 when m_run = -inf
            rescale = t > it.t0;
            m_run = m_new;
          }
          const float m_use = m_run == -INFINITY ? 0.f : m_run;
          const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
          const float2 nm2 = make_float2(-m_use, -m_use);
          float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                           make_float2(0.f, 0.f)};
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 z = __ffma2_rn(make_float2(x[2 * i], x[2 * i + 1]), sc2, nm2);
            const float2 e = make_float2(ex2(z.x), ex2(z.y));
            acc[i & 3] = __fadd2_rn(acc[i & 3], e);
            pk[i] = pack2<kBF16>(e.x, e.y);
          }
          const float2 a01 = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
          sum = a01.x + a01.y;
          tmem_st32(tS, pk);
        }
        l_run = l_run * alpha + sum;
        tmem_st_wait();
        if (it.hi - s < kPtBN) {
          // Rows of V past the visible keys hold what the page holds there, NaN included, and
          // P = 0 does not cancel that: zero this warpgroup's half of them before P V.
          const int st = Jg % kPtStages;
          ok = mbar_wait_warp(&v_full[st], (Jg / kPtStages) & 1);
          if (!ok) break;
          const int key = g * 64 + (row >> 1);
          if (key >= it.hi - s) {
            uint8_t* v = smem + PtSmem::kV + st * kTile16 + key * 128 + (row & 1) * 64;
#pragma unroll
            for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(v + 16 * c) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        if (t > it.t0) {
          ok = mbar_wait_warp(&o_done[g], (Jg - 1) & 1);  // O_g += P_g V of the tile before
          if (!ok) break;
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, rescale)) {  // rows that do not need it multiply by 1
          uint32_t u[2][32];
          tmem_ld32_async(tO, u[0]);
          tmem_ld32_async(tO + 32, u[1]);
          tmem_ld_wait();
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2) {
            reg_fence(u[c2]);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              u[c2][i] = __float_as_uint(__uint_as_float(u[c2][i]) * alpha);
            tmem_st32(tO + c2 * 32, u[c2]);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(&p_full[g]);
      }
      // ---- the item's end: merge the halves; write O, or this share's partial ----
      if (ok) ok = mbar_wait_warp(&o_done[g], (Jg - 1) & 1);
      J = Jg;
      float* merge_m = reinterpret_cast<float*>(smem + PtSmem::kMerge) + (n & 1) * 256;
      float* merge_l = merge_m + 128;
      if (g == 1) {
        merge_m[row] = m_run;
        merge_l[row] = l_run;
      }
      tc_fence_before();
      if (!bar_and(1, 256, ok)) break;
      tc_fence_after();
      if (g == 1) continue;
      const float m1 = merge_m[row], l1 = merge_l[row];
      float M = fmaxf(m_run, m1);
      float Mu = M == -INFINITY ? 0.f : M;
      const float w0 = ex2(m_run - Mu), w1 = ex2(m1 - Mu);  // 0 for a half that saw no key
      float L = l_run * w0 + l1 * w1;
      float o[64];
      {
        uint32_t u0[2][32], u1[2][32];
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          tmem_ld32_async(tmem + lane_base + 256 + c2 * 32, u0[c2]);
          tmem_ld32_async(tmem + lane_base + 320 + c2 * 32, u1[c2]);
        }
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(o_free);  // the next item may overwrite O_0 and O_1
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          reg_fence(u0[c2]);
          reg_fence(u1[c2]);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            o[c2 * 32 + i] = __uint_as_float(u0[c2][i]) * w0 + __uint_as_float(u1[c2][i]) * w1;
        }
      }
      if (it.parts > 1) {
        float* slot = p.partials + static_cast<long long>(it.slot) * kPtSlot;
        if (live) {
          slot[row] = M;
          slot[128 + row] = L;
          float4* dst = reinterpret_cast<float4*>(slot + 256) + row;
#pragma unroll
          for (int c = 0; c < 16; ++c)
            dst[c * 128] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        }
        // the share that finishes last merges the item's partials, in CTA order
        asm volatile("bar.sync 2, 128;" ::: "memory");
        if (threadIdx.x == 0) {
          __threadfence();
          const int before = atomicAdd(&p.counters[it.slot0], 1);
          *last_flag = before == it.parts - 1;
          if (before == it.parts - 1) p.counters[it.slot0] = 0;
          __threadfence();
        }
        asm volatile("bar.sync 2, 128;" ::: "memory");
        const bool last = *last_flag != 0;
        if (!last) continue;
        M = -INFINITY;
        L = 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) o[i] = 0.f;
        for (int j = 0; live && j < it.parts; ++j) {
          const float* src = p.partials + static_cast<long long>(paged_part_slot(it, j)) * kPtSlot;
          const float m = __ldcg(src + row), l = __ldcg(src + 128 + row);
          const float4* so = reinterpret_cast<const float4*>(src + 256) + row;
          const float m_new = fmaxf(M, m), mu = m_new == -INFINITY ? 0.f : m_new;
          const float a = ex2(M - mu), w = ex2(m - mu);
          M = m_new;
          L = L * a + l * w;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float4 v = __ldcg(so + c * 128);
            o[4 * c] = o[4 * c] * a + v.x * w;
            o[4 * c + 1] = o[4 * c + 1] * a + v.y * w;
            o[4 * c + 2] = o[4 * c + 2] * a + v.z * w;
            o[4 * c + 3] = o[4 * c + 3] * a + v.w * w;
          }
        }
        Mu = M == -INFINITY ? 0.f : M;
      }
      if (live) {
        const float inv = L == 0.f ? 0.f : 1.f / L;  // L = 0: a row without keys
        const int hq = it.h * p.G + (r - tok * p.G);
        const long long off = (it.s.q0 + tok) * p.o_st + hq * p.o_sh;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = o[8 * c + i] * inv;
          paged_store8<kBF16>(p, off + 8 * c, v);
        }
        if (p.lse != nullptr)
          p.lse[static_cast<long long>(it.s.q0 + tok) * (p.Hkv * p.G) + hq] =
              L == 0.f ? -INFINITY : (Mu + log2f(L)) * 0.69314718055994530942f;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace bd3
