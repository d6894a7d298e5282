// Attention of many new rows per sequence over a paged KV cache on tcgen05 tensor cores
// (sm_100a): prompt chunks, blocks of grouped heads, and batches that mix them with short
// sequences. paged_sched.cuh has the layout, the visible keys and the distribution of work,
// paged_attn.cuh the mathematics (the same, on 128-row tiles).
//
// The tensor cores need 512 cycles for a 128 x 128 tile at D = 64 and the exponentials 1024 (16 a
// cycle and SM), so the softmax bounds it, and within it the latency of its chain (TMEM load,
// row max, exponentials, P store): one warpgroup alone leaves the exponential units idle for
// most of a tile. So each SM runs two independent workers, each with its own chunk of the work
// list, Q tile, K/V ring, TMEM columns and three roles, and nothing synchronises them: one's
// exponentials fill the other's loads and waits. (Measured on a 2048-token chunk after 8192, 12
// heads: key columns of one tile split between the warpgroups 126 us, two workers 119 us, with
// registers moved to the softmax 113 us. Three workers on 64-key tiles: 131 us, their rings and
// TMEM leave each too little. The row max by 32-column chunks, ahead of or behind the
// exponentials: 119 to 134 us. A quarter of the exponentials on the FMA pipe: 109 us there, but
// 88 against 82 us on short prompts, whose code then no longer fits the instruction cache.)
// Per worker x (384 threads in all):
//   warps 4x..4x+3  softmax: thread t owns row t (TMEM lane t) and all 128 columns of a tile; at a
//                   share's end O / l to global memory, or the share's partial
//   warp 8 + x      producer: Q rows (token, head) by cp.async into the swizzled tile, K and V
//                   pieces page by page by TMA
//   warp 10 + x     UMMA issuer (warp 10 owns the TMEM): S = Q K^T (SS), then O += P V (P from TMEM)
// TMEM columns: S_x [128x, +128), P_x (16-bit pairs) [256 + 64x, +64), O_x [384 + 64x, +64). S_x is
// released as soon as its rows are in registers, so the next S is computed during the
// exponentials. O is rescaled only when a row's max grows by more than 2^8 (log2 domain),
// voted per warp.
#pragma once

#include "attn_fwd_pair.cuh"
#include "paged_attn.cuh"

namespace bd3 {

constexpr int kPtBM = 128, kPtBN = 128;
constexpr int kPtWorkers = 2;
constexpr int kPtStages = 3;
constexpr int kPtThreads = 384;
constexpr int kPtItemCost = 2;     // an item's fixed cost in key tiles
// Registers a thread, of the 168 that 384 threads launch with: the softmax holds a row's 128
// scores (ptxas reports 238 bytes of spill stores a thread without the split, 84 with it), the
// other four warps need few. 256 x 192 + 128 x 120 = 384 x 168;
// the host checks that the kernel has the 168 (more than the launch's own would wait for ever).
constexpr int kPtRegs = 168, kPtRegsSoftmax = 192, kPtRegsOther = 120;
static_assert(256 * kPtRegsSoftmax + 128 * kPtRegsOther <= kPtThreads * kPtRegs, "register split");
constexpr int kPtSlot = 128 * 66;  // floats of a partial: m[128], l[128], O[16][128] float4

struct PtSmem {
  // per worker: Q, then K and V of each stage
  static constexpr uint32_t kQ = 0, kK = kTile16, kV = kK + kPtStages * kTile16;
  static constexpr uint32_t kWorker = kV + kPtStages * kTile16;
  static constexpr uint32_t kBar = 2 * kWorker;
  // per worker: q_full, q_empty, s_full, s_free, p_full, o_done, o_free, k_full[S], v_full[S],
  // kv_empty[S]
  static constexpr uint32_t kNumBars = 7 + 3 * kPtStages;
  static constexpr uint32_t kScan = kBar + 2 * kNumBars * 8;
  static constexpr uint32_t kTmemSlot = kScan + sizeof(PagedScan);
  static constexpr uint32_t kLast = kTmemSlot + 8;  // [worker]
  static constexpr uint32_t kBytes = kLast + 8;
  static constexpr uint32_t kAlloc = kBytes + 1024;
};
static_assert(PtSmem::kAlloc <= 227 * 1024, "shared memory of one CTA");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 16u : 0u)
               : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

template <bool kBF16>
__global__ void __launch_bounds__(kPtThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v,
                         const __grid_constant__ PagedParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + PtSmem::kTmemSlot);
  const int warp = static_cast<int>(warp_id());
  const int lane = static_cast<int>(lane_id());
  const int x = warp < 8 ? warp >> 2 : warp & 1;  // this warp's worker
  uint8_t* const wsm = smem + x * PtSmem::kWorker;
  const uint32_t wbase = smem_u32(wsm);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + PtSmem::kBar) + x * PtSmem::kNumBars;
  uint64_t* const q_full = bars;
  uint64_t* const q_empty = bars + 1;
  uint64_t* const s_full = bars + 2;
  uint64_t* const s_free = bars + 3;
  uint64_t* const p_full = bars + 4;
  uint64_t* const o_done = bars + 5;
  uint64_t* const o_free = bars + 6;
  uint64_t* const k_full = bars + 7;
  uint64_t* const v_full = k_full + kPtStages;
  uint64_t* const kv_empty = v_full + kPtStages;

  if (threadIdx.x < 2) {
    uint64_t* bb = reinterpret_cast<uint64_t*>(smem + PtSmem::kBar) + threadIdx.x * PtSmem::kNumBars;
    for (int i = 0; i < static_cast<int>(PtSmem::kNumBars); ++i)
      mbar_init(&bb[i], i == 3 || i == 4 || i == 6 ? 128 : 1);  // s_free, p_full, o_free
    fence_mbar_init();
  }
  if (warp == 10) {
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
  PagedCursor cur = paged_chunk<kPtThreads, 2, kPtBM, kPtBN, kPtItemCost>(
      p, reinterpret_cast<PagedScan*>(smem + PtSmem::kScan), x);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  PagedItem it;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPtRegsOther));
    if (warp < 10) {
      // ---------------- producer ----------------
      bool ok = true;
      int J = 0;  // key tiles loaded so far
      for (int n = 0; ok && paged_next<kPtBM, kPtBN, kPtItemCost>(p, cur, it); ++n) {
        // Q: issued first for the first item, and for a later one after its first K/V tile (the Q
        // tile is in use until the last S of the item before)
        bool q_sent = false;
        auto load_q = [&]() {
          if (n > 0 && !mbar_wait_warp(q_empty, (n - 1) & 1)) return false;
          const int rows = it.s.qn * p.G, r0 = it.i * kPtBM;
#pragma unroll 4
          for (int i = 0; i < 32; ++i) {
            const int row = i * 4 + (lane >> 3), c = lane & 7;
            const int r = r0 + row;
            const bool live = r < rows;
            const int t = live ? p.by_G.div(r) : 0;
            const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + (it.s.q0 + t) * p.q_st +
                                  (it.h * p.G + (live ? r - t * p.G : 0)) * p.q_sh + c * 8;
            cp_async16(wbase + PtSmem::kQ + sw128_offset(row ^ (64 * x), c), src, live);
          }
          return true;
        };
        auto send_q = [&]() {  // the rows are in shared memory: hand them to the tensor cores
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(q_full);
          q_sent = true;
        };
        const int J0 = J;
        if (n == 0) ok = load_q();
        ok = ok && paged_stream<kPtBN>(
            p, it, J,
            [&](int j) {
              if (j == J0 + 1 && !q_sent) {
                if (n > 0 && !load_q()) return false;
                send_q();
              }
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
              tma_load_4d(&tm_k, &k_full[st], wsm + PtSmem::kK + off, 0, row, it.h, page);
              tma_load_4d(&tm_v, &v_full[st], wsm + PtSmem::kV + off, 0, row, it.h, page);
            });
        if (ok && !q_sent) {
          if (n > 0) ok = load_q();
          if (ok) send_q();
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    } else {
      // ---------------- UMMA issuer ----------------
      if (elect_one()) {
        constexpr uint32_t idesc_qk = idesc_f16(128, 128, false, false, kBF16);
        constexpr uint32_t idesc_pv = idesc_f16(128, 64, false, true, kBF16);
        const uint64_t qdesc = sw128_desc(wbase + PtSmem::kQ, 16, 1024);
        bool ok = true, first = false, pending = false;
        int J = 0, pn = 0;
        // O += P V of tile J - 1, then release its K/V stage; the first one of item pn overwrites
        // O, after the epilogue of the item before has read it
        auto issue_pv = [&]() {
          const int j = J - 1, st = j % kPtStages;
          pending = false;
          ok = ok && mbar_wait(&v_full[st], (j / kPtStages) & 1);
          if (ok && first && pn > 0) ok = mbar_wait(o_free, (pn - 1) & 1);
          ok = ok && mbar_wait(p_full, j & 1);
          if (!ok) return;
          tc_fence_after();
          const uint64_t vdesc = sw128_desc(wbase + PtSmem::kV + st * kTile16, kTile16, 1024);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ts(tmem + 384 + x * 64, tmem + 256 + x * 64 + kk * 8, vdesc + ((kk * 2048) >> 4),
                    idesc_pv, (!first || kk > 0) ? 1u : 0u);
          umma_commit(o_done);
          umma_commit(&kv_empty[st]);
        };
        for (int n = 0; ok && paged_next<kPtBM, kPtBN, kPtItemCost>(p, cur, it); ++n) {
          // S of a tile goes before O += P V of the one before it, so that it is ready when that
          // tile's softmax ends; at an item's start only if its Q and K are there already
          if (pending && !(mbar_test(q_full, n & 1) &&
                           mbar_test(&k_full[J % kPtStages], (J / kPtStages) & 1)))
            issue_pv();
          ok = ok && mbar_wait(q_full, n & 1);
          for (int t = it.t0; ok && t < it.t1; ++t) {
            const int st = J % kPtStages;
            ok = mbar_wait(&k_full[st], (J / kPtStages) & 1);
            if (ok && J > 0) ok = mbar_wait(s_free, (J - 1) & 1);  // S is in registers
            if (!ok) break;
            tc_fence_after();
            const uint64_t kdesc = sw128_desc(wbase + PtSmem::kK + st * kTile16, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_ss(tmem + x * 128, qdesc + ((kk * 32) >> 4), kdesc + ((kk * 32) >> 4), idesc_qk,
                      kk > 0 ? 1u : 0u);
            umma_commit(s_full);
            if (t == it.t1 - 1) umma_commit(q_empty);
            if (pending) issue_pv();
            ++J;
            pending = true;
            first = t == it.t0;
            pn = n;
          }
        }
        if (ok && pending) issue_pv();
      }
      __syncwarp();
    }
  } else {
    // ---------------- softmax ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPtRegsSoftmax));
    // TMEM lane t holds row t of worker 0's tiles and row t ^ 64 of worker 1's, so that the rows of
    // two short items (64 or fewer) keep all four of the SM's sub-partitions busy
    const int lane128 = threadIdx.x & 127, row = lane128 ^ (64 * x);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_base + x * 128;
    const uint32_t tP = tmem + lane_base + 256 + x * 64;
    const uint32_t tO = tmem + lane_base + 384 + x * 64;
    int* const last_flag = reinterpret_cast<int*>(smem + PtSmem::kLast) + x;
    bool ok = true;
    int J = 0;  // key tiles consumed so far
    PagedItem next;
    for (bool more = paged_next<kPtBM, kPtBN, kPtItemCost>(p, cur, next); more;) {
      it = next;
      const int rows = it.s.qn * p.G, r = it.i * kPtBM + row;
      const bool live = r < rows;
      const int tok = live ? p.by_G.div(r) : 0;
      const int row_hi = live ? paged_hi(p, it.s, tok) : 0;
      const int full_all = paged_hi(p, it.s, p.by_G.div(it.i * kPtBM));  // seen by every row
      const bool dead = !__any_sync(0xffffffffu, live);  // a warp without rows computes nothing
      float m_run = -INFINITY, l_run = 0.f;
      for (int t = it.t0; t < it.t1; ++t, ++J) {
        const int s = t * kPtBN;
        ok = mbar_wait_warp(s_full, J & 1);
        if (!ok) break;
        tc_fence_after();
        if (dead) {  // (the P and O rows of a dead warp are never read)
          tc_fence_before();
          mbar_arrive(s_free);
          // as the other warps do: an arrival for this P before the last one is complete would
          // count for the last one
          if (t > it.t0) ok = mbar_wait_warp(o_done, (J - 1) & 1);
          if (!ok) break;
        } else {
          const bool masked = s + kPtBN > full_all;
          const int hi = masked ? row_hi - s : kPtBN;  // this row sees columns [0, hi)
          uint32_t vis = 0;  // 32-column chunks that some row of the warp sees
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (__any_sync(0xffffffffu, hi > 32 * c)) vis |= 1u << c;
          float xs[128];
          uint32_t u[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32_async(tS + c * 32, u[c]);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            reg_fence(u[c]);
#pragma unroll
            for (int k = 0; k < 32; ++k) xs[c * 32 + k] = __uint_as_float(u[c][k]);
          }
          tc_fence_before();
          mbar_arrive(s_free);  // S is in registers: the next one may be computed
          const float mx = max3(chunk_max<0>(xs, vis, masked, 0, hi),
                                chunk_max<1>(xs, vis, masked, 0, hi),
                                fmaxf(chunk_max<2>(xs, vis, masked, 0, hi),
                                      chunk_max<3>(xs, vis, masked, 0, hi))) *
                           p.scale_log2;
          float alpha = 1.f;
          bool up = false;
          const float m_new = fmaxf(m_run, mx);
          if (m_new - m_run > kRescaleLog2) {  // false for NaN (-inf - -inf)
            alpha = ex2(m_run - m_new);        // 0 when m_run = -inf
            up = t > it.t0;
            m_run = m_new;
          }
          const bool rescale = __any_sync(0xffffffffu, up);
          const float m_use = m_run == -INFINITY ? 0.f : m_run;
          const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
          const float2 nm2 = make_float2(-m_use, -m_use);
          float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                           make_float2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
            if (vis & (1u << c)) {
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const int gi = c * 16 + k;  // column pair of the row
                const float2 z = __ffma2_rn(make_float2(xs[2 * gi], xs[2 * gi + 1]), sc2, nm2);
                const float2 e = make_float2(ex2(z.x), ex2(z.y));
                acc[k & 3] = __fadd2_rn(acc[k & 3], e);
                pk[k] = pack2<kBF16>(e.x, e.y);
              }
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k) pk[k] = 0u;
            }
            if (c == 0 && t > it.t0) {
              ok = mbar_wait_warp(o_done, (J - 1) & 1);  // the P of the tile before is used up
              tc_fence_after();
            }
            tmem_st16(tP + c * 16, pk);
          }
          l_run *= alpha;
          if (!ok) break;
          const float2 a01 = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
          l_run += a01.x + a01.y;
          if (rescale) {  // rows that do not need it multiply by 1
            tmem_ld32_async(tO, u[0]);
            tmem_ld32_async(tO + 32, u[1]);
            tmem_ld_wait();
#pragma unroll
            for (int c2 = 0; c2 < 2; ++c2) {
              reg_fence(u[c2]);
#pragma unroll
              for (int k = 0; k < 32; ++k)
                u[c2][k] = __float_as_uint(__uint_as_float(u[c2][k]) * alpha);
              tmem_st32(tO + c2 * 32, u[c2]);
            }
          }
          tmem_st_wait();
        }
        if (it.hi - s < kPtBN) {
          // Rows of V past the visible keys hold what the page holds there, NaN included, and
          // P = 0 does not cancel that: zero them before P V.
          const int st = J % kPtStages;
          ok = mbar_wait_warp(&v_full[st], (J / kPtStages) & 1);
          if (!ok) break;
          if (lane128 >= it.hi - s) {
            uint8_t* v = wsm + PtSmem::kV + st * kTile16 + lane128 * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(v + 16 * c) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        mbar_arrive(p_full);
      }
      more = paged_next<kPtBM, kPtBN, kPtItemCost>(p, cur, next);  // (while the last P V runs)
      // ---- the share's end: the last O += P V has landed; O / l, or the share's partial ----
      if (ok) ok = mbar_wait_warp(o_done, (J - 1) & 1);
      if (!bar_and(1 + x, 128, ok)) break;
      tc_fence_after();
      float o[64], L = l_run, M = m_run;
      {
        uint32_t u[2][32];
        tmem_ld32_async(tO, u[0]);
        tmem_ld32_async(tO + 32, u[1]);
        tmem_ld_wait();
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          reg_fence(u[c2]);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[c2 * 32 + k] = __uint_as_float(u[c2][k]);
        }
      }
      tc_fence_before();
      mbar_arrive(o_free);  // O is in registers: the next item may overwrite it
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
        // the share that finishes last merges the item's partials, in list order
        asm volatile("bar.sync %0, 128;" ::"r"(1 + x) : "memory");
        if (lane128 == 0) *last_flag = paged_finish(p, it);
        asm volatile("bar.sync %0, 128;" ::"r"(1 + x) : "memory");
        if (*last_flag == 0) continue;
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
              L == 0.f ? -INFINITY
                       : ((M == -INFINITY ? 0.f : M) + log2f(L)) * 0.69314718055994530942f;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 10) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace bd3
