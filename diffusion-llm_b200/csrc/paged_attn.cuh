// Attention of few new rows per sequence over a paged KV cache (sm_100a): the denoising step's
// block of tokens, single tokens with grouped heads. paged_sched.cuh has the layout, the visible
// keys and the distribution of work; this is the kernel for row tiles of 16 kMB rows.
//
//   O_r = sum_c p_rc V_c / sum_c p_rc,  p_rc = 2^(scale log2(e) q_r . k_c - m_r),
// over the keys c < hi(r), in one pass with the running maximum m and sum l of each row; a row
// without keys gets O = 0 and LSE = -inf. Scores, m, l and O are fp32; P is rounded to the
// inputs' type as the operand of the P V product (what the tensor cores take).
//
// 16 to 32 rows do 16 to 32 FLOP per byte of K and V, so DRAM bounds it: a producer warp keeps a
// ring of 64-key K/V tiles full with TMA (one box per page piece, page ids looked up 32 pieces
// ahead so that no tile waits for a dependent load), and four consumer warps take 16 keys of
// each tile through mma.sync m16n8k16 (16 rows are far below tcgen05's 64-row minimum, and the
// tensor cores are nowhere near the bound). Each warp has its own (m, l, O); they are merged in
// shared memory at the end of the share. Two CTAs an SM keep 160 KB of loads in flight. (Their ten
// warps put three on a sub-partition, which caps a thread at 168 registers: enough for 16 rows; at
// 32 rows ptxas spills 96 bytes a thread.)
// Measured: 32 sequences of 1K to 16K positions, 12 heads, 16 rows each, 74 us (5.7 TB/s, 0.87 of
// the copy rate); 64 single tokens of 32 heads over 8 KV heads, 1 to 8192 positions, 24 us
// (3.3 TB/s: most of its 512 items are short and pay their fixed 2 to 3 us a share); one
// sequence's 16-token block over 1056 positions 9.6 us, most of it launch, one pass of loads and
// the merge.
#pragma once

#include "decode.cuh"
#include "paged_sched.cuh"

namespace bd3 {

constexpr int kPgBN = 64;                      // keys per tile
constexpr int kPgThreads = 160;                // 4 consumer warps + 1 producer warp
constexpr int kPgItemCost = 4;                 // an item's fixed cost in tiles (1 to 9 measured)
constexpr uint32_t kPgTile = kPgBN * 128u;     // 64 keys x 128 B

template <int kMB>
struct PgSmem {
  static constexpr int kRows = 16 * kMB;
  static constexpr int kStages = kMB == 1 ? 5 : 4;  // two CTAs an SM
  static constexpr uint32_t kRing = 0;              // K then V, per stage
  static constexpr uint32_t kO = kRing + kStages * 2 * kPgTile;  // [4][kRows][64] warps' O
  static constexpr uint32_t kML = kO + 4 * kRows * 64 * 4;       // [2][4][kRows] their m, l
  static constexpr uint32_t kBar = kML + 2 * 4 * kRows * 4;      // full[S], empty[S]
  static constexpr uint32_t kScan = kBar + 2 * kStages * 8;
  static constexpr uint32_t kLast = kScan + sizeof(PagedScan);
  static constexpr uint32_t kBytes = kLast + 16;
  static constexpr uint32_t kAlloc = kBytes + 1024;  // room to align the base to 1 KB
};

// Barrier `id` of `threads` threads that ANDs their `ok`: all go on, or none does.
__device__ __forceinline__ bool bar_and(int id, int threads, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, %2, %3, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok)), "r"(id), "r"(threads)
      : "memory");
  return all != 0;
}

// Store 8 consecutive output values of one row.
template <bool kBF16>
__device__ __forceinline__ void paged_store8(const PagedParams& p, long long off,
                                             const float (&o)[8]) {
  if (p.out_f32) {
    float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.o) + off);
    dst[0] = make_float4(o[0], o[1], o[2], o[3]);
    dst[1] = make_float4(o[4], o[5], o[6], o[7]);
  } else {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.o) + off) =
        make_uint4(pack2<kBF16>(o[0], o[1]), pack2<kBF16>(o[2], o[3]), pack2<kBF16>(o[4], o[5]),
                   pack2<kBF16>(o[6], o[7]));
  }
}

template <int kMB, bool kBF16>
__global__ void __launch_bounds__(kPgThreads, 2)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ PagedParams p) {
  using S = PgSmem<kMB>;
  constexpr int kRows = S::kRows;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* empty = full + S::kStages;
  PagedScan* scan = reinterpret_cast<PagedScan*>(smem + S::kScan);
  int* last_flag = reinterpret_cast<int*>(smem + S::kLast);
  const int warp = static_cast<int>(warp_id());
  const int lane = static_cast<int>(lane_id());

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // the lengths, the new rows of the cache and the workspace come from the kernels before
  griddep_wait();
  griddep_launch_dependents();
  PagedCursor cur = paged_chunk<kPgThreads, 1, kRows, kPgBN, kPgItemCost>(p, scan, 0);  // (its barriers cover the init)
  PagedItem it;

  if (warp == 4) {
    // ---------------- producer ----------------
    int J = 0;
    bool ok = true;
    while (ok && paged_next<kRows, kPgBN, kPgItemCost>(p, cur, it)) {
      ok = paged_stream<kPgBN>(
          p, it, J,
          [&](int j) {
            const int st = j % S::kStages;
            if (j >= S::kStages && !mbar_wait_warp(&empty[st], ((j / S::kStages) - 1) & 1))
              return false;
            if (lane == 0) mbar_expect_tx(&full[st], 2 * kPgTile);
            return true;
          },
          [&](int j, int piece, int page, int row) {
            const int st = j % S::kStages;
            uint8_t* dst = smem + S::kRing + st * 2 * kPgTile + piece * p.box * 128;
            tma_load_4d(&tm_k, &full[st], dst, 0, row, it.h, page);
            tma_load_4d(&tm_v, &full[st], dst + kPgTile, 0, row, it.h, page);
          });
    }
    return;
  }

  // ---------------- consumers: warp w takes keys [16w, 16w+16) of every tile ----------------
  const int g = lane >> 2, tq = lane & 3;
  float* s_o = reinterpret_cast<float*>(smem + S::kO);
  float* s_m = reinterpret_cast<float*>(smem + S::kML);
  float* s_l = s_m + 4 * kRows;
  int J = 0;
  bool ok = true;
  while (paged_next<kRows, kPgBN, kPgItemCost>(p, cur, it)) {
    const int rows = it.s.qn * p.G, r0 = it.i * kRows;
    uint32_t qa[kMB][4][4];  // A fragments: m-block, k-step (16 of the 64 dims), regs
    int row_hi[kMB][2];
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        const int r = r0 + mb * 16 + g + 8 * hr;
        const bool live = r < rows;
        const int t = live ? p.by_G.div(r) : 0;
        row_hi[mb][hr] = live ? paged_hi(p, it.s, t) : 0;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) +
                              (it.s.q0 + t) * p.q_st + (it.h * p.G + (r - t * p.G)) * p.q_sh + 2 * tq;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          qa[mb][ks][hr] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * ks) : 0u;
          qa[mb][ks][2 + hr] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 8) : 0u;
        }
      }
    const int full_all = paged_hi(p, it.s, p.by_G.div(r0));  // keys below this are seen by every row

    float acc[kMB][8][4], m_run[kMB][2], l_run[kMB][2];
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb) {
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[mb][nt][i] = 0.f;
      m_run[mb][0] = m_run[mb][1] = -INFINITY;
      l_run[mb][0] = l_run[mb][1] = 0.f;
    }

    for (int t = it.t0; ok && t < it.t1; ++t, ++J) {
      const int st = J % S::kStages;
      ok = mbar_wait_warp(&full[st], (J / S::kStages) & 1);
      if (!ok) break;
      const uint32_t sk = sbase + S::kRing + st * 2 * kPgTile;
      // Rows of the page past the visible keys hold anything, NaN included, and P = 0 does not
      // cancel that: V's count as zero.
      dec_tile_step<kMB, kBF16, true>(sk, sk + kPgTile, &empty[st], warp, lane, t * kPgBN, full_all,
                                      row_hi, qa, acc, m_run, l_run, p.scale_log2, it.hi);
    }

    // ---- merge the four warps' states (each row's sum is still spread over its quad) ----
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        float l = l_run[mb][hr];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int r = mb * 16 + g + hr * 8;
        if (tq == 0) {
          s_m[warp * kRows + r] = m_run[mb][hr];
          s_l[warp * kRows + r] = l;
        }
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
          *reinterpret_cast<float2*>(&s_o[(warp * kRows + r) * 64 + nt * 8 + 2 * tq]) =
              make_float2(acc[mb][nt][2 * hr], acc[mb][nt][2 * hr + 1]);
      }
    if (!bar_and(1, 128, ok)) return;  // a wait ran out (status bit 1 is set)
    float* const slot = p.partials + static_cast<long long>(it.slot) * (kRows * 66);
    for (int idx = threadIdx.x; idx < kRows * 8; idx += 128) {
      const int rl = idx >> 3, c8 = (idx & 7) * 8;
      const int r = r0 + rl;
      if (r >= rows) continue;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w * kRows + rl]);
      const float M_use = M == -INFINITY ? 0.f : M;
      float L = 0.f, o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float sc = ex2(s_m[w * kRows + rl] - M_use);  // 0 for a warp that saw no key
        L += sc * s_l[w * kRows + rl];
        const float4* src = reinterpret_cast<const float4*>(&s_o[(w * kRows + rl) * 64 + c8]);
        const float4 a = src[0], b = src[1];
        o[0] += sc * a.x; o[1] += sc * a.y; o[2] += sc * a.z; o[3] += sc * a.w;
        o[4] += sc * b.x; o[5] += sc * b.y; o[6] += sc * b.z; o[7] += sc * b.w;
      }
      if (it.parts > 1) {
        if (c8 == 0) {
          slot[rl] = M;
          slot[kRows + rl] = L;
        }
        float4* dst = reinterpret_cast<float4*>(slot + 2 * kRows + rl * 64 + c8);
        dst[0] = make_float4(o[0], o[1], o[2], o[3]);
        dst[1] = make_float4(o[4], o[5], o[6], o[7]);
        continue;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;  // L = 0: a row without keys
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] *= inv;
      const int t = p.by_G.div(r), hq = it.h * p.G + (r - t * p.G);
      paged_store8<kBF16>(p, (it.s.q0 + t) * p.o_st + hq * p.o_sh + c8, o);
      if (p.lse != nullptr && c8 == 0)
        p.lse[static_cast<long long>(it.s.q0 + t) * (p.Hkv * p.G) + hq] =
            L == 0.f ? -INFINITY : (M_use + log2f(L)) * 0.69314718055994530942f;
    }
    if (it.parts > 1) {
      // the share that finishes last merges the item's partials, in CTA order
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (threadIdx.x == 0) *last_flag = paged_finish(p, it);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (*last_flag) {
        for (int idx = threadIdx.x; idx < kRows * 8; idx += 128) {
          const int rl = idx >> 3, c8 = (idx & 7) * 8;
          const int r = r0 + rl;
          if (r >= rows) continue;
          float M = -INFINITY, L = 0.f, o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = 0.f;
#pragma unroll 4
          for (int j = 0; j < it.parts; ++j) {
            const float* src = p.partials + static_cast<long long>(paged_part_slot(it, j)) * (kRows * 66);
            const float m = __ldcg(src + rl), l = __ldcg(src + kRows + rl);
            const float4* so = reinterpret_cast<const float4*>(src + 2 * kRows + rl * 64 + c8);
            const float4 a = __ldcg(so), b = __ldcg(so + 1);
            const float m_new = fmaxf(M, m), mu = m_new == -INFINITY ? 0.f : m_new;
            const float u = ex2(M - mu), w = ex2(m - mu);
            M = m_new;
            L = L * u + l * w;
            o[0] = o[0] * u + a.x * w; o[1] = o[1] * u + a.y * w;
            o[2] = o[2] * u + a.z * w; o[3] = o[3] * u + a.w * w;
            o[4] = o[4] * u + b.x * w; o[5] = o[5] * u + b.y * w;
            o[6] = o[6] * u + b.z * w; o[7] = o[7] * u + b.w * w;
          }
          const float M_use = M == -INFINITY ? 0.f : M;
          const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] *= inv;
          const int t = p.by_G.div(r), hq = it.h * p.G + (r - t * p.G);
          paged_store8<kBF16>(p, (it.s.q0 + t) * p.o_st + hq * p.o_sh + c8, o);
          if (p.lse != nullptr && c8 == 0)
            p.lse[static_cast<long long>(it.s.q0 + t) * (p.Hkv * p.G) + hq] =
                L == 0.f ? -INFINITY : (M_use + log2f(L)) * 0.69314718055994530942f;
        }
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");  // s_o, s_m, s_l and the flag are free again
  }
}

}  // namespace bd3
