// Work distribution of attention over a paged KV cache (sm_100a), shared by its two kernels.
//
// The new tokens of all sequences are packed; sequence b has the rows [cu_q[b], cu_q[b+1]) and
// they are the last of its kv_lens[b] positions. A token at position p sees the keys
// [0, min((p / bs + 1) * bs, kv_len)): block-causal attention, causal for bs = 1. The G = Hq/Hkv
// query heads that share a KV head are folded into the row index, r = token * G + g, so a
// KV head's keys are read once for all of them.
//
// Work is a list of items (sequence b, row tile i, KV head h), each with n(b, i) key tiles, laid
// end to end in that order; an item also counts kItemCost tiles for what it costs whatever its
// length (finding it, its Q rows, its epilogue). W is the list's length. The lengths live on
// the device (a captured launch serves every step of a growing batch), so each CTA computes
// the prefix sums itself: the threads add up their share of the (b, i) pairs, a block scan
// gives every share's start. Worker w (a CTA, or one of its independent halves) then takes
// [w * chunk, (w + 1) * chunk) of the list, chunk = ceil(W / workers) (more for a few long items): the
// same work for every worker whatever the mix of lengths, so one 64K-token sequence among
// short ones does not set the time.
// An item cut by chunk borders leaves one partial (m, l, unnormalised O) per worker in the
// workspace; the worker that finishes last (an atomic count per cut item) merges the partials
// in list order, so the order of the sums does not depend on timing. Nothing waits for another
// worker. The counts are zero before the first call (the caller's zeroed workspace) and the
// merging worker sets its count back to zero, so calls in stream order share one workspace.
#pragma once

#include "common.cuh"
#include "tile_ranges.h"

namespace bd3 {

// Division of 0 <= x < 2^31 by a launch constant d, as a multiplication (Granlund and Montgomery,
// "Division by invariant integers using multiplication", PLDI 1994): with l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d) < 2^32, m d - 2^(31 + l) < 2^l, so floor(x m / 2^(31 + l)) = floor(x / d).
struct FastDiv {
  uint32_t m, s;  // s = l - 1; d = 1: m = 0
  __host__ static FastDiv of(uint32_t d) {
    if (d == 1) return FastDiv{0, 0};
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    return FastDiv{static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d), l - 1};
  }
  __device__ __forceinline__ int div(int x) const {
    return m == 0 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), m) >> s);
  }
};

struct PagedParams {
  const void* q;              // (total_q, Hq, 64); token and head strides in elements
  void* o;                    // (total_q, Hq, 64) in the output dtype
  float* lse;                 // optional (total_q, Hq) contiguous natural-log LSE
  long long q_st, q_sh, o_st, o_sh;
  const int* page_table;      // (B, max_pages): page of positions [j * page_size, ...)
  long long pt_stride;
  const int* kv_lens;         // (B)
  const int* cu_q;            // (B + 1)
  int* counters;              // 2 per worker, zero between calls
  float* partials;            // 2 slots per worker of (m, l, O) of a row tile
  int B, Hkv, G, total_q, max_q;
  int num_pages, page_size, max_pages;
  int box;                    // rows of one TMA piece: divides the page size and the key tile
  int bs;
  FastDiv by_G, by_bs, by_page;  // by G, bs and page_size
  int row_tiles;              // row tiles of max_q tokens
  int out_f32;
  float scale_log2;           // softmax scale * log2(e)
};

// Sequence b as the kernels use it: its first packed row, its new tokens and its keys. Values
// outside the call's own bounds are cut to them (no address depends on the uncut ones).
struct PagedSeq {
  int q0, qn, kv;
  bool bad;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
  const int a = p.cu_q[b], e = p.cu_q[b + 1], kv = p.kv_lens[b];
  const long long cap = static_cast<long long>(p.max_pages) * p.page_size;
  PagedSeq s;
  s.q0 = imin(a < 0 ? 0 : a, p.total_q);
  s.qn = e > s.q0 ? imin(e, p.total_q) - s.q0 : 0;
  s.qn = s.qn < 0 ? 0 : imin(s.qn, p.max_q);
  s.kv = kv < 0 ? 0 : (kv > cap ? static_cast<int>(cap) : kv);
  s.bad = s.q0 != a || s.qn != e - a || s.kv != kv;
  return s;
}

// Exclusive end of the keys that new token t of the sequence sees (0: none).
__device__ __forceinline__ int paged_hi(const PagedParams& p, const PagedSeq& s, int t) {
  const int pos = s.kv - s.qn + t;
  if (pos < 0) return 0;
  const long long hi = (static_cast<long long>(p.by_bs.div(pos)) + 1) * p.bs;
  return hi < s.kv ? static_cast<int>(hi) : s.kv;
}

// Key tiles of row tile i: up to the last key that its last row sees; 0 past the sequence's rows
// and 1 for rows that see no key (their output is written too).
template <int kBM, int kBN>
__device__ __forceinline__ int paged_tiles(const PagedParams& p, const PagedSeq& s, int i,
                                           int* hi_out) {
  const int rows = s.qn * p.G, r0 = i * kBM;
  if (r0 >= rows) return 0;
  const int hi = paged_hi(p, s, p.by_G.div(imin(r0 + kBM, rows) - 1));
  *hi_out = hi;
  return hi > kBN ? (hi - 1) / kBN + 1 : 1;
}

// One worker's share of an item.
struct PagedItem {
  PagedSeq s;
  int b, i, h;
  int hi;         // exclusive end of the keys that any row of the item sees
  int t0, t1;     // key tiles of this share
  int parts;      // workers that share the item; 1: this one alone
  int slot;       // this share's partial
  int slot0;      // the first share's partial, and the item's count
  int w0;         // the first share's worker
  int n;          // key tiles of the item
};

struct PagedCursor {
  int w;                      // this worker
  int b, i;
  bool same;                  // the item holds the pair (b, i)'s s, n and hi already
  long long base;             // list position of the pair (b, i)
  long long pos, lo, end, chunk;
};

// The next share of this worker's chunk; false at its end.
template <int kBM, int kBN, int kItemCost>
__device__ __forceinline__ bool paged_next(const PagedParams& p, PagedCursor& c, PagedItem& it) {
  while (c.pos < c.end && c.b < p.B) {
    if (!c.same) {
      it.s = paged_seq(p, c.b);
      it.n = paged_tiles<kBM, kBN>(p, it.s, c.i, &it.hi);
      if (it.n == 0) {  // past the sequence's rows
        ++c.b;
        c.i = 0;
        continue;
      }
      c.same = true;
    }
    const int n = it.n;
    const int cost = n + kItemCost;
    const long long w = static_cast<long long>(cost) * p.Hkv;
    if (c.pos >= c.base + w) {
      c.base += w;
      c.same = false;
      if (++c.i == p.row_tiles) {
        ++c.b;
        c.i = 0;
      }
      continue;
    }
    it.b = c.b;
    it.i = c.i;
    it.h = static_cast<int>(c.pos - c.base) / cost;  // (the host bounds cost * Hkv)
    const long long first = c.base + static_cast<long long>(it.h) * cost + kItemCost;  // tile 0
    const long long stop = first + n < c.end ? first + n : c.end;
    const long long from = c.pos > first ? c.pos : first;
    c.pos = stop > c.pos ? stop : c.end;
    if (stop <= first) continue;  // only the item's fixed cost falls into this chunk
    it.t0 = static_cast<int>(from - first);
    it.t1 = static_cast<int>(stop - first);
    // the workers of the item's first and last tile, counted from this one (32-bit divisions:
    // a 64-bit one costs hundreds of cycles, and every role of a worker does this per share)
    const uint32_t chunk = c.chunk < 0x7FFFFFFF ? static_cast<uint32_t>(c.chunk) : 0x7FFFFFFFu;
    const int before = c.lo > first ? static_cast<int>((static_cast<uint32_t>(c.lo - first) + chunk - 1u) / chunk) : 0;
    const int after = first + n > c.end ? static_cast<int>(static_cast<uint32_t>(first + n - 1 - c.lo) / chunk) : 0;
    it.w0 = c.w - before;
    it.parts = before + after + 1;
    it.slot0 = 2 * it.w0 + (first == c.lo - before * c.chunk ? 0 : 1);
    it.slot = 2 * c.w + (from == c.lo ? 0 : 1);
    return true;
  }
  return false;
}
// Count one more finished share of a cut item; true for the last one. For one thread, after a barrier
// behind every thread's stores of the partial; release and acquire at device scope.
__device__ __forceinline__ bool paged_finish(const PagedParams& p, const PagedItem& it) {
  int before;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;"
               : "=r"(before)
               : "l"(&p.counters[it.slot0])
               : "memory");
  if (before != it.parts - 1) return false;
  p.counters[it.slot0] = 0;
  return true;
}
// Partial slot of share j of an item.
__device__ __forceinline__ int paged_part_slot(const PagedItem& it, int j) {
  return j == 0 ? it.slot0 : 2 * (it.w0 + j);
}

struct PagedScan {
  long long warp_sum[18];
  long long base[3];
  int b[3], i[3];
};

// The chunk of worker kWorkers * blockIdx.x + x, found by all kThreads threads of the CTA for all
// its workers at once; ends with a barrier. The chunk is empty for a worker past the list.
template <int kThreads, int kWorkers, int kBM, int kBN, int kItemCost>
__device__ __forceinline__ PagedCursor paged_chunk(const PagedParams& p, PagedScan* sc, int x) {
  static_assert(kThreads <= 576 && kWorkers <= 3, "PagedScan");
  const int pairs = p.B * p.row_tiles;
  const int per = cdiv(pairs, kThreads);
  const int e0 = imin(static_cast<int>(threadIdx.x) * per, pairs), e1 = imin(e0 + per, pairs);
  auto cost = [&](int e, int b) -> long long {
    const PagedSeq s = paged_seq(p, b);
    if (s.bad && blockIdx.x == 0) atomicOr(&g_bd3_status, kStatusBadLaunch);
    int hi;
    const int n = paged_tiles<kBM, kBN>(p, s, e - b * p.row_tiles, &hi);
    return n == 0 ? 0 : static_cast<long long>(n + kItemCost) * p.Hkv;
  };
  long long mine = 0;
  for (int e = e0; e < e1; ++e) mine += cost(e, e / p.row_tiles);
  const int lane = static_cast<int>(lane_id()), w = static_cast<int>(threadIdx.x) >> 5;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) sc->warp_sum[w] = incl;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int k = 0; k < kThreads / 32; ++k) {
    if (k == w) before = total;
    total += sc->warp_sum[k];
  }
  const long long workers = static_cast<long long>(gridDim.x) * kWorkers;
  PagedCursor c;
  c.chunk = (total + workers - 1) / workers;
  // not below half the root of the mean item: a long item cut into hundreds of shares would wait
  // for the merge of as many partials (8 heads over one KV head of 60004 positions: one token 38
  // us in 296 shares, 20 so; four tokens 70 and 36; 16 tokens, the large kernel's, 112 and 49)
  const int least = static_cast<int>(0.5f * sqrtf(static_cast<float>(total) / (static_cast<float>(pairs) * p.Hkv)));
  if (c.chunk < least) c.chunk = least;
  if (c.chunk < 1) c.chunk = 1;
#pragma unroll
  for (int k = 0; k < kWorkers; ++k) {
    const long long lo = c.chunk * (static_cast<long long>(blockIdx.x) * kWorkers + k);
    long long at = before + incl - mine;
    if (lo >= at && lo < at + mine) {  // this thread's share holds the chunk's start
      for (int e = e0; e < e1; ++e) {
        const int b = e / p.row_tiles;
        const long long n = cost(e, b);
        if (lo < at + n) {
          sc->base[k] = at;
          sc->b[k] = b;
          sc->i[k] = e - b * p.row_tiles;
          break;
        }
        at += n;
      }
    }
  }
  __syncthreads();
  c.w = static_cast<int>(blockIdx.x) * kWorkers + x;
  c.lo = c.chunk * c.w;
  c.end = c.lo + c.chunk < total ? c.lo + c.chunk : total;
  c.pos = c.lo;
  c.base = sc->base[x];
  c.b = c.lo < c.end ? sc->b[x] : p.B;
  c.i = sc->i[x];
  c.same = false;
  return c;
}

// Pages of the kBN / box pieces of key tiles, looked up by a whole warp ahead of their use: lane
// l holds piece l % pieces of tile l / pieces of a batch of 32 / pieces tiles. Pieces past the
// visible keys get page num_pages, which is outside the tensor map: the TMA fills their rows
// with zeros and reads nothing. A page id outside [0, num_pages) is treated the same way and
// sets status bit 2.
template <int kBN>
__device__ __forceinline__ int paged_lookup(const PagedParams& p, const PagedItem& it, int tile,
                                            int* row) {
  const int pieces = kBN / p.box, lane = static_cast<int>(lane_id());
  const long long key = static_cast<long long>(tile + lane / pieces) * kBN + (lane % pieces) * p.box;
  *row = 0;
  if (key >= it.hi) return p.num_pages;
  const int pg = p.by_page.div(static_cast<int>(key));
  *row = static_cast<int>(key) - pg * p.page_size;
  const int id = p.page_table[it.b * p.pt_stride + pg];
  if (id < 0 || id >= p.num_pages) {
    atomicOr(&g_bd3_status, kStatusBadLaunch);
    return p.num_pages;
  }
  return id;
}

// Stream K and V pieces of the item's key tiles [t0, t1) into a ring, whole warp: wait(j) waits
// for the ring slot of tile j (false: gave up) and announces its bytes, issue(j, piece, page,
// row) loads one piece. J counts the tiles of all items.
template <int kBN, typename Wait, typename Issue>
__device__ __forceinline__ bool paged_stream(const PagedParams& p, const PagedItem& it, int& J,
                                             Wait&& wait, Issue&& issue) {
  const int pieces = kBN / p.box, per = 32 / pieces, lane = static_cast<int>(lane_id());
  int row, row_next = 0, id_next = 0;
  int id = paged_lookup<kBN>(p, it, it.t0, &row);
  for (int t = it.t0; t < it.t1; t += per) {
    if (t + per < it.t1) id_next = paged_lookup<kBN>(p, it, t + per, &row_next);
    const int m = imin(per, it.t1 - t);
    for (int k = 0; k < m; ++k, ++J) {
      if (!wait(J)) return false;
      __syncwarp();
      if (lane / pieces == k) issue(J, lane % pieces, id, row);
    }
    id = id_next;
    row = row_next;
  }
  return true;
}

}  // namespace bd3
