// paged_draft.cuh - what a step with drafted tokens does around its attention:
// which rows of each tree the model's answers confirm (accept), the confirmed
// rows' keys and values moved up behind the cache in every layer (keep), and
// sequences that go on from another's cache (fork).
//
// All three move few bytes: the smallest calls are a launch and a chain of
// dependent loads, the largest forks are bound by HBM. Each is one launch for
// all sequences and all layers of a model.
#pragma once

#include "paged_append.cuh"
#include "paged_index.cuh"
#include "ptx.cuh"

namespace abft {

// ---- accept -------------------------------------------------------------------
// Row i of a tree is confirmed when it has no parent, or its parent p is
// confirmed and ids[i] == answers[p]. The deepest confirmed row (the lowest of
// equals) ends the path that is kept:
//   depth[i] = [i confirmed] (1 + depth[parent]),  0 otherwise.
// One CTA per sequence: all threads fetch rows (parent, id, the parent's
// answer: independent loads), the first warp resolves depths 32 rows at a time,
// parents of the same 32 by shuffles. Bound: a launch and four loads in a row
// (boundaries, parent, its answer, the last row's answer): 1 tree of 16 rows 2.1-2.5 us,
// 256 of up to 61 2.5-2.9 from a graph.
struct AcceptParams {
  const int32_t* cu;
  const int32_t* parents;
  const void *ids, *answers;
  int32_t* kept;
  int32_t* counts;
  void* next;
  uint32_t* status;
  int32_t tokens, batch;
};
constexpr int kAcceptThreads = 128;
constexpr int kAcceptHeld = 1024;  // rows in shared memory at a time
constexpr int kNotConfirmed = -2;  // in the place of a row's parent

template <typename Id>
__global__ void __launch_bounds__(kAcceptThreads) draft_accept_kernel(const AcceptParams p) {
  __shared__ int32_t s_up[kAcceptHeld];     // parent, or kNotConfirmed
  __shared__ int32_t s_depth[kAcceptHeld];  // of a tree that fits; of a larger one depths lie in `kept`
  __shared__ int32_t s_best, s_count;
  griddep_wait();
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  if (b == p.batch) {  // rows behind the last sequence, and a look at the boundaries
    const int end = p.batch > 0 ? p.cu[p.batch] : 0;
    for (int t = max(0, min(end, p.tokens)) + threadIdx.x; t < p.tokens; t += kAcceptThreads) p.kept[t] = -1;
    if (threadIdx.x < 32) check_boundaries(p.cu, p.batch, p.tokens, lane, p.status);
    return;
  }
  int begin, end;
  packed_range(p.cu, b, p.tokens, &begin, &end);
  const int n = end - begin;
  const Id* ids = static_cast<const Id*>(p.ids) + begin;
  const Id* answers = static_cast<const Id*>(p.answers) + begin;
  const int32_t* parents = p.parents + begin;
  int32_t* kept = p.kept + begin;
  int32_t* depth = n <= kAcceptHeld ? s_depth : kept;
  bool bad = false;
  int best = -1, most = 0;  // of this lane's rows (first warp)
  for (int c0 = 0; c0 < n; c0 += kAcceptHeld) {
    const int here = min(kAcceptHeld, n - c0);
    for (int r = threadIdx.x; r < here; r += kAcceptThreads) {
      const int i = c0 + r, up = parents[i];
      const bool ok = up >= -1 && up < i;
      bad = bad || !ok;
      s_up[r] = ok && (up < 0 || ids[i] == answers[up]) ? up : kNotConfirmed;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      for (int t0 = 0; t0 < here; t0 += 32) {
        const int r = t0 + lane, i = c0 + r;
        const int up = r < here ? s_up[r] : kNotConfirmed;
        const int near = up - (c0 + t0);  // the parent's lane when it is one of these 32 rows
        int d = up == -1 ? 1 : 0;
        bool open = up >= 0 && near >= 0;
        if (up >= 0 && near < 0) {
          // Between 0 and up + 1 whatever another sequence that claims the same rows has written there.
          const int above = max(0, min(depth[up], up + 1));
          d = above > 0 ? above + 1 : 0;
        }
        // Every round settles the rows whose parent is settled: the lowest open one at least.
        uint32_t left;
        while ((left = __ballot_sync(0xFFFFFFFFu, open)) != 0) {
          const int above = __shfl_sync(0xFFFFFFFFu, d, near & 31);
          if (open && !(left >> near & 1u)) {
            d = above > 0 ? above + 1 : 0;
            open = false;
          }
        }
        if (r < here) depth[i] = d;
        if (d > most) most = d, best = i;
        __syncwarp();
      }
    }
    __syncthreads();
  }
  if (bad && p.status != nullptr) atomicOr(p.status, ABFT_PAGED_BAD_DRAFT);
  if (threadIdx.x < 32) {
    const int top = __reduce_max_sync(0xFFFFFFFFu, most);
    const int row = __reduce_min_sync(0xFFFFFFFFu, most == top && top > 0 ? best : 0x7FFFFFFF);
    if (lane == 0) {
      s_best = row;
      s_count = top;
    }
    __syncwarp();
  }
  __syncthreads();
  const int count = s_count;
  // Depths are not needed any more: the rows' places in `kept` are written, each once.
  if (threadIdx.x == 0) {
    int at = s_best;
    for (int k = count - 1; k >= 0 && at >= 0 && at < n; --k) {
      kept[k] = at;
      const int up = n <= kAcceptHeld ? s_up[at] : parents[at];
      at = up < at ? up : -1;
    }
    p.counts[b] = count;
    static_cast<Id*>(p.next)[b] = count > 0 ? answers[s_best] : static_cast<Id>(-1);
  }
  for (int k = count + threadIdx.x; k < n; k += kAcceptThreads) kept[k] = -1;
}

// ---- keep -----------------------------------------------------------------------
// A model's pools: [layers][2] base addresses of keys and values (in the launch's
// parameters: nothing in memory has to outlive the call), which share
// one page table, one array of lengths and one geometry; or one layer's, in kv.
constexpr int kFewLayers = 64, kMostLayers = 512;  // of the two instances of each kernel
template <int kLayers>
struct LayerPools {
  uint16_t* pools[2 * kLayers];
  int32_t layers;
};

// Of sequence b's n new tokens (its last slots) the rows kept[0] < kept[1] < ...
// < kept[m - 1] move to the slots of rows 0 to m - 1, and its length becomes
// L - n + m. kept[i] >= i, so that in ascending order no row is overwritten
// before it has moved; a thread owns 16 bytes of a row in one layer and head
// and takes them through all rows in that order, four rows asked for before
// the first is written (row i + 3's source lies at or behind row i + 3). So no
// thread waits for another. A cluster of CTAs shares a sequence's layers: the
// length, which all of them read, is written when all have read it.
// Bound: a launch and five loads in a row (boundaries and length, kept rows, table,
// the rows); 28 layers of 4 heads of 128: 1 tree of 26 rows 3.3 us, 64 trees 5.4 (their
// bytes alone 1.4).
//
// A sequence with anything wrong (boundaries, count, rows that do not rise,
// length, pages) is left as it was.
template <int kLayers>
struct KeepParams {
  PagedView kv;
  LayerPools<kLayers> layers;
  const int32_t *cu, *kept, *counts;
  int32_t* lens_out;
  int32_t tokens;
  int32_t cluster;  // CTAs of a sequence
};
constexpr int kKeepThreads = 512;  // at most
constexpr int kKeepHeld = 256;  // rows whose places are in shared memory at a time
constexpr int kKeepCluster = 8;

template <int D, int kLayers>
__global__ void __launch_bounds__(kKeepThreads, 3) kv_keep_kernel(const __grid_constant__ KeepParams<kLayers> p) {
  // Where a row comes from (-1: it stays) and goes, in elements of head 0: in the
  // key pools, in the value pools.
  __shared__ longlong2 s_move[2][kKeepHeld];
  constexpr int kShift = D == 128 ? 7 : 6, kChunks = D / 8;
  griddep_wait();
  const int threads = blockDim.x;
  const PagedView& kv = p.kv;
  const int b = blockIdx.x / p.cluster, rank = blockIdx.x - b * p.cluster;
  int begin, end;
  packed_range(p.cu, b, p.tokens, &begin, &end);
  const int n = end - begin, m = p.counts[b], len = kv.seq_lens[b];
  uint32_t bad = 0;
  {
    const int lo = p.cu[b], hi = p.cu[b + 1];
    if (hi < lo || hi > p.tokens || lo < 0 || (b == 0 && lo != 0)) bad |= ABFT_PAGED_BAD_ROWS;
  }
  if (m < 0 || m > n) bad |= ABFT_PAGED_BAD_DRAFT;
  if (len < n || len > static_cast<int64_t>(kv.max_pages) << kv.page_shift) bad |= ABFT_PAGED_BAD_LEN;
  const int32_t* table = kv.page_table + b * kv.table_stride;
  const int base = len - n, page_mask = (1 << kv.page_shift) - 1;
  auto place = [&](int row, int* page, int* slot) {
    const int at = base + row;
    *page = table[at >> kv.page_shift];
    *slot = at & page_mask;
    return *page >= 0 && *page < kv.num_pages;
  };
  auto stage = [&](int i) {  // row i's move; what is wrong with it
    const int from = p.kept[begin + i], last = i > 0 ? p.kept[begin + i - 1] : -1;
    if (from <= last || from >= n || from < 0) return ABFT_PAGED_BAD_DRAFT;
    int page0, slot0, page1, slot1;
    const bool ok = place(from, &page0, &slot0) & place(i, &page1, &slot1);
#pragma unroll
    for (int values = 0; values < 2; ++values) {
      const int64_t stride = values ? kv.v_page_stride : kv.k_page_stride;
      longlong2 move;
      move.x = from == i ? -1 : paged_offset(page0, stride, 0, slot0, kv.page_shift, kShift);
      move.y = paged_offset(page1, stride, 0, slot1, kv.page_shift, kShift);
      s_move[values][i % kKeepHeld] = move;
    }
    return ok ? 0u : ABFT_PAGED_BAD_PAGE;
  };
  if (bad == 0)  // looks at all rows; those of a path that fits are staged for good
    for (int i = threadIdx.x; i < m; i += threads) bad |= stage(i);
  const bool wrong = __syncthreads_or(bad != 0);
  if (bad != 0 && rank == 0 && kv.status != nullptr) atomicOr(kv.status, bad);
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  if (!wrong) {
    const int columns = p.layers.layers * 2 * kv.kv_heads * kChunks;
    for (int i0 = 0; i0 < m; i0 += kKeepHeld) {
      const int here = min(kKeepHeld, m - i0);
      if (m > kKeepHeld) {
        __syncthreads();
        for (int i = threadIdx.x; i < here; i += threads) stage(i0 + i);
        __syncthreads();
      }
      for (int column = rank * threads + threadIdx.x; column < columns; column += p.cluster * threads) {
        const int c = column % kChunks, row = column / kChunks;
        const int head = row % kv.kv_heads, pool = row / kv.kv_heads, values = pool & 1;
        uint16_t* at = p.layers.pools[pool] + (static_cast<int64_t>(head) << kv.page_shift << kShift) + c * 8;
        const longlong2* moves = s_move[values];
        constexpr int kBatch = 4;
        for (int i = 0; i < here; i += kBatch) {
          uint4 x[kBatch];
#pragma unroll
          for (int k = 0; k < kBatch; ++k)
            if (i + k < here && moves[i + k].x >= 0) x[k] = *reinterpret_cast<const uint4*>(at + moves[i + k].x);
#pragma unroll
          for (int k = 0; k < kBatch; ++k)
            if (i + k < here && moves[i + k].x >= 0) *reinterpret_cast<uint4*>(at + moves[i + k].y) = x[k];
        }
      }
    }
  }
  if (p.cluster > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (rank == 0 && threadIdx.x == 0) p.lens_out[b] = wrong ? len : len - n + m;
}

// ---- fork -----------------------------------------------------------------------
// Pair i: sequence dst[i] becomes a copy of src[i]'s cache: its table row gets
// the source's full pages (shared from now on), its length the source's, and
// where that ends inside a page, pages[i] gets the slots of it and follows in
// the row. A pair with -1 for either is none.
//
// Pairs work side by side, so none may write what another reads or writes: a
// destination that is also a source or named twice, or a page named twice, is
// refused with all that name it, and so is a page that another pair copies from.
//
// Bound: HBM, by rest slots of 2 * layers * heads rows in and out; slots of a head lie
// one after another, and its warps take them in turn, eight 16-byte pieces a lane in
// flight (32 forks of 64 slots on average, 28 layers of 4 heads: 30.8 us, 6.7 TB/s).
// What the other pairs name and copy from is looked up beside the own chain of loads (3
// forks 2.7 us).
template <int kLayers>
struct ForkParams {
  PagedView kv;
  LayerPools<kLayers> layers;
  const int32_t *src, *dst, *pages;
  int32_t pairs;
  int32_t per_pair;  // CTAs of a pair: 2^shift warps for each head of each pool
  int32_t shift;
};
constexpr int kForkWarps = 8;

template <int D, int kLayers>
__global__ void __launch_bounds__(32 * kForkWarps) kv_fork_kernel(const __grid_constant__ ForkParams<kLayers> p) {
  constexpr int kShift = D == 128 ? 7 : 6;
  griddep_wait();
  const PagedView& kv = p.kv;
  const int i = blockIdx.x / p.per_pair, part = blockIdx.x - i * p.per_pair;
  const int s = p.src[i], d = p.dst[i], fresh = p.pages[i];
  if (s == -1 || d == -1) return;
  // Where a source's length ends: its full pages, and the slots behind them.
  auto ends = [&](int sequence, int* full, int* rest) {
    const int len = kv.seq_lens[sequence];
    *full = len >> kv.page_shift;
    *rest = len & ((1 << kv.page_shift) - 1);
    return len >= 0 && len <= static_cast<int64_t>(kv.max_pages) << kv.page_shift;
  };
  bool clash = false, same_page = false;
  for (int j = threadIdx.x; j < p.pairs; j += 32 * kForkWarps) {
    const int sj = p.src[j], dj = p.dst[j];
    if (sj == -1 || dj == -1) continue;
    clash = clash || sj == d || (j != i && dj == d);
    int full, rest;
    if (j == i || sj < 0 || sj >= kv.batch || !ends(sj, &full, &rest) || rest == 0) continue;  // needs no page
    same_page = same_page || p.pages[j] == fresh;
    if (sj != s) same_page = same_page || kv.page_table[sj * kv.table_stride + full] == fresh;  // (the own source's: below)
  }
  uint32_t bad = 0;
  if (s < 0 || s >= kv.batch || d < 0 || d >= kv.batch) bad = ABFT_PAGED_BAD_FORK;
  int full = 0, rest = 0, old = 0;
  if (bad == 0 && !ends(s, &full, &rest)) bad = ABFT_PAGED_BAD_LEN;
  if (bad == 0 && rest > 0) {
    old = kv.page_table[s * kv.table_stride + full];
    if (old < 0 || old >= kv.num_pages || fresh < 0 || fresh >= kv.num_pages || fresh == old) bad = ABFT_PAGED_BAD_PAGE;
  }
  if (clash || (same_page && rest > 0)) bad |= ABFT_PAGED_BAD_FORK;
  const bool wrong = __syncthreads_or(bad != 0);
  if (wrong) {
    if (bad != 0 && part == 0 && kv.status != nullptr) atomicOr(kv.status, bad);
    return;
  }
  if (part == 0) {
    const int32_t* from = kv.page_table + s * kv.table_stride;
    int32_t* to = const_cast<int32_t*>(kv.page_table) + d * kv.table_stride;
    for (int j = threadIdx.x; j < full; j += 32 * kForkWarps) to[j] = from[j];
    if (threadIdx.x == 0) {
      if (rest > 0) to[full] = fresh;
      const_cast<int32_t*>(kv.seq_lens)[d] = (full << kv.page_shift) + rest;
    }
  }
  const int lane = threadIdx.x & 31;
  const int items = p.layers.layers * 2 * kv.kv_heads;
  const int w = part * kForkWarps + (threadIdx.x >> 5), item = w >> p.shift, share = w & ((1 << p.shift) - 1);
  if (item >= items) return;
  const int head = item % kv.kv_heads, pool = item / kv.kv_heads, values = pool & 1;
  uint16_t* at = p.layers.pools[pool];
  const int64_t stride = values ? kv.v_page_stride : kv.k_page_stride;
  const uint4* from = reinterpret_cast<const uint4*>(at + paged_offset(old, stride, head, 0, kv.page_shift, kShift));
  uint4* to = reinterpret_cast<uint4*>(at + paged_offset(fresh, stride, head, 0, kv.page_shift, kShift));
  const int units = rest * (D / 8);
  constexpr int kBatch = 8;
  for (int u0 = share * 32 * kBatch + lane; u0 < units; u0 += 32 * kBatch << p.shift) {
    uint4 x[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (u0 + 32 * k < units) x[k] = __ldcs(from + u0 + 32 * k);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (u0 + 32 * k < units) to[u0 + 32 * k] = x[k];
  }
}

}  // namespace abft
