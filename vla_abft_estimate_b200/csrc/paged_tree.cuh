// paged_tree.cuh - attention of trees of drafted tokens over the paged cache.
//
// Row i of the n new tokens of a sequence of length L sees the slots before the
// new ones, its own and its ancestors':
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,   j < L - n  or  j - (L - n) in path(i).
// Parents come before their children, so a row sees no more than a causal one.
//
// Bound: trees are small (a tile of 128 rows holds the (token, head) rows of 18
// tokens of a group of 7) and caches long: every key and value is read once for a
// tile's rows, which the tensor cores take in faster than HBM gives it (32 KB of 64
// keys: 0.74 us of an SM's share of HBM, 0.4 us of products). What counts is that
// all SMs read all the time, and, for short caches, the chain of latencies. A step
// takes the issuing warp 1,400 cycles (heads of 64) to 1,700, and the row warps 1,370,
// which is what small tiles are bound by, with one CTA on an SM or two. (Shorter
// alone was either, and the whole no faster: rows of small tiles spread over idle warps,
// a part of the keys each, 770 cycles, but the warps' sums had to be added up, 12
// trees of up to 13 tokens of 32 heads 25.4 -> 30.7 us; a step's waits first and its
// products in one go, 800 cycles, 25.4 -> 25.6, 24 of up to 26 22.8 -> 23.2 with the
// join as it was then.)
//
// A CTA takes one tile of 128 rows of one kv head, in steps of 64 keys:
//   S = Q K^T   tcgen05.mma, S in TMEM, two of them: the next one is computed
//               while the rows work on the last
//   P = 2^(x - m) by one thread per row; over S, as 16-bit operand
//   O += P V    tcgen05.mma with P from TMEM
// with the running maximum, lagging rescaling and lift of paged_prefill.cuh. It uses
// half of an SM's registers, shared memory and TMEM: two CTAs an SM, of which one
// reads while the other begins, ends or changes its segment. (One CTA with two row
// groups on steps of 128 keys of the same segment, the causal kernel's form for few
// rows: 32 trees of 4 tokens of 32 heads on 512 slots 80 us, 54 so; up to 26 tokens on
// up to 4,122 slots 29, 20.9; 64 trees of 8 on 8,188 slots 198, 175, where HBM's time is
// 165.) One tree of 64 tokens on 131,008 slots takes 135-155 us (163 in a loop, at the
// power cap) where 73 are HBM's and the products' time: each of its four tiles takes in
// all keys and values by itself, 1.07 GB at the 62 GB/s that an SM takes in.
//
// Rounding: P has the 16 bits that the product takes, l sums it unrounded, O, m, l and
// the pieces have 32 (why: paged_prefill.cuh). Relative error against 64 bits 1.8-2.3e-3
// bf16 and 2.2e-4 fp16, of which the output's rounding alone is 1.6-1.7e-3 and 2.0e-4.
//
// Work: a call's steps over all (sequence, kv head, block of rows) segments are one
// list, cut into equal shares for two CTAs per SM. A segment inside a share is
// finished by its CTA; pieces of one that crosses CTAs are joined by a second, small
// kernel, in a fixed order. Short caches get a CTA or a cluster of CTAs per segment,
// whose sums meet in shared memory, in the one launch.
//
// Warps: 0-3 the rows (TMEM lane quadrant = warp), 4 TMA loads of pages into a ring
// of tiles, 5 the MMA issuer, 6 finds the work, 7 brings query rows and parents.
#pragma once

#include <cuda.h>

#include "paged_prefill.cuh"

namespace abft {

constexpr int kTreeRows = kPreRows;  // query rows of a tile
constexpr int kTreeKeys = 64;        // keys of a step
constexpr int kTreeThreads = 256;
// Parents of a tree that are held in shared memory, where a hop of the walk up takes a
// tenth of the time. A larger tree takes its steps from the last to the first, as the walk
// goes: each row goes on from where it was, so that a step costs 64 hops at most, and its
// warp brings the parents of a step's rows to shared memory, if one of its walks is there.
// (Each step from the row itself takes a time that grows with the square of the depth: a
// chain of 4,000 rows 17.8 ms, of 8,000 141, where prefill takes 0.13 and 0.39; so 0.96
// and 3.4. Random trees of 8,000 rows 1.02 -> 0.95, where each step of larger trees is
// brought 1.08. A chain of 512 on 3,000 slots, as it is held: 163 us, prefill 47.)
constexpr int kTreeHeld = 512;

template <int D>
struct TreeCfg {
  static constexpr int kQBytes = kTreeRows * D * 2;
  static constexpr int kBlockBytes = kTreeRows * 128;   // one 64-column block of the Q tile
  static constexpr int kTileBytes = kTreeKeys * D * 2;  // a K or V tile
  static constexpr int kGroupBytes = 8 * D * 2;         // 8 keys of a tile
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr int kOffRing = kQBytes;
  static constexpr int kOffBar = kOffRing + kSlots * kTileBytes;
  // full, empty, sfull, pfull, ofull, item full and empty, upfull, qfull, qempty, drain, one unused (an even number)
  static constexpr int kBars = 2 * kSlots + 2 + 2 + 2 + 4 + 2 + 4;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kOffItems = kOffMisc + 16;
  static constexpr int kOffUp = kOffItems + 2 * 48;  // parents of the items in the two slots
  static constexpr int kOffWindow = kOffUp + 2 * kTreeHeld * 4;  // [4][kTreeKeys]: of each row warp's step, in larger trees
  static constexpr int kSmemBytes = kOffWindow + 4 * kTreeKeys * 4 + 1024;
  // A cluster's pieces take the tiles' place: D / 4 quads of sums a row, then (m, l) of each piece.
  static_assert(kTreeRows * (D * 4 + kDecCluster * 8) <= kQBytes + kSlots * kTileBytes, "the pieces' place");
  static_assert(kSmemBytes <= 113 * 1024, "two CTAs per SM");
  // TMEM columns: two S (P over the first half of each), then O.
  static constexpr int kTmemCols = 256, kColO = 128;
};

// Places in the list that a segment takes before its first step, for its start and
// end (1, 2, 3, 4 of them: 24 trees of up to 26 tokens on up to 4,122 slots 22.9, 21.9,
// 20.8, 21.3 us; 96 of 8 on 300  27.1, 26.8, 25.0, 25.3; 8 of up to 4, 32 heads, on up
// to 1,200  13.5, 13.7, 14.3, 14.9).
constexpr int kTreeCost = 3;

struct TreeWork {
  const int32_t* parents;  // [tokens]
  int32_t cluster;         // CTAs of a segment (a cluster, or one), no pieces in memory, no second kernel; 0: the list
  int32_t cluster_shift;   // log2 of it
  // Pieces of segments that cross CTAs: each CTA has place 0 for one that began
  // earlier, place 1 for one that goes on. Rows are the fastest index: a thread has
  // a row.
  float4* part;            // [grid][2][head_dim / 4][128]
  float2* part_ml;         // [grid][2][128] (m, l)
  // The segment that begins in this CTA and ends in a later one: its pieces (0: there
  // is none) + rows << 14 + units of its join << 22, and (kv head, first packed row).
  int32_t* pieces;         // [grid]
  int2* spill;             // [grid]
};

struct TreeParams {
  PagedView kv;
  const void* q;
  void* out;
  int64_t qt, qh, ot, oh;  // token and head strides, elements
  const int32_t* cu;
  int32_t tokens;          // rows of q
  int32_t group;           // query heads per kv head
  int32_t tile_tokens;     // tokens of a tile: 128 / group, or fewer (tree_plan)
  float scale_log2;        // |scale| * log2(e), never 0
  int32_t negate;          // scale < 0
  uint32_t group_inv;      // ceil(2^16 / group): row_token()
  TreeWork work;
};

// Parents of a tree's rows from `first` on.
struct TreeParents {
  const int32_t* at;
  int first;
  __host__ __device__ __forceinline__ int operator[](int row) const { return at[row - first]; }
};

// What a row sees of a step's 64 slots, 32 to a word: every slot before the
// drafted ones (`base` of them from the step's first on, may be negative), and of
// those the row's own and its ancestors'. The walk up goes from `row`, the row itself
// or the first of its ancestors that no later step holds, to the first before this
// step, which is returned, -1 behind the root or a parent that does not come before its
// child.
template <typename Parents>
__host__ __device__ __forceinline__ int tree_words(Parents parents, int row, int base, uint32_t (&w)[2]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int below = base - c * 32;
    w[c] = below >= 32 ? 0xFFFFFFFFu : below > 0 ? (1u << below) - 1u : 0u;
  }
  while (row >= 0 && base + row >= 0) {
    const int key = base + row;
    if (key < 32) w[0] |= 1u << key;
    if (key >= 32 && key < 64) w[1] |= 1u << (key & 31);
    const int up = parents[row];
    row = up < row ? up : -1;
  }
  return row;
}

// A sequence in the list: its rows, its length, tiles of rows, and steps
// of 64 keys (one where there are no keys: its rows get their zeros).
struct TreeSeq {
  int row0, n, len, tiles, steps;
  bool bad;
};
__device__ __forceinline__ TreeSeq tree_sequence(const PagedView& kv, const int32_t* cu, int tokens, int tile_tokens, int b) {
  TreeSeq s;
  int end;
  const int raw = kv.seq_lens[b];
  packed_range(cu, b, tokens, &s.row0, &end);
  s.n = end - s.row0;
  s.len = paged_clamp_len(raw, kv.max_pages, kv.page_shift, &s.bad);
  s.bad = s.n > 0 && (s.bad || s.len < s.n);
  s.tiles = (s.n + tile_tokens - 1) / tile_tokens;
  s.steps = s.len > kTreeKeys ? (s.len + kTreeKeys - 1) / kTreeKeys : 1;
  return s;
}

// Places of the list, counted up to kNoMore. The host keeps those of sequences that
// follow one another below it, but boundaries that fall may give each of many sequences
// all rows; such a list is not worked on, whatever its sum would be.
__host__ __device__ __forceinline__ int add_places(int a, int b) {
  const uint32_t sum = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);  // both at most kNoMore
  return sum < static_cast<uint32_t>(kNoMore) ? static_cast<int>(sum) : kNoMore;
}
__device__ __forceinline__ int scan_places(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x = add_places(x, up);
  }
  return x;
}

// A CTA's share of the list, found and walked by one warp: segment y = (kv head,
// tile) of sequence b, from `step` on.
struct TreeShare {
  int total, shares;  // the list's places, and what it is cut into
  int u, u1;          // the next place, and the end of the share
  int b, y, step;
  TreeSeq seq;
};

// The list's places: of a sequence segments * (steps + cost), or, with clusters,
// segments. Lane i counts the sequences [i * part, (i + 1) * part): the lane that
// holds a place is found by one scan, its sequence by another.
//
// Shares: one for each CTA. Where all sequences have as many steps, some of the last
// fifth of the CTAs are left out if the segments then divide evenly among the rest:
// those do not cross CTAs, and four fifths of the SMs read at full speed.
// `bad`: some lane's sequence has a bad length.
__device__ __forceinline__ void tree_locate(const TreeParams& p, int lane, TreeShare* out, bool* bad) {
  const PagedView& kv = p.kv;
  const TreeWork& work = p.work;
  const int part = (kv.batch + 31) >> 5;
  TreeSeq mine;
  auto places_of = [&](int b) {
    if (b >= kv.batch) return 0;
    mine = tree_sequence(kv, p.cu, p.tokens, p.tile_tokens, b);
    return mine.tiles * kv.kv_heads * (work.cluster > 0 ? 1 : mine.steps + kTreeCost);
  };
  int sum = 0, last = 0, segments = 0, least = kNoMore, most = 0;
  *bad = false;
#pragma unroll 2
  for (int b = lane * part; b < min(kv.batch, (lane + 1) * part); ++b) {
    last = places_of(b);
    sum = add_places(sum, last);
    *bad = *bad || mine.bad;
    if (mine.tiles > 0) {
      segments += mine.tiles * kv.kv_heads;
      least = min(least, mine.steps);
      most = max(most, mine.steps);
    }
  }
  const int upto_all = scan_places(sum, lane);
  const int total = __shfl_sync(0xFFFFFFFFu, upto_all, 31);
  const int rank = work.cluster > 0 ? static_cast<int>(blockIdx.x) & (work.cluster - 1) : 0;
  int at;
  out->total = total;
  out->shares = gridDim.x;
  out->seq.tiles = 0;  // none
  out->u = out->u1 = 0;
  if (total == kNoMore) return;  // (the boundaries are told of by list_tree)
  if (work.cluster > 0) {
    at = static_cast<int>(blockIdx.x) >> work.cluster_shift;
    if (at >= total) return;
  } else {
    if (__reduce_min_sync(0xFFFFFFFFu, least) == static_cast<int>(__reduce_max_sync(0xFFFFFFFFu, most))) {
      segments = __reduce_add_sync(0xFFFFFFFFu, segments);
      const int ctas = gridDim.x;
      for (int g0 = ctas; 5 * g0 >= 4 * ctas && segments > 0; g0 -= 32) {
        const int g = g0 - lane;
        const uint32_t even =
            __ballot_sync(0xFFFFFFFFu, 5 * g >= 4 * ctas && g > 0 && (segments % max(g, 1) == 0 || g % segments == 0));
        if (even != 0) {
          out->shares = g0 - (__ffs(even) - 1);
          break;
        }
      }
    }
    at = out->u = share_start(total, out->shares, min(static_cast<int>(blockIdx.x), out->shares));
    out->u1 = share_start(total, out->shares, min(static_cast<int>(blockIdx.x) + 1, out->shares));
    if (out->u >= out->u1) return;
  }
  int src = __ffs(__ballot_sync(0xFFFFFFFFu, upto_all > at)) - 1;
  int before = __shfl_sync(0xFFFFFFFFu, upto_all - sum, src), from = 0, places = last;
  if (part > 1) {  // which of that lane's sequences
    const int end = min(kv.batch, (src + 1) * part);
    for (from = src * part; from < end; from += 32) {
      places = from + lane < end ? places_of(from + lane) : 0;
      const int upto = warp_scan(places, lane);
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + upto > at);
      if (past != 0) {
        src = __ffs(past) - 1;
        before += __shfl_sync(0xFFFFFFFFu, upto - places, src);
        break;
      }
      before += __shfl_sync(0xFFFFFFFFu, upto, 31);
      places = 0;
    }
  }
  if (__shfl_sync(0xFFFFFFFFu, places, src) == 0) {  // never, unless lengths change under the call
    out->u1 = out->u;
    return;
  }
  out->b = from + src;
  out->seq.row0 = __shfl_sync(0xFFFFFFFFu, mine.row0, src);
  out->seq.n = __shfl_sync(0xFFFFFFFFu, mine.n, src);
  out->seq.len = __shfl_sync(0xFFFFFFFFu, mine.len, src);
  out->seq.tiles = __shfl_sync(0xFFFFFFFFu, mine.tiles, src);
  out->seq.steps = __shfl_sync(0xFFFFFFFFu, mine.steps, src);
  out->seq.bad = false;
  if (work.cluster > 0) {
    out->y = at - before;
    const int base = out->seq.steps >> work.cluster_shift, rest = out->seq.steps & (work.cluster - 1);  // share_start()
    out->u = out->step = rank * base + min(rank, rest);
    out->u1 = out->u + base + (rank < rest);
  } else {
    const int per = out->seq.steps + kTreeCost, in = at - before;
    out->y = in / per;
    const int off = in - out->y * per;
    out->step = max(0, off - kTreeCost);
    out->u += kTreeCost + out->step - off;  // the first step at or behind u
  }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, uint64_t* bar, int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// One segment, or a piece of one.
struct __align__(16) TreeItem {
  int32_t valid;    // 0: no more work
  int32_t hk;       // kv head
  int32_t place;    // of its sums: the CTA's 0 or 1, or -1: the whole segment, its rows are results
  int32_t seq, len; // sequence, its keys
  int32_t row0, n;  // its first packed row and its rows
  int32_t tok0;     // first token of the tile within them
  int32_t j0, j1;   // steps
  // The step that is taken first, and the way to the next (kTreeHeld).
  __device__ __forceinline__ int first() const { return n > kTreeHeld ? j1 - 1 : j0; }
  __device__ __forceinline__ int way() const { return n > kTreeHeld ? -1 : 1; }
};
static_assert(sizeof(TreeItem) == 48, "items' place in shared memory");

// log2 of a unit's (row, 4 columns), of which a thread has one or, where that still
// asks for all pieces in one round, several of a row, which share the pieces' weights:
// what the join of many rows is bound by are its instructions (96 trees of 56 rows on
// 300 slots: 25.0 us, with one each 26.9), that of few rows by round trips, and it is
// spread as far as it goes (12 trees of up to 13 rows, 32 heads: 22.6 with several, 21.6
// with one). Of more than 16 pieces four threads share one.
__device__ __forceinline__ int tree_join_shift(int pieces, int rows) {
  return pieces > 16 ? 5 : pieces > 8 || rows <= 32 ? 7 : pieces > 2 ? 8 : 9;
}

// The work warp: this CTA's share of the list (or of its cluster's segment), item by
// item into the two slots.
template <int D>
__device__ __forceinline__ void list_tree(const TreeParams& p, TreeItem* items, uint64_t* item_full, uint64_t* item_empty,
                                          volatile int* abort_flag, int lane) {
  const PagedView& kv = p.kv;
  TreeShare at;
  bool bad_len;
  tree_locate(p, lane, &at, &bad_len);
  if (bad_len && blockIdx.x == 0 && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_LEN);
  int pieces = 0;
  int2 spill;
  bool ok = true;
  // A CTA of a cluster has one item, without steps if there are too few.
  const bool single = p.work.cluster > 0 && at.seq.tiles > 0;
  for (int published = 0; ok; ++published) {
    TreeItem x;
    x.valid = at.u < at.u1 || (single && published == 0);
    if (x.valid) {
      const int end = min(at.seq.steps, at.step + (at.u1 - at.u));
      x.hk = at.seq.tiles == 1 ? at.y : at.y / at.seq.tiles;
      x.place = p.work.cluster > 1 || at.step > 0 ? 0 : end < at.seq.steps ? 1 : -1;
      x.seq = at.b;
      x.len = at.seq.len;
      x.row0 = at.seq.row0;
      x.n = at.seq.n;
      x.tok0 = (at.y - x.hk * at.seq.tiles) * p.tile_tokens;
      // Steps that the tile's last row sees.
      const int last = min(x.tok0 + p.tile_tokens, x.n) - 1;
      const int most = (visible_keys(x.len, x.n, last) + kTreeKeys - 1) / kTreeKeys;
      x.j0 = min(at.step, most);
      x.j1 = min(end, most);
      if (!single && at.step == 0 && end < at.seq.steps) {
        pieces = share_of(at.total, at.shares, at.u + at.seq.steps - 1) - static_cast<int>(blockIdx.x) + 1;
        const int rows = (last + 1 - x.tok0) * p.group, shift = tree_join_shift(pieces, rows);
        pieces |= rows << 14 | (rows * (D / 4) + (1 << shift) - 1) >> shift << 22;
        spill = make_int2(x.hk, x.row0 + x.tok0);
      }
    }
    if (published >= 2)
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(&item_empty[published & 1], ((published >> 1) - 1) & 1, abort_flag));
    if (ok && lane == 0) {
      items[published & 1] = x;
      mbar_arrive(&item_full[published & 1]);
    }
    if (!x.valid || !ok) break;
    // The next segment (a share's end is found by its place).
    at.u += at.seq.steps - at.step + kTreeCost;
    at.step = 0;
    if (single) at.u = at.u1;
    if (at.u < at.u1 && ++at.y == kv.kv_heads * at.seq.tiles) {
      at.y = 0;
      do {
        if (++at.b >= kv.batch)
          at.u = at.u1;  // never, unless lengths change under the call
        else
          at.seq = tree_sequence(kv, p.cu, p.tokens, p.tile_tokens, at.b);
      } while (at.u < at.u1 && at.seq.tiles == 0);
    }
  }
  if (p.work.cluster == 0 && lane == 0) {
    p.work.pieces[blockIdx.x] = pieces;
    if (pieces > 0) p.work.spill[blockIdx.x] = spill;
  }
  if (blockIdx.x == gridDim.x - 1) check_boundaries(p.cu, kv.batch, p.tokens, lane, kv.status);
}

// Where the row (token, head of the group) r of a tile that begins with packed row
// `first` goes.
__device__ __forceinline__ uint16_t* tree_out(const TreeParams& p, int64_t first, int hk, int r, int token) {
  return static_cast<uint16_t*>(p.out) + (first + token) * p.ot + (hk * p.group + (r - token * p.group)) * p.oh;
}

// The pieces of a cluster's CTAs: each CTA joins D / cluster columns. The rows of each
// send every CTA its part of their sums, from TMEM into its shared memory, where all
// pieces then lie, in their order. (Each CTA reading its part out of the others' took
// 2.6 us, and one more barrier.) All threads of the cluster come here, with or without
// an item, so that no CTA has ended when another sends to it; `m` and `l` are those of
// the row, -infinity and 0 where it saw nothing.
template <int D, bool F16>
__device__ __forceinline__ void join_tree_cluster(const TreeParams& p, const TreeItem& x, uint8_t* smem, uint32_t row_tmem, float m,
                                                  float l) {
  constexpr int kQuads = D / 4;
  const int cluster = p.work.cluster, shift = p.work.cluster_shift, rank = static_cast<int>(blockIdx.x) & (cluster - 1);
  const int per = kQuads >> shift;  // a CTA's columns, by four
  const int per_shift = (D == 128 ? 5 : 4) - shift;
  const int r = threadIdx.x & (kTreeRows - 1), token = row_token(r, p.group_inv);
  const bool live = x.valid && token < min(p.tile_tokens, x.n - x.tok0);
  float4* sums = reinterpret_cast<float4*>(smem);                                // [piece][per][row]
  float2* sums_ml = reinterpret_cast<float2*>(smem + kQuads * kTreeRows * 16);   // [piece][row]
  // Nobody's products read the tiles any more: they have ended, and what copies and the
  // issuing warp had written there, over which the other CTAs' sums now come, is ordered by
  // that warp's fence in its last step. (A barrier that releases orders it too, here, where
  // all wait for it: 1 tree of 16 tokens on 512 slots 8.4 us, 8.2 if only that warp's
  // arrival does, 7.7 so.)
  asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait;" ::: "memory");
  tc_fence_after();
  if (__any_sync(0xFFFFFFFFu, live)) {
    if (x.j0 < x.j1) {
#pragma unroll 1
      for (int i = threadIdx.x / kTreeRows; i < D / 32; i += kTreeThreads / kTreeRows) {
        const int c = ((i + (rank >> 1)) & (D / 32 - 1)) * 32;  // not all to the same CTA at once
        uint32_t o[32];
        tmem_ld_32x32b_x32(row_tmem + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int quad = c / 4 + k, to = quad >> per_shift;
          if (live)
            st_cluster_f4(map_rank(smem_u32(sums + (rank * per + (quad & (per - 1))) * kTreeRows + r), to),
                          make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]),
                                      __uint_as_float(o[4 * k + 3])));
        }
      }
    }
    if (live && threadIdx.x < kTreeRows)
      for (int to = 0; to < cluster; ++to) st_cluster_f2(map_rank(smem_u32(sums_ml + rank * kTreeRows + r), to), make_float2(m, l));
  }
  cluster_barrier();
  if (!live) return;
  float2 ml[kDecCluster];
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int c = 0; c < kDecCluster; ++c) {
    ml[c] = c < cluster ? sums_ml[c * kTreeRows + r] : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[c].x);
  }
  if (top == -INFINITY) top = 0.f;
#pragma unroll
  for (int c = 0; c < kDecCluster; ++c) {
    ml[c].x = exp2_approx(ml[c].x - top);
    if (ml[c].y != 0.f) sum += ml[c].x * ml[c].y;
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  uint16_t* dst = tree_out(p, x.row0 + x.tok0, x.hk, r, token);
  for (int quad = threadIdx.x / kTreeRows; quad < per; quad += kTreeThreads / kTreeRows) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kDecCluster; ++c) {
      if (ml[c].y == 0.f) continue;  // its sums may not have been written
      const float4 v = sums[(c * per + quad) * kTreeRows + r];
      o.x += v.x * ml[c].x;
      o.y += v.y * ml[c].x;
      o.z += v.z * ml[c].x;
      o.w += v.w * ml[c].x;
    }
    *reinterpret_cast<uint2*>(dst + (rank * per + quad) * 4) =
        make_uint2(pack2<F16>(o.x * inv, o.y * inv), pack2<F16>(o.z * inv, o.w * inv));
  }
}

template <int D, bool F16>
__global__ void __launch_bounds__(kTreeThreads, 2)
    paged_tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_q, const TreeParams p) {
  using Cfg = TreeCfg<D>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* empty = full + Cfg::kSlots;
  uint64_t* sfull = empty + Cfg::kSlots;
  uint64_t* pfull = sfull + 2;
  uint64_t* ofull = pfull + 2;
  uint64_t* item_full = ofull + 2;
  uint64_t* item_empty = item_full + 2;
  uint64_t* upfull = item_empty + 2;
  uint64_t* qfull = upfull + 2;
  uint64_t* qempty = qfull + 1;
  uint64_t* drain = qempty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  TreeItem* items = reinterpret_cast<TreeItem*>(smem + Cfg::kOffItems);
  int32_t* held = reinterpret_cast<int32_t*>(smem + Cfg::kOffUp);        // [2][kTreeHeld]
  int32_t* window = reinterpret_cast<int32_t*>(smem + Cfg::kOffWindow);  // [4][kTreeKeys]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedView& kv = p.kv;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sfull[t], 1);
      mbar_init(&pfull[t], kTreeRows);
      mbar_init(&ofull[t], 1);
      mbar_init(&item_full[t], 1);
      mbar_init(&item_empty[t], 7);  // a lane of each row warp, the loader's, the issuer's and that of the query rows
      mbar_init(&upfull[t], 1);
    }
    mbar_init(qfull, 1);
    mbar_init(qempty, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_q);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch();

  // The i-th item of this CTA, copied out of its slot. (The rows give the slot free
  // when they are done: its parents stay until then.)
  auto free_slot = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[i & 1]);
  };
  auto get_item = [&](int i, TreeItem* x) {
    const bool got = __all_sync(0xFFFFFFFFu, mbar_wait(&item_full[i & 1], (i >> 1) & 1, abort_flag));
    if (!got) {
      x->valid = 0;
      return false;
    }
    *x = items[i & 1];
    if (warp >= 4) free_slot(i);
    return x->valid != 0;
  };

  float row_m = -INFINITY, row_l = 0.f;  // of a cluster's one item
  if (warp < 4) {
    // ------------------------------------------------------------ softmax rows
    const int r = threadIdx.x;
    const int token = row_token(r, p.group_inv);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t to = lanes + Cfg::kColO;
    int count = 0;  // steps so far
    bool ok = true;
    // The product of step c has been added to O. (S and O have a barrier for even and
    // one for odd steps: a row may be two steps behind the products, and a phase's
    // parity tells one from the next only.)
    auto summed = [&](int c) {
      const bool done = __all_sync(0xFFFFFFFFu, mbar_wait(&ofull[c & 1], (c >> 1) & 1, abort_flag));
      tc_fence_after();
      return done;
    };
    TreeItem x;
    for (int i = 0; ok && get_item(i, &x); ++i) {
      const int own = x.tok0 + token;  // the row's token among the sequence's new ones
      const bool live = token < min(p.tile_tokens, x.n - x.tok0);
      // A warp without rows only keeps step: what the products make of its lanes nobody
      // reads (exponentials are a step's longest part, and a tile may have few rows).
      const bool used = __any_sync(0xFFFFFFFFu, live);
      int up_to = own;  // where the walk up has come to
      bool parents_there = false;
      float m = -INFINITY, l = 0.f;  // m: maximum that P refers to (raw scores)
      bool first = true;
      int left = x.j1 - x.j0;
      int base = x.len - x.n - x.first() * kTreeKeys;  // of the step's slots those before the drafted ones
      for (; left > 0; --left, first = false, ++count, base += x.n > kTreeHeld ? kTreeKeys : -kTreeKeys) {
        const uint32_t ts = lanes + (count & 1) * 64;
        ok = mbar_wait(&sfull[count & 1], (count >> 1) & 1, abort_flag);
        tc_fence_after();
        if (!used) {
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          mbar_arrive(&pfull[count & 1]);
          continue;
        }
        uint32_t s[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32b_x32(ts + c * 32, s[c]);
        tmem_ld_wait();
        if (p.negate) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) s[c][k] ^= 0x80000000u;
        }
        if (base < kTreeKeys) {
          uint32_t w[2] = {0u, 0u};
          if (!parents_there) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&upfull[i & 1], (i >> 1) & 1, abort_flag)) && ok;
            parents_there = true;
          }
          const bool sees = live && own >= x.n - x.len;  // of more rows than tokens the first have no slots and see none
          TreeParents parents = {held + (i & 1) * kTreeHeld, 0};
          if (x.n <= kTreeHeld) {
            if (sees) tree_words(parents, own, base, w);
          } else {
            // This step's rows, and on the way to it those that the piece does not hold.
            int32_t* mine = window + warp * kTreeKeys;
            parents.at = mine;
            int row = -base;
            if (first) row += (min(x.tok0 + p.tile_tokens, x.n) - 1 - row) / kTreeKeys * kTreeKeys;
            for (; row >= -base; row -= kTreeKeys) {
              parents.first = row;
              __syncwarp();
              if (__any_sync(0xFFFFFFFFu, sees && up_to >= row)) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const int at = row + c * 32 + lane;
                  if (at >= 0 && at < x.n) mine[c * 32 + lane] = p.work.parents[x.row0 + at];
                }
              }
              __syncwarp();
              if (sees) up_to = tree_words(parents, up_to, -row, w);
            }
          }
          // A row's own slot is in one step and one piece: there its parent is looked at.
          if (sees && base + own >= 0 && base + own < kTreeKeys) {
            const int up = parents[own];
            if ((up < -1 || up >= own) && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_DRAFT);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!(w[c] >> k & 1u)) s[c][k] = 0xFF800000u;  // -inf
        }
        float mx[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mx[c] = max3(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]), __uint_as_float(s[c][2]));
#pragma unroll
          for (int k = 3; k < 31; k += 2) mx[c] = max3(mx[c], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
        }
        float mn = max3(max3(mx[0], mx[1], __uint_as_float(s[0][31])), __uint_as_float(s[1][31]), m);  // NaN if a score is
        // Also true from m = -inf and for NaN, but not while all is -inf. Rows that
        // are none have what memory held as scores, and nobody reads their sums.
        const bool raise = live && !((mn - m) * p.scale_log2 <= kPreLag<F16>) && mn != -INFINITY;
        if (first || __any_sync(0xFFFFFFFFu, raise || !ok)) {
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          if (mn == INFINITY) mn = __int_as_float(0x7FC00000);  // inf - inf: the row is NaN
          const float f = m == -INFINITY ? 0.f : exp2_approx((m - mn) * p.scale_log2);
          m = mn;
          if (!first) {
            ok = summed(count - 1);
            if (!ok) break;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(to + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st_32x32b_x32(to + c * 32, o);
            }
            tmem_st_wait();
          }
        }
        const float shift = m == -INFINITY ? 0.f : fmaf(-m, p.scale_log2, kPreLift<F16>);
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), shift2 = make_float2(shift, shift);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float2 y = fma2(make_float2(__uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1])), scale2, shift2);
            y.x = exp2_approx(y.x);
            y.y = exp2_approx(y.y);
            sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], y);
            pk[c * 16 + (k >> 1)] = pack2<F16>(y.x, y.y);
          }
        tmem_st_32x32b_x32(ts, pk);
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&pfull[count & 1]);
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      const bool any = x.j1 > x.j0;
      if (any) {
        ok = summed(count - 1);
        if (!ok) break;
      }
      if (!used) {
        free_slot(i);
        continue;
      }
      if (p.work.cluster > 1) {  // joined below
        row_m = any ? m * p.scale_log2 : -INFINITY;
        row_l = any ? l : 0.f;
        break;
      }
      // Sums of a piece go to its place.
      const int64_t place = static_cast<int64_t>(blockIdx.x) * 2 + max(x.place, 0);
      float4* sums = p.work.part + place * (D / 4) * kTreeRows;
      float2* sums_ml = p.work.part_ml + place * kTreeRows;
      uint16_t* dst = tree_out(p, x.row0 + x.tok0, x.hk, r, token);
      if (live && x.place >= 0) sums_ml[r] = make_float2(m == -INFINITY ? m : m * p.scale_log2, l);
      if (!any) {  // no keys
        if (live && x.place < 0)
          for (int k = 0; k < D; k += 8) *reinterpret_cast<uint4*>(dst + k) = make_uint4(0u, 0u, 0u, 0u);
      } else {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(to + c, o);
          tmem_ld_wait();
          if (!live) continue;
          if (x.place >= 0) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              sums[((c + k) >> 2) * kTreeRows + r] = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]),
                                                                 __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint4 w;
              w.x = pack2<F16>(__uint_as_float(o[k]) * inv, __uint_as_float(o[k + 1]) * inv);
              w.y = pack2<F16>(__uint_as_float(o[k + 2]) * inv, __uint_as_float(o[k + 3]) * inv);
              w.z = pack2<F16>(__uint_as_float(o[k + 4]) * inv, __uint_as_float(o[k + 5]) * inv);
              w.w = pack2<F16>(__uint_as_float(o[k + 6]) * inv, __uint_as_float(o[k + 7]) * inv);
              *reinterpret_cast<uint4*>(dst + c + k) = l == 0.f ? make_uint4(0u, 0u, 0u, 0u) : w;
            }
          }
        }
      }
      tc_fence_before();  // O is read before the next item's first P is announced
      free_slot(i);
    }
    tc_fence_before();
  } else if (warp == 4) {
    // ------------------------------------------------------------ page loads
    const int box_shift = min(kv.page_shift, 6);  // slots of a box: a page's, or half of one of 128
    const int box = 1 << box_shift, per_step = kTreeKeys >> box_shift;
    int issued = 0;  // tiles so far: slot and phase of the ring
    TreeItem x;
    bool ok = true;
    for (int i = 0; ok && get_item(i, &x); ++i) {
      const int32_t* table = kv.page_table + x.seq * kv.table_stride;
      const int held = (x.len + box - 1) >> box_shift;  // boxes of the sequence
      const int steps = x.j1 - x.j0, way = x.way(), first = x.first();
      auto entry = [&](int k) {  // a lane per box of the step
        const int at = (first + k * way) * per_step + lane;
        return k < steps && lane < per_step && at < held ? table[at >> (kv.page_shift - box_shift)] : 0;
      };
      // Keys come two steps before the values: K of the first two steps, then V and the
      // next K in turn, as the issuer uses them.
      int ids[4];  // table entries of the steps k to k + 3
#pragma unroll
      for (int k = 0; k < 4; ++k) ids[k] = entry(k);
      auto load = [&](int k, int id, bool values) {
        const int j = first + k * way;
        const int boxes = min(per_step, held - j * per_step);
        const bool mine = lane < boxes;
        if (!values && mine && (id < 0 || id >= kv.num_pages) && kv.status != nullptr)
          atomicOr(kv.status, ABFT_PAGED_BAD_PAGE);
        const int slot = issued % Cfg::kSlots;
        if (issued >= Cfg::kSlots && !mbar_wait(&empty[slot], (issued / Cfg::kSlots - 1) & 1, abort_flag)) ok = false;
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&full[slot], static_cast<uint32_t>(boxes * box * D * 2));
        __syncwarp();
        if (mine) {
          // A bad id lies outside the map's page dimension and loads zeros.
          const uint32_t dst = smem_u32(smem + Cfg::kOffRing + slot * Cfg::kTileBytes) + lane * box * D * 2;
          const int slot0 = ((j * per_step + lane) << box_shift) & ((1 << kv.page_shift) - 1);  // of the page's slots
          tma_load_5d(dst, values ? &tm_v : &tm_k, &full[slot], 0, 0, 0, ((x.hk << kv.page_shift) + slot0) >> 3, id);
        }
        ++issued;
      };
      if (steps > 0) load(0, ids[0], false);
      if (steps > 1 && ok) load(1, ids[1], false);
      for (int k = 0; k < steps && ok; ++k) {
        load(k, ids[0], true);
        if (k + 2 < steps && ok) load(k + 2, ids[2], false);
        ids[0] = ids[1];
        ids[1] = ids[2];
        ids[2] = ids[3];
        ids[3] = entry(k + 4);
      }
    }
    // Copies in flight have landed before shared memory goes (all have, but after an
    // abort).
    for (int it = max(0, issued - Cfg::kSlots); it < issued; ++it)
      mbar_wait_bounded(&full[it % Cfg::kSlots], (it / Cfg::kSlots) & 1);
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issuer
    // Control values through a shuffle and one elected lane: the compiler then keeps
    // descriptors in uniform registers.
    constexpr uint32_t fmt = F16 ? 0u : 1u;
    constexpr uint32_t idesc_s = umma_idesc(kTreeRows, kTreeKeys, fmt);
    constexpr uint32_t idesc_o = umma_idesc(kTreeRows, D, fmt) | kIdescBNMajor;
    const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
    const uint32_t q_base = __shfl_sync(0xFFFFFFFFu, smem_u32(smem), 0);
    const uint64_t desc_q = sw128_kmajor_desc(q_base);
    const uint64_t desc_k = ring_desc(q_base + Cfg::kOffRing, 16, Cfg::kGroupBytes);
    const uint64_t desc_v = ring_desc(q_base + Cfg::kOffRing, 1024, Cfg::kGroupBytes);
    bool ok = true;
    int slot = 0, phase = 0;      // of the next tile in the ring
    int scored = 0, summed = 0;   // S and O products so far
    int begun = 0;                // items with steps so far
    auto ready = [&]() {
      ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(&full[slot], phase, abort_flag));
      tc_fence_after();
      return ok;
    };
    auto release = [&]() {  // the ring's next slot, once the MMAs so far have read it
      if (elect_one()) umma_commit(&empty[slot]);
      __syncwarp();
      if (++slot == Cfg::kSlots) {
        slot = 0;
        phase ^= 1;
      }
    };
    auto scores = [&](bool last) {
      if (!ready()) return;
      if (elect_one()) {
        const uint64_t dk = desc_k + slot * (Cfg::kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_bf16_ss(tm + (scored & 1) * 64, desc_q + (((k / 4) * Cfg::kBlockBytes + (k % 4) * 32) >> 4),
                       dk + (((k / 4) * 1024 + (k % 4) * 32) >> 4), idesc_s, k > 0);
        umma_commit(&sfull[scored & 1]);
        if (last) umma_commit(qempty);
      }
      __syncwarp();
      ++scored;
      release();
    };
    TreeItem x;
    for (int i = 0; ok && get_item(i, &x); ++i) {
      // `keys` of the sequence from the step's first on.
      const int steps = __shfl_sync(0xFFFFFFFFu, x.j1 - x.j0, 0), way = __shfl_sync(0xFFFFFFFFu, x.way() * kTreeKeys, 0);
      int keys = __shfl_sync(0xFFFFFFFFu, x.len - x.first() * kTreeKeys, 0);
      // (The query rows of an item without steps are not brought.)
      if (steps <= 0) continue;
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(qfull, begun & 1, abort_flag));
      ++begun;
      tc_fence_after();
      if (!ok) break;
      scores(steps == 1);
      if (steps > 1 && ok) scores(steps == 2);
      for (int k = 0; k < steps && ok; ++k, keys -= way) {
        if (!ready()) break;
        // Weights of slots behind the length are 0, but the slots may hold anything (a
        // page's last owner, NaN): only whole groups of 16 keys that the sequence
        // reaches are multiplied, the rest of the last group is cleared.
        const int valid = min(kTreeKeys, keys);
        const int groups = (valid + 15) / 16;
        if (valid & 15) {
          uint8_t* v = smem + Cfg::kOffRing + slot * Cfg::kTileBytes;
          for (int at = valid * (D / 8) + lane; at < groups * 16 * (D / 8); at += 32) {
            const int row = at / (D / 8), c = at % (D / 8);  // every piece of the row: its order does not matter
            *reinterpret_cast<uint4*>(v + (row >> 3) * Cfg::kGroupBytes + (c >> 3) * 1024 + (row & 7) * 128 + ((c & 7) << 4)) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        // All tiles have been written and seen here: before another CTA's sums come over
        // them (join_tree_cluster). The rows' weights are waited for meanwhile.
        if (p.work.cluster > 1 && k + 1 == steps) asm volatile("fence.acq_rel.cluster;" ::: "memory");
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&pfull[summed & 1], (summed >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dv = desc_v + slot * (Cfg::kTileBytes >> 4);
          const uint32_t a = tm + (summed & 1) * 64, d = tm + Cfg::kColO;
          umma_f16_ts(d, a, dv, idesc_o, k > 0);
          for (int g = 1; g < groups; ++g) umma_f16_ts(d, a + g * 8, dv + g * (2 * Cfg::kGroupBytes >> 4), idesc_o, 1);
          umma_commit(&ofull[summed & 1]);
        }
        __syncwarp();
        ++summed;
        release();
        if (k + 2 < steps) scores(k + 3 == steps);
      }
    }
    // Nothing still writes TMEM when it is freed.
    if (elect_one()) umma_commit(drain);
    __syncwarp();
    mbar_wait_bounded(drain, 0);
  } else if (warp == 6) {
    list_tree<D>(p, items, item_full, item_empty, abort_flag, lane);
  } else {
    // ------------------------------------------------------------ query rows and parents
    // Query rows by one box for each 64 columns, (token, head) rows of the tile, once
    // the last item's scores have all been computed; rows behind the sequence's are
    // another's, which nobody reads the sums of.
    int brought = 0;
    bool ok = true;
    TreeItem x;
    for (int i = 0; ok && get_item(i, &x); ++i) {
      if (x.j0 < x.j1) {
        if (brought > 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait(qempty, (brought - 1) & 1, abort_flag));
        if (!ok) break;
        ++brought;
        if (lane == 0) {
          mbar_arrive_expect_tx(qfull, static_cast<uint32_t>(p.tile_tokens * p.group * D * 2));
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(smem_u32(smem) + c * Cfg::kBlockBytes, &tm_q, qfull, c * 64, x.hk * p.group, x.row0 + x.tok0);
        }
        __syncwarp();
        if (x.n <= kTreeHeld && x.j1 * kTreeKeys > x.len - x.n)
          for (int k = lane; k < x.n; k += 32) held[(i & 1) * kTreeHeld + k] = p.work.parents[x.row0 + k];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&upfull[i & 1]);
    }
    // The last copy has landed before shared memory goes (it has, but after an abort).
    if (brought > 0) mbar_wait_bounded(qfull, (brought - 1) & 1);
  }
  __syncthreads();
  if (p.work.cluster > 1)
    join_tree_cluster<D, F16>(p, items[0], smem, tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + Cfg::kColO, row_m, row_l);
  if (threadIdx.x == 0 && *abort_flag && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_TIMEOUT);
  tc_fence_after();
  __syncwarp();  // lanes without rows come from the join before the others
  if (warp == 5) tmem_dealloc(tmem, Cfg::kTmemCols);
}

// Joins the segments that cross CTAs: of one that begins in CTA c the pieces are CTA
// c's place 1 and the following CTAs' place 0. A thread has (row, 4 columns) of a
// segment, or several of a row, and asks for up to 16 sums at once,
// by asynchronous copies into its own column of shared memory: what counts is the
// number of round trips. (In registers, three or six at once, the join of 18 pieces
// took 14 us.) Of more pieces than that each warp takes every fourth. Units of a
// block's work of all segments are one list, dealt to the blocks in turn.
constexpr int kTreeJoinThreads = 128;
constexpr int kTreeJoinSlots = 16;

template <int D, bool F16, int kParts, int kQuads>
__device__ __forceinline__ void join_tree_unit(const TreeParams& p, int c, int pieces, int rows, int unit, float4* s_o, float2* s_ml) {
  constexpr int kLane = kTreeJoinThreads / kParts;  // threads of a part
  const int part = kParts == 1 ? 0 : threadIdx.x / kLane;
  const int mine = unit * kLane + threadIdx.x - part * kLane, all = rows * (D / 4 / kQuads);
  const int index = min(mine, all - 1);  // behind the end the last one again, which is not written
  const int2 spill = p.work.spill[c];
  const uint32_t rows_inv = ((1u << 20) + rows - 1) / rows;
  const uint32_t to = smem_u32(s_o + threadIdx.x), to_ml = smem_u32(s_ml + threadIdx.x);
  // index / rows: exact, since the product overshoots by less than index / 2^20 < 1 / rows.
  const int group = static_cast<int>(static_cast<uint32_t>(index) * rows_inv >> 20), row = index - group * rows;
  float m = -INFINITY, l = 0.f;
  float4 o[kQuads];
#pragma unroll
  for (int i = 0; i < kQuads; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float2 ml, const float4* v, int stride) {
    const float top = fmaxf(m, ml.x), ms = top == -INFINITY ? 0.f : top;
    const float f = exp2_approx(m - ms), f2 = exp2_approx(ml.x - ms);
    const bool any = ml.y != 0.f;  // what a row saw nothing of was not written
    m = top;
    l = l * f + ml.y * f2;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const float4 x = v[i * stride];
      o[i].x = o[i].x * f + (any ? x.x * f2 : 0.f);
      o[i].y = o[i].y * f + (any ? x.y * f2 : 0.f);
      o[i].z = o[i].z * f + (any ? x.z * f2 : 0.f);
      o[i].w = o[i].w * f + (any ? x.w * f2 : 0.f);
    }
  };
  constexpr int kAtOnce = kTreeJoinSlots / kQuads;  // pieces
#pragma unroll 1
  for (int s0 = part; s0 < pieces; s0 += kParts * kAtOnce) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int piece = s0 + k * kParts;
      if (piece >= pieces) break;
      // (Places stay below 2^14, sums below 2^26 float4.)
      const int at = (c + piece) * 2 + (piece == 0 ? 1 : 0);
      const float4* from = p.work.part + ((at * (D / 4) + group * kQuads) * kTreeRows + row);
#pragma unroll
      for (int i = 0; i < kQuads; ++i) cp_async16(to + (k * kQuads + i) * kTreeJoinThreads * 16, from + i * kTreeRows, 16u);
      cp_async8(to_ml + k * kTreeJoinThreads * 8, p.work.part_ml + (at * kTreeRows + row));
    }
    cp_async_commit();
    cp_async_wait<0>();
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (s0 + k * kParts >= pieces) break;
      add(s_ml[k * kTreeJoinThreads + threadIdx.x], s_o + k * kQuads * kTreeJoinThreads + threadIdx.x, kTreeJoinThreads);
    }
  }
  if constexpr (kParts > 1) {
    static_assert(kQuads == 1, "one place for a thread's sums");
    __syncthreads();
    s_ml[threadIdx.x] = make_float2(m, l);
    s_o[threadIdx.x] = o[0];
    __syncthreads();
    if (part == 0)
#pragma unroll
      for (int k = 1; k < kParts; ++k) add(s_ml[k * kLane + threadIdx.x], s_o + k * kLane + threadIdx.x, 0);
    __syncthreads();  // read before the next unit's sums come
    if (part > 0) return;
  }
  if (mine >= all) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint16_t* dst = tree_out(p, spill.y, spill.x, row, row_token(row, p.group_inv)) + group * kQuads * 4;
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
    *reinterpret_cast<uint2*>(dst + i * 4) = make_uint2(pack2<F16>(o[i].x * inv, o[i].y * inv), pack2<F16>(o[i].z * inv, o[i].w * inv));
}

template <int D, bool F16>
__global__ void __launch_bounds__(kTreeJoinThreads, 4) paged_tree_join_kernel(const TreeParams p, const int grid) {
  __shared__ float4 s_o[kTreeJoinSlots * kTreeJoinThreads];
  __shared__ float2 s_ml[kTreeJoinSlots * kTreeJoinThreads];
  const int lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  int before = 0, unit = blockIdx.x;
  constexpr int kLook = 10;  // CTAs that a lane looks at
#pragma unroll 1
  for (int c0 = 0; c0 < grid; c0 += 32 * kLook) {
    int n[kLook], units = 0;
#pragma unroll
    for (int k = 0; k < kLook; ++k) {
      const int c = c0 + lane * kLook + k;
      n[k] = c < grid ? p.work.pieces[c] : 0;
    }
#pragma unroll
    for (int k = 0; k < kLook; ++k) units += n[k] >> 22;
    const int upto = warp_scan(units, lane);
    const int here = __shfl_sync(0xFFFFFFFFu, upto, 31);
#pragma unroll 1
    for (; unit < before + here; unit += gridDim.x) {
      const int src = __ffs(__ballot_sync(0xFFFFFFFFu, before + upto > unit)) - 1;
      int at = unit - before - (upto - units), c = 0, x = 0;  // of the lane that has it: the unit among a CTA's
#pragma unroll
      for (int k = 0; k < kLook; ++k) {
        const int mine = n[k] >> 22;
        if (x == 0 && at < mine) c = c0 + lane * kLook + k, x = n[k];
        if (x == 0) at -= mine;
      }
      at = __shfl_sync(0xFFFFFFFFu, at, src);
      c = __shfl_sync(0xFFFFFFFFu, c, src);
      x = __shfl_sync(0xFFFFFFFFu, x, src);
      const int pieces = x & 0x3FFF, rows = x >> 14 & 0xFF;
      switch (tree_join_shift(pieces, rows)) {
        case 9: join_tree_unit<D, F16, 1, 4>(p, c, pieces, rows, at, s_o, s_ml); break;
        case 8: join_tree_unit<D, F16, 1, 2>(p, c, pieces, rows, at, s_o, s_ml); break;
        case 7: join_tree_unit<D, F16, 1, 1>(p, c, pieces, rows, at, s_o, s_ml); break;
        default: join_tree_unit<D, F16, 4, 1>(p, c, pieces, rows, at, s_o, s_ml); break;
      }
    }
    before += here;
  }
}

}  // namespace abft
