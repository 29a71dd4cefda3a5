// paged_prefill.cuh - causal attention of prompt chunks over the paged cache.
//
// Query row i of sequence b (n new tokens of L in all) sees the slots
// j <= L - n + i:   o = sum_j softmax_j(scale q . k_j) v_j.
//
// Bound: 4 d flops per visible (query, key) pair against 2 bytes of K and V
// per key and 128-row tile: a chunk of some hundred tokens is bound by the
// tensor cores and by the exponentials (one per pair: 16 a clock and SM,
// as long as the 4 d = 512 flops of the pair take at 8192 a clock), a short
// one by reading the cache.
//
// One CTA takes two tiles of 128 query rows of one kv head. A tile's rows are
// (token, query head of the group) pairs, so that a group shares each key and
// a short chunk fills its rows. Per 128 keys:
//   S = Q K^T   tcgen05.mma, both operands in shared memory, S in TMEM
//   P = 2^(x - m) by one thread per row (no exchange between lanes): S is read
//       from TMEM, P goes back over it as 16-bit operand (heads of 64: beside
//       it, and the next S is computed meanwhile; 8,192 tokens of 32 heads: 366
//       us, 395 without)
//   O += P V    tcgen05.mma with P from TMEM, V as N-major operand
// The two tiles alternate: while the tensor core works on one, the other's
// rows are exponentiated. O stays in TMEM; it is rescaled only when a row's
// maximum has risen by more than 2^8 (fp16: 2^5) since the last rescaling, which
// after the first tiles of a row hardly happens: P and the sum l then still fit
// their formats. fp16 ends at 2^-24, and the many keys of a long cache may weigh
// less than that each and still count together: there P is lifted by 2^10 (2^15
// at most, within the format), so that weights down to 2^-24 of the greatest keep
// all their bits, smaller ones steps of 2^-34; the quotient takes it out again.
// P is rounded to 16 bits for the product, l sums it unrounded. The weights'
// errors mostly cancel (relative error against 64 bits, 600 rows on 2,000 keys:
// 2.2e-3 bf16, 2.7e-4 fp16, where the output's rounding alone is 1.7e-3 and
// 2.1e-4; rows of a few great weights 1.9e-3, of one 1.6e-3), at worst, a row of
// one weight whose maximum lags, they add half a step: with an exact maximum
// that weight would be 1. l of the rounded weights makes 2.17e-3 and 1.8e-3 of
// 2.19e-3 and 1.9e-3 and costs 7-10% with heads of 64, 1.4% with 128; two terms of
// P, as in decode, would double the second product.
//
// A call with few rows takes one tile an item, and both groups of row warps
// work on it, on every other step each ("shared" below), with an O of their
// own; the two are added at the end (512 tokens on 8,192 slots: 118 us with one
// group at work, 86 with both, the rate at which an SM takes in K and V).
//
// The grid has a block for every work item (one or two tiles, kv head, piece of
// the keys); a resident CTA takes over the items of blocks that have not
// started (cluster launch control), so that the next item's loads, Q K^T and
// set-up run under the last one's end, and items without work cost no launch.
//
// Warps: 0-3 and 4-7 the rows of tile 0 and 1 (TMEM lane quadrant = warp % 4),
// 8 TMA loads of pages into a ring of tiles, 9 the MMA issuer, 10 finds the
// work, 11 idle (registers move between groups of four warps).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_decode.cuh"
#include "paged_index.cuh"
#include "ptx.cuh"

namespace abft {

constexpr int kPreRows = 128;   // query rows of a tile
constexpr int kPreKeys = 128;   // keys of a step
constexpr int kPreThreads = 384;
// Registers: 384 threads launch with at most 168 each (64,512 in all); the
// rows' warps hold a whole row of S and take 200, the others keep 104:
// 256 * 200 + 128 * 104 = 64,512. (The issuer's loop in local memory for want
// of registers doubles the kernel's time.)
constexpr int kPreRegsRows = 200, kPreRegsOther = 104;
// How far (powers of 2) a row's maximum may have risen above the one that P
// refers to, and what P is lifted by: lag + lift stay below fp16's 2^16. (fp16,
// 8,192 tokens, 28 heads of 128 / 32 of 64, chunks on a prefix: lag 8 417 / 392 /
// 88.4 us, 5 414 / 403 / 88.4, 3 430 / 408 / 90.9, 2 456 / 418 / 92.4.)
template <bool F16>
constexpr float kPreLag = F16 ? 5.f : 8.f;
template <bool F16>
constexpr float kPreLift = F16 ? 10.f : 0.f;

template <int D>
struct PrefillCfg {
  static constexpr int kTileBytes = kPreKeys * D * 2;        // a K, V or Q tile
  static constexpr int kBlockBytes = kPreRows * 128;         // one 64-column block of a Q tile
  static constexpr int kGroupBytes = 8 * D * 2;              // 8 keys of a ring tile
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kOffRing = 2 * kTileBytes;            // after the two Q tiles
  static constexpr int kOffBar = kOffRing + kSlots * kTileBytes;
  // full, empty, qfull, sfull, pfull, ofull, sread, item full and empty, work,
  // loaded, both, drain (an even number)
  static constexpr int kBars = 2 * kSlots + 2 + 2 + 2 + 2 + 2 + 4 + 1 + 1 + 1 + 1;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kOffItems = kOffMisc + 16;  // two items and the launch-control answer
  static constexpr int kSmemBytes = kOffItems + 2 * 48 + 16 + 1024;
  static_assert(kBars % 2 == 0, "the answer is 16-byte aligned");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
  static_assert(kSmemBytes > 232448 / 2, "one CTA per SM: each takes all of TMEM");
  // TMEM columns: S of both tiles (P over its first half), then O of both; with
  // heads of 64 there is room for a P of their own behind them.
  static constexpr int kTmemCols = 512;
  static constexpr int kColO = 256, kColP = kColO + 2 * D;
};

struct PrefillParams {
  PagedView kv;
  const void* q;
  void* out;
  int64_t qt, qh, ot, oh;  // token and head strides, elements
  const int32_t* cu;
  int32_t tokens;          // rows of q
  int32_t group;           // query heads per kv head
  int32_t tile_tokens;     // tokens of one tile: 128 / group
  int32_t block_tokens;    // tokens of an item: one tile's or two's
  int32_t splits;          // pieces of an item's keys at most
  int32_t piece;           // steps of a piece; 0: chosen by the kernel, for the lengths it finds
  int32_t sms;             // items that run at once
  int32_t* chosen;         // [1] the piece chosen, for the join
  float scale_log2;        // |scale| * log2(e), never 0
  int32_t negate;          // scale < 0
  uint32_t group_inv;      // ceil(2^16 / group): row_token()
  float* part_o;           // [tokens * heads][splits][head_dim]
  float2* part_ml;         // [tokens * heads][splits]
};

// row / group for a row of a tile: exact for rows below 128 and groups up to 64
// (the product overshoots the quotient by less than 128 / 2^16 < 1 / 64).
__host__ __device__ __forceinline__ int row_token(int row, uint32_t group_inv) {
  return static_cast<int>((static_cast<uint32_t>(row) * group_inv) >> 16);
}

// Pieces of `piece` steps that `steps` steps are cut into, one at least.
__host__ __device__ __forceinline__ int pieces_of(int steps, int piece) {
  return steps <= piece ? 1 : (steps + piece - 1) / piece;
}

// Keys that local token i of n sees in a sequence of length len.
__host__ __device__ __forceinline__ int visible_keys(int len, int n, int i) {
  const int v = len - n + i + 1;
  return v > 0 ? v : 0;
}

// The list of work: the packed sequences, each cut into blocks of tokens, their
// keys into pieces (as many for each block as the sequence's length gives, so
// that places without work are few and at the end), as a warp holds it: lane i
// has the sequences [i * share, (i + 1) * share). Read once per CTA: a scan of
// the whole batch for every item made 4 tokens for each of 1,024 sequences of
// 500 slots 381 us instead of 240.
struct WorkScan {
  int share, piece;
  int places, upto;       // of this lane's sequences; with those of all lanes before
  int begin, count, len;  // share 1: the lane's sequence
};

// A sequence's packed rows and raw length (boundaries and length are asked for
// together); returns its blocks and the steps of its whole length.
__device__ __forceinline__ int blocks_of(const PrefillParams& p, int b, int* begin, int* count, int* len, int* steps) {
  int end;
  bool bad;
  *len = p.kv.seq_lens[b];
  packed_range(p.cu, b, p.tokens, begin, &end);
  *count = end - *begin;
  const int keys = paged_clamp_len(*len, p.kv.max_pages, p.kv.page_shift, &bad);
  *steps = (keys + kPreKeys - 1) / kPreKeys;
  return (*count + p.block_tokens - 1) / p.block_tokens;
}

// Blocks of sequences, and what the choice of the piece needs of their steps. A
// block without keys still takes a place in the list, so it weighs a step.
struct WorkSums {
  int blocks, most;        // blocks; the most steps of one
  int weight, weight256;   // steps of all blocks, and in units of 256 (rounded up)
  __host__ __device__ void add(int count, int steps) {
    blocks += count;
    weight += count * (steps > 1 ? steps : 1);
    weight256 += count * (steps > 256 ? (steps + 255) >> 8 : 1);
    if (count > 0 && steps > most) most = steps;
  }
  __host__ __device__ bool units() const { return most >= 65536; }
};

// A piece that leaves no more than `room` items, those that run at once, so that
// the longest sequences, whatever their share of the table, are cut and the
// others are not; kPreLeast steps at least, and `splits` pieces of a sequence at
// most. When the blocks alone are as many, nothing is cut. A block of s >= 1
// steps is ceil(s / piece) <= (s - 1) / piece + 1 items, so all are at most
// (weight - blocks) / piece + blocks; 2^16 steps and more are counted in units.
constexpr int kPreLeast = 4;

__host__ __device__ __forceinline__ int fitting_piece(const WorkSums& all, int room, int splits) {
  if (all.blocks >= room) return all.most > 1 ? all.most : 1;
  int piece = ((all.units() ? all.weight256 : all.weight) - all.blocks) / (room - all.blocks) + 1;
  if (all.units()) piece <<= 8;
  if (piece < kPreLeast) piece = kPreLeast;
  const int least = (all.most + splits - 1) / splits;
  return piece > least ? piece : least;
}

__device__ __forceinline__ WorkScan scan_work(const PrefillParams& p, int lane) {
  WorkScan s;
  s.share = (p.kv.batch + 31) >> 5;
  s.piece = p.piece;
  s.begin = s.count = s.len = 0;
  const int b0 = lane * s.share, b1 = min(p.kv.batch, b0 + s.share);
  WorkSums sums = {0, 0, 0, 0};
  int steps = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    const int mine = blocks_of(p, b, &s.begin, &s.count, &s.len, &steps);
    sums.add(mine, steps);
  }
  auto places = [&](int piece) {  // of this lane's sequences
    if (s.share == 1) return sums.blocks * pieces_of(steps, piece);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
      int begin, count, len, of;
      const int mine = blocks_of(p, b, &begin, &count, &len, &of);
      sum += mine * pieces_of(of, piece);
    }
    return sum;
  };
  if (s.piece == 0) {  // chosen here; every CTA finds the same
    WorkSums all;
    all.most = __reduce_max_sync(0xFFFFFFFFu, sums.most);
    all.blocks = __reduce_add_sync(0xFFFFFFFFu, sums.blocks);
    all.weight = all.weight256 = __reduce_add_sync(0xFFFFFFFFu, all.units() ? sums.weight256 : sums.weight);
    const int room = p.sms / p.kv.kv_heads;
    s.piece = fitting_piece(all, room, p.splits);
    if (all.blocks < room) {
      // The longest sequence in as many pieces, of equal length, if the others
      // allow it.
      const int even = max(kPreLeast, pieces_of(all.most, pieces_of(all.most, s.piece)));
      if (even < s.piece && static_cast<int>(__reduce_add_sync(0xFFFFFFFFu, places(even))) <= room) s.piece = even;
    }
  }
  s.places = places(s.piece);
  s.upto = warp_scan(s.places, lane);
  return s;
}

// Place `index` of the list; called by one warp. First pieces of a sequence
// come first, of them the heavier blocks (later tokens). Up to 32 sequences are
// held in registers; of more, the share that has the place is read again.
// Returns false behind the last place.
__device__ __forceinline__ bool find_work(const PrefillParams& p, const WorkScan& s, int index, int lane, int* seq, int* block,
                                          int* split, int* begin, int* count, int* len) {
  const uint32_t past = __ballot_sync(0xFFFFFFFFu, s.upto > index);
  if (past == 0) return false;
  const int owner = __ffs(past) - 1;
  int before = __shfl_sync(0xFFFFFFFFu, s.upto - s.places, owner);
  int mine = s.places, lo = s.begin, n = s.count, length = s.len, src = owner, from = 0;
  if (s.share > 1) {
    const int end = min(p.kv.batch, (owner + 1) * s.share);
    for (from = owner * s.share;; from += 32) {
      if (from >= end) return false;  // boundaries that do not rise
      mine = 0;
      if (from + lane < end) {
        int steps;
        mine = blocks_of(p, from + lane, &lo, &n, &length, &steps);
        mine *= pieces_of(steps, s.piece);
      }
      const int upto = warp_scan(mine, lane);
      const uint32_t in = __ballot_sync(0xFFFFFFFFu, before + upto > index);
      if (in != 0) {
        src = __ffs(in) - 1;
        before += __shfl_sync(0xFFFFFFFFu, upto - mine, src);
        break;
      }
      before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
  }
  const int at = index - before, places = __shfl_sync(0xFFFFFFFFu, mine, src);
  if (at < 0 || at >= places) return false;  // boundaries that do not rise
  *seq = from + src;
  *begin = __shfl_sync(0xFFFFFFFFu, lo, src);
  *count = __shfl_sync(0xFFFFFFFFu, n, src);
  *len = __shfl_sync(0xFFFFFFFFu, length, src);
  const int blocks = (*count + p.block_tokens - 1) / p.block_tokens;
  *split = -1;
  *block = blocks - 1 - at;
  if (places != blocks) {
    *split = at / blocks;
    *block += *split * blocks;
  }
  return true;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* map, uint64_t* bar, int32_t x, int32_t y, int32_t z,
                                            int32_t w, int32_t v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
      : "memory");
}

// One lane of a converged warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
// The largest of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// D += A B with A (16-bit pairs, one row per lane) in TMEM.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptors of a ring tile: groups of 8 keys, each group D / 64 blocks of
// 8 x 128 bytes (128-byte swizzle), one per 64 elements of the head dimension:
// the order in which one TMA box brings a whole page. As K-major operand (Q
// K^T) a group follows the last after D * 16 bytes, and a block of 64 elements
// starts 1024 bytes after the last one; as N-major operand (P V, the keys are
// the MMA's K dimension) the leading offset is the blocks' distance and the
// stride offset the groups'.
__device__ __forceinline__ uint64_t ring_desc(uint32_t saddr, uint32_t leading, uint32_t group) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(leading >> 4) << 16;
  d |= static_cast<uint64_t>(group >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
constexpr uint32_t kIdescBNMajor = 1u << 16;

// Whether the phase is over, without waiting for it.
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// mbar_wait that goes on after an abort: for what is still in flight.
__device__ __forceinline__ void mbar_wait_bounded(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = global_timer_ns();
  while (!mbar_try_wait(bar, parity))
    if (global_timer_ns() - t0 > kWaitTimeoutNs) return;
}

// One work item.
struct __align__(16) PrefillItem {
  int32_t valid;    // 0: no more work
  int32_t hk;       // kv head
  int32_t split;    // piece; -1: the only one, its rows are results
  int32_t seq, len; // sequence, its keys
  int32_t row0, n;  // its first packed row and its rows
  int32_t tok0;     // first token of the item within them
  int32_t j0, j1;   // steps of the piece
  int32_t end0, end1;  // steps of the tiles within it (j0: none)
};
static_assert(sizeof(PrefillItem) == 48, "items' place in shared memory");

// Asks for a block of the grid that has not started; the answer (16 bytes)
// completes a phase of `bar`.
__device__ __forceinline__ void ask_for_work(void* answer, uint64_t* bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// The block taken over, or -1 when all have started.
__device__ __forceinline__ int work_answer(const void* answer) {
  uint32_t x = 0, ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      ".reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %1, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}\n"
      : "=r"(x), "=r"(ok)
      : "r"(smem_u32(answer))
      : "memory");
  return ok ? static_cast<int>(x) : -1;
}

// kShared: one tile an item, its steps shared by both groups of row warps. (A
// template argument: asked at run time it cost the two-tile form 2.5%.)
template <int D, bool F16, bool kShared>
__global__ void __launch_bounds__(kPreThreads, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                         const PrefillParams p) {
  using Cfg = PrefillCfg<D>;
  // The next scores are computed while the rows work on the last ones: P does
  // not take the place of S, and products of O run behind those of S.
  constexpr bool kAhead = D == 64 && !kShared;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* empty = full + Cfg::kSlots;
  uint64_t* qfull = empty + Cfg::kSlots;
  uint64_t* sfull = qfull + 2;
  uint64_t* pfull = sfull + 2;
  uint64_t* ofull = pfull + 2;
  uint64_t* sread = ofull + 2;
  uint64_t* item_full = sread + 2;
  uint64_t* item_empty = item_full + 2;
  uint64_t* work = item_empty + 2;
  uint64_t* loaded_all = work + 1;
  uint64_t* both = loaded_all + 1;  // shared items: all row warps have come this far
  uint64_t* drain = both + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PrefillItem* items = reinterpret_cast<PrefillItem*>(smem + Cfg::kOffItems);
  void* answer = items + 2;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedView& kv = p.kv;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&qfull[t], kPreRows);
      mbar_init(&sfull[t], 1);
      mbar_init(&pfull[t], kPreRows);
      mbar_init(&ofull[t], 1);
      mbar_init(&sread[t], kPreRows);
      mbar_init(&item_full[t], 1);
      mbar_init(&item_empty[t], 10);  // a lane of each row warp, the loader's and the issuer's
    }
    mbar_init(work, 1);
    mbar_init(loaded_all, 1);
    mbar_init(both, 2 * kPreRows);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();

  // The i-th item of this CTA, copied out of its slot.
  auto get_item = [&](int i, PrefillItem* x) {
    const bool got = __all_sync(0xFFFFFFFFu, mbar_wait(&item_full[i & 1], (i >> 1) & 1, abort_flag));
    if (!got) {
      x->valid = 0;
      return false;
    }
    *x = items[i & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[i & 1]);
    return x->valid != 0;
  };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax rows
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPreRegsRows));
    const int t = warp >> 2;
    // The thread's row, hidden from the compiler: what follows from it outside
    // the steps is computed where it is used instead of being kept in
    // registers across them.
    auto row_of_thread = []() {
      int r = threadIdx.x & 127;
      asm volatile("" : "+r"(r));
      return r;
    };
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t ts = lanes + t * 128, to = lanes + Cfg::kColO + t * D;
    const uint32_t tp = kAhead ? lanes + Cfg::kColP + t * (kPreKeys / 2) : ts;
    const int tile = kShared ? 0 : t;                            // whose rows these are
    const int lag = kShared ? t : 0, stride = kShared ? 2 : 1;  // this group's steps: j0 + lag, by stride
    int met = 0;  // times the groups have waited for each other
    auto meet = [&]() {
      mbar_arrive(both);
      const bool all = __all_sync(0xFFFFFFFFu, mbar_wait(both, met & 1, abort_flag));
      ++met;
      return all;
    };
    // Items stay in their slots while the rows work on them and are read
    // there: a row of S leaves few registers.
    auto wait_item = [&](int i) {
      return __all_sync(0xFFFFFFFFu, mbar_wait(&item_full[i & 1], (i >> 1) & 1, abort_flag)) &&
             items[i & 1].valid != 0;
    };
    auto steps_end = [&](const PrefillItem& x) { return t == 0 ? x.end0 : x.end1; };
    auto has_q = [&](const PrefillItem& x) { return steps_end(x) > x.j0 && (t == 0 || !kShared); };
    // Q tile into shared memory, in the swizzled layout of a TMA box.
    auto load_q = [&](const PrefillItem& x) {
      int r = row_of_thread();
      const int first = x.tok0 + tile * p.tile_tokens;
      const int here = max(0, min(p.tile_tokens, x.n - first)) * p.group;
      const uint32_t dst = smem_u32(smem + t * Cfg::kTileBytes);
      constexpr int kCpr = D / 8;
      const int c = r % kCpr;
      const uint16_t* src =
          static_cast<const uint16_t*>(p.q) + (x.row0 + first) * p.qt + x.hk * p.group * p.qh + c * 8;
#pragma unroll 4
      for (int i = 0; i < kCpr; ++i) {
        const int row = i * (kPreRows / kCpr) + r / kCpr;
        const bool in = row < here;
        const int qtok = in ? row_token(row, p.group_inv) : 0, g = in ? row - qtok * p.group : 0;
        cp_async16(dst + (c >> 3) * Cfg::kBlockBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                   src + qtok * p.qt + g * p.qh, in ? 16u : 0u);
      }
      cp_async_commit();
    };
    auto send_q = [&]() {
      cp_async_wait<0>();
      fence_proxy_async_smem();
      mbar_arrive(&qfull[t]);
    };
    bool ok = wait_item(0);
    int count = 0, used = 0;  // steps and items of this tile so far
    if (ok && has_q(items[0])) {
      load_q(items[0]);
      send_q();
    }
    for (int i = 0; ok; ++i) {
      const PrefillItem& x = items[i & 1];
      const int end = steps_end(x), j0 = x.j0;
      int vis, vis_min;  // keys seen by the row (0: not in use) and by the tile's first token
      {
        const int first = x.tok0 + tile * p.tile_tokens, r = row_of_thread();
        const bool live = r < max(0, min(p.tile_tokens, x.n - first)) * p.group;
        vis = live ? visible_keys(x.len, x.n, first + row_token(r, p.group_inv)) : 0;
        vis_min = visible_keys(x.len, x.n, first);
      }
      float m = -INFINITY, l = 0.f;                         // m: maximum that P refers to (raw scores)
      const int begin = j0 + lag;
      for (int j = begin; j < end; j += stride, ++count) {
        ok = mbar_wait(&sfull[t], count & 1, abort_flag);
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(ts + c * 32, s[c]);
        tmem_ld_wait();
        if (kAhead) {
          tc_fence_before();
          mbar_arrive(&sread[t]);
        }
        if (p.negate) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) s[c][k] ^= 0x80000000u;
        }
        if (vis_min < (j + 1) * kPreKeys) {
          const int lim = vis - j * kPreKeys;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c * 32 + k >= lim) s[c][k] = 0xFF800000u;  // -inf
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = max3(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]), __uint_as_float(s[c][2]));
#pragma unroll
          for (int k = 3; k < 31; k += 2) mx[c] = max3(mx[c], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
          mx[c] = max3(mx[c], __uint_as_float(s[c][31]), m);
        }
        float mn = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);  // NaN if a score is
        // Also true from m = -inf and for NaN, but not while all is -inf.
        const bool raise = !((mn - m) * p.scale_log2 <= kPreLag<F16>) && mn != -INFINITY;
        if (kAhead && j > begin) {  // the last product has read P and written O
          ok = mbar_wait(&ofull[t], (count - 1) & 1, abort_flag) && ok;
          tc_fence_after();
        }
        if (j == begin || __any_sync(0xFFFFFFFFu, raise || !ok)) {
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          if (mn == INFINITY) mn = __int_as_float(0x7FC00000);  // inf - inf: the row is NaN
          const float f = m == -INFINITY ? 0.f : exp2_approx((m - mn) * p.scale_log2);
          m = mn;
          if (j > begin) {
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
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              float2 y = fma2(make_float2(__uint_as_float(s[2 * h + c][k]), __uint_as_float(s[2 * h + c][k + 1])),
                              scale2, shift2);
              y.x = exp2_approx(y.x);
              y.y = exp2_approx(y.y);
              sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], y);
              pk[c * 16 + (k >> 1)] = pack2<F16>(y.x, y.y);
            }
          tmem_st_32x32b_x32(tp + h * 32, pk);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&pfull[t]);
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      // The next item's Q comes while the last product runs (all of this
      // item's Q K^T are done: the rows have seen the last scores; of a shared
      // item they have when both groups' last product is done), if the item is
      // there already.
      const PrefillItem& y = items[(i + 1) & 1];
      const bool early = __all_sync(0xFFFFFFFFu, mbar_test_wait(&item_full[(i + 1) & 1], ((i + 1) >> 1) & 1));
      bool next = early && y.valid != 0;
      const bool soon = next && has_q(y);
      if (soon && !kShared) load_q(y);
      const bool any = end > begin;
      if (any) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&ofull[t], (kAhead ? count - 1 : used) & 1, abort_flag));
        tc_fence_after();
        ++used;
      }
      if (soon && !kShared) send_q();
      if (!ok) break;
      const int first = x.tok0 + tile * p.tile_tokens, r = row_of_thread();
      const int tok = row_token(r, p.group_inv);
      const bool live = r < max(0, min(p.tile_tokens, x.n - first)) * p.group;
      const int head = x.hk * p.group + (r - tok * p.group);
      const int64_t row = x.row0 + first + tok;
      const int64_t at = (row * (kv.kv_heads * p.group) + head) * p.splits + x.split;
      uint16_t* dst = static_cast<uint16_t*>(p.out) + row * p.ot + head * p.oh;
      if (kShared ? end == j0 : !any) {  // no keys
        if (live && (t == 0 || !kShared)) {
          if (x.split < 0)
            for (int k = 0; k < D; k += 8) *reinterpret_cast<uint4*>(dst + k) = make_uint4(0u, 0u, 0u, 0u);
          else
            p.part_ml[at] = make_float2(-INFINITY, 0.f);
        }
        if (soon && kShared) {
          load_q(y);
          send_q();
        }
      } else {
        // Factors of the sums in TMEM: for a tile of its own 1 / l, or 1 when
        // pieces are joined later; for a shared one those of both groups' (m,
        // l), exchanged through the second Q tile's place, and each group takes
        // half the columns.
        int c0 = 0, c1 = D;
        float f0 = 1.f, f1 = 0.f;  // of O 0 (or the tile's own O), of O 1
        if (kShared) {
          float2* swap = reinterpret_cast<float2*>(smem + Cfg::kTileBytes);
          swap[t * kPreRows + r] = make_float2(m, l);
          tc_fence_before();
          ok = meet();
          if (!ok) break;
          tc_fence_after();
          if (soon) load_q(y);
          const float2 a = swap[r], z = swap[kPreRows + r];
          m = fmaxf(a.x, z.x);
          f0 = a.x == -INFINITY ? 0.f : exp2_approx((a.x - m) * p.scale_log2);
          f1 = z.x == -INFINITY ? 0.f : exp2_approx((z.x - m) * p.scale_log2);
          l = a.y * f0 + z.y * f1;
          c0 = t * (D / 2);
          c1 = c0 + D / 2;
        }
        if (x.split >= 0) {
          if (live && c0 == 0) p.part_ml[at] = make_float2(m == -INFINITY ? m : m * p.scale_log2, l);
        } else {
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
          f0 *= inv;
          f1 *= inv;
        }
        const bool add = kShared && end > j0 + 1;  // the second group had a step
        const uint32_t from = kShared ? lanes + Cfg::kColO : to;
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(from + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f0);
          if (add) {
            uint32_t z[32];
            tmem_ld_32x32b_x32(from + D + c, z);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(z[k]), f1, __uint_as_float(o[k])));
          }
          if (!live) continue;
          if (x.split >= 0) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<uint4*>(p.part_o + at * D + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint4 w;
              w.x = pack2<F16>(__uint_as_float(o[k]), __uint_as_float(o[k + 1]));
              w.y = pack2<F16>(__uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
              w.z = pack2<F16>(__uint_as_float(o[k + 4]), __uint_as_float(o[k + 5]));
              w.w = pack2<F16>(__uint_as_float(o[k + 6]), __uint_as_float(o[k + 7]));
              *reinterpret_cast<uint4*>(dst + c + k) = l == 0.f ? make_uint4(0u, 0u, 0u, 0u) : w;
            }
          }
        }
        if (kShared) {
          if (soon) send_q();
          tc_fence_before();
          ok = meet();  // both O are read before either is written again
          if (!ok) break;
        }
      }
      tc_fence_before();  // O is read before the next item's first P is announced
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[i & 1]);
      if (!early) {
        next = wait_item(i + 1);
        if (next && has_q(y)) {
          load_q(y);
          send_q();
        }
      }
      ok = next;
    }
    tc_fence_before();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPreRegsOther));
    if (warp == 8) {
      // ---------------------------------------------------------- page loads
      const int page = 1 << kv.page_shift;
      const int per_step = kPreKeys >> kv.page_shift;
      int issued = 0;  // tiles so far: slot and phase of the ring
      PrefillItem x;
      bool ok = true;
      for (int i = 0; ok && get_item(i, &x); ++i) {
        const int32_t* table = kv.page_table + x.seq * kv.table_stride;
        const int held = (x.len + page - 1) >> kv.page_shift;  // pages of the sequence
        auto entry = [&](int j) {  // a lane per page of the step
          const int at = j * per_step + lane;
          return lane < per_step && at < held ? table[at] : 0;
        };
        // Keys come `lead` steps before the values: K of the first steps, then
        // V and the next K in turn, as the issuer uses them.
        const int lead = kShared || kAhead ? 2 : 1;
        int ids[3];  // table entries of steps j, j + 1, j + 2
#pragma unroll
        for (int k = 0; k < 3; ++k) ids[k] = x.j0 + k < x.j1 ? entry(x.j0 + k) : 0;
        auto load = [&](int j, int id, bool values) {
          const int pieces = min(per_step, held - j * per_step);
          const bool mine = lane < pieces;
          if (!values && mine && (id < 0 || id >= kv.num_pages) && kv.status != nullptr)
            atomicOr(kv.status, ABFT_PAGED_BAD_PAGE);
          const int slot = issued % Cfg::kSlots;
          if (issued >= Cfg::kSlots && !mbar_wait(&empty[slot], (issued / Cfg::kSlots - 1) & 1, abort_flag)) ok = false;
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) return;
          if (lane == 0) mbar_arrive_expect_tx(&full[slot], static_cast<uint32_t>(pieces * page * D * 2));
          __syncwarp();
          if (mine) {
            // A bad id lies outside the map's page dimension and loads zeros.
            const uint32_t dst = smem_u32(smem + Cfg::kOffRing + slot * Cfg::kTileBytes) + lane * page * D * 2;
            tma_load_5d(dst, values ? &tm_v : &tm_k, &full[slot], 0, 0, 0, x.hk << (kv.page_shift - 3), id);
          }
          ++issued;
        };
        if (x.j0 < x.j1) load(x.j0, ids[0], false);
        if (lead == 2 && x.j0 + 1 < x.j1 && ok) load(x.j0 + 1, ids[1], false);
        for (int j = x.j0; j < x.j1 && ok; ++j) {
          load(j, ids[0], true);
          if (j + lead < x.j1 && ok) load(j + lead, lead == 2 ? ids[2] : ids[1], false);
          ids[0] = ids[1];
          ids[1] = ids[2];
          ids[2] = j + 3 < x.j1 ? entry(j + 3) : 0;
        }
        if (lane == 0) mbar_arrive(loaded_all);
      }
      // Copies in flight have landed before shared memory goes (all have, but
      // after an abort).
      for (int it = max(0, issued - Cfg::kSlots); it < issued; ++it)
        mbar_wait_bounded(&full[it % Cfg::kSlots], (it / Cfg::kSlots) & 1);
    } else if (warp == 9) {
      // ---------------------------------------------------------- MMA issuer
      // Control values through a shuffle and one elected lane: the compiler
      // then keeps descriptors in uniform registers. (With values it could
      // not prove uniform each MMA cost 130 clocks to issue, twice its run
      // time.)
      constexpr uint32_t fmt = F16 ? 0u : 1u;
      constexpr uint32_t idesc_s = umma_idesc(kPreRows, kPreKeys, fmt);
      constexpr uint32_t idesc_o = umma_idesc(kPreRows, D, fmt) | kIdescBNMajor;
      const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
      const uint32_t q_base = __shfl_sync(0xFFFFFFFFu, smem_u32(smem), 0);
      const uint64_t desc_q = sw128_kmajor_desc(q_base);
      const uint64_t desc_k = ring_desc(q_base + Cfg::kOffRing, 16, Cfg::kGroupBytes);
      const uint64_t desc_v = ring_desc(q_base + Cfg::kOffRing, 1024, Cfg::kGroupBytes);
      bool ok = true;
      int slot = 0, phase = 0;     // of the next tile in the ring
      int pcount[2] = {0, 0};      // steps of each tile so far
      int qcount[2] = {0, 0};      // items of each tile so far
      auto ready = [&](int at, int ph) {
        ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(&full[at], ph, abort_flag));
        tc_fence_after();
        return ok;
      };
      constexpr int kStride = kShared ? 2 : 1;        // steps between a group's own
      constexpr int kLead = kShared || kAhead ? 2 : 1;  // steps that scores come before the product of O
      auto scores = [&](int t, int at) {
        if (elect_one()) {
          const uint64_t dq = desc_q + (kShared ? 0 : t) * (Cfg::kTileBytes >> 4), dk = desc_k + at * (Cfg::kTileBytes >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            umma_bf16_ss(tm + t * 128, dq + (((k / 4) * Cfg::kBlockBytes + (k % 4) * 32) >> 4),
                         dk + (((k / 4) * 1024 + (k % 4) * 32) >> 4), idesc_s, k > 0);
          }
          umma_commit(&sfull[t]);
        }
        __syncwarp();
      };
      auto seen = [&](int t) {  // the rows have the scores of step pcount[t] in registers
        ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(&sread[t], pcount[t] & 1, abort_flag));
        tc_fence_after();
        return ok;
      };
      auto release = [&](int at) {  // once the MMAs so far have read the slot
        if (elect_one()) umma_commit(&empty[at]);
        __syncwarp();
      };
      auto step_ring = [&]() {
        if (++slot == Cfg::kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      PrefillItem x;
      for (int i = 0; ok && get_item(i, &x); ++i) {
        const int first_j = __shfl_sync(0xFFFFFFFFu, x.j0, 0), last_j = __shfl_sync(0xFFFFFFFFu, x.j1, 0);
        const int stop[2] = {__shfl_sync(0xFFFFFFFFu, x.end0, 0), __shfl_sync(0xFFFFFFFFu, x.end1, 0)};
        const int length = __shfl_sync(0xFFFFFFFFu, x.len, 0);
        if (first_j >= last_j) continue;
        // The first scores of each tile (of a shared item: of its first two
        // steps).
        if (!ready(slot, phase)) break;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (stop[t] > first_j && (t == 0 || !kShared) && ok) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&qfull[t], qcount[t] & 1, abort_flag));
            ++qcount[t];
            tc_fence_after();
            if (ok) scores(t, slot);
          }
        if (!ok) break;
        release(slot);
        step_ring();
        if (kLead == 2 && first_j + 1 < last_j) {
          if (!ready(slot, phase)) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (kShared && t == 0) continue;
            if (kAhead && (first_j + 1 >= stop[t] || !seen(t))) continue;
            scores(t, slot);
          }
          if (!ok) break;
          release(slot);
          step_ring();
        }
        for (int j = first_j; j < last_j && ok; ++j) {
          const int vs = slot;
          if (!ready(vs, phase)) break;
          step_ring();
          // Weights of slots behind the length are 0, but the slots may hold
          // anything (a page's last owner, NaN): only whole groups of 16 keys
          // that the sequence reaches are multiplied, the rest of the last
          // group is cleared.
          const int valid = min(kPreKeys, length - j * kPreKeys);
          const int groups = (valid + 15) / 16;
          if (valid & 15) {
            uint8_t* v = smem + Cfg::kOffRing + vs * Cfg::kTileBytes;
            for (int k = valid * (D / 8) + lane; k < groups * 16 * (D / 8); k += 32) {
              const int row = k / (D / 8), c = k % (D / 8);  // every piece of the row: its order does not matter
              *reinterpret_cast<uint4*>(v + (row >> 3) * Cfg::kGroupBytes + (c >> 3) * 1024 + (row & 7) * 128 +
                                        ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          bool loaded = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (kShared && t != ((j - first_j) & 1)) continue;
            if (j < stop[t] && ok) {
              ok = __all_sync(0xFFFFFFFFu, mbar_wait(&pfull[t], pcount[t] & 1, abort_flag));
              ++pcount[t];
              if (ok) {
                tc_fence_after();
                if (elect_one()) {
                  const uint64_t dv = desc_v + vs * (Cfg::kTileBytes >> 4);
                  const uint32_t d = tm + Cfg::kColO + t * D;
                  const uint32_t a = kAhead ? tm + Cfg::kColP + t * (kPreKeys / 2) : tm + t * 128;
                  umma_f16_ts(d, a, dv, idesc_o, j >= first_j + kStride);
                  if (groups == kPreKeys / 16) {
#pragma unroll
                    for (int k = 1; k < kPreKeys / 16; ++k)
                      umma_f16_ts(d, a + k * 8, dv + k * (2 * Cfg::kGroupBytes >> 4), idesc_o, 1);
                  } else {
                    for (int k = 1; k < groups; ++k)
                      umma_f16_ts(d, a + k * 8, dv + k * (2 * Cfg::kGroupBytes >> 4), idesc_o, 1);
                  }
                  if (kAhead || j + kStride >= stop[t]) umma_commit(&ofull[t]);
                }
                __syncwarp();
              }
            }
            if (j + kLead < stop[t] && ok) {
              if (!loaded) ready(slot, phase);
              loaded = true;
              if (kAhead && ok) seen(t);
              if (ok) scores(t, slot);
            }
          }
          if (!ok) break;
          release(vs);
          if (loaded) {
            release(slot);
            step_ring();
          }
        }
      }
      // Nothing still writes TMEM when it is freed.
      if (elect_one()) umma_commit(drain);
      __syncwarp();
      mbar_wait_bounded(drain, 0);
    } else if (warp == 10) {
      // ---------------------------------------------------------- work
      int index = blockIdx.x, published = 0, asked = 0;
      bool ok = true, first = false;
      const WorkScan scan = scan_work(p, lane);
      // Every CTA writes the same: the join reads it even if the CTA that took an
      // item gave up.
      if (p.chosen != nullptr && lane == 0) *p.chosen = scan.piece;
      while (ok) {
        PrefillItem x;
        x.valid = 0;
        bool publish = index < 0;
        if (index >= 0) {
          first = first || index == 0;
          x.hk = index % kv.kv_heads;
          int seq = 0, block = 0, raw_len = 0;
          if (find_work(p, scan, index / kv.kv_heads, lane, &seq, &block, &x.split, &x.row0, &x.n, &raw_len)) {
            bool bad_len;
            x.seq = seq;
            x.len = paged_clamp_len(raw_len, kv.max_pages, kv.page_shift, &bad_len);
            if ((bad_len || x.len < x.n) && lane == 0 && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_LEN);
            // Steps of each tile (a tile behind the rows' end has none) and of
            // this piece.
            x.tok0 = block * p.block_tokens;
            int steps[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int first = x.tok0 + t * p.tile_tokens;
              const int last = min(min(first + p.tile_tokens, x.n), x.tok0 + p.block_tokens) - 1;
              steps[t] = last >= first ? (visible_keys(x.len, x.n, last) + kPreKeys - 1) / kPreKeys : 0;
            }
            const int most = max(steps[0], steps[1]);
            x.j0 = min(max(x.split, 0) * scan.piece, most);
            x.j1 = min(x.j0 + scan.piece, most);
            x.end0 = max(x.j0, min(x.j1, steps[0]));
            x.end1 = kShared ? x.end0 : max(x.j0, min(x.j1, steps[1]));
            // Without keys the rows still get their zeros when no join follows.
            publish = x.j0 < x.j1 || x.split < 0;
            x.valid = 1;
          }
        }
        if (publish) {
          const int at = published & 1;
          if (published >= 2) ok = __all_sync(0xFFFFFFFFu, mbar_wait(&item_empty[at], ((published >> 1) - 1) & 1, abort_flag));
          if (ok && lane == 0) {
            items[at] = x;
            mbar_arrive(&item_full[at]);
          }
          ++published;
          // The next block is asked for when this item's last tile has been
          // loaded: early enough to find it meanwhile, too late to take one
          // that an idle SM could start.
          if (index >= 0 && ok)
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(loaded_all, (published - 1) & 1, abort_flag));
        }
        if (index < 0 || !ok) break;
        if (lane == 0) ask_for_work(answer, work);
        __syncwarp();
        const bool told = __all_sync(0xFFFFFFFFu, mbar_wait(work, asked & 1, abort_flag));
        ++asked;
        if (!told) {
          mbar_wait_bounded(work, (asked - 1) & 1);  // the answer is not written after shared memory goes
          ok = false;
          break;
        }
        index = work_answer(answer);
        fence_proxy_async_smem();  // read before the next answer is written there
        __syncwarp();
      }
      // By the CTA that had item 0, its own or taken over.
      if (first) check_boundaries(p.cu, kv.batch, p.tokens, lane, kv.status);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_TIMEOUT);
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, Cfg::kTmemCols);
}

// Joins the pieces of each (packed row, head): one warp per row and head,
// D / 32 elements per lane, the pieces in their order.
struct PrefillJoinParams {
  PagedView kv;
  const int32_t* cu;
  void* out;
  int64_t ot, oh;
  int32_t tokens, heads, splits, piece, block_tokens;
  const int32_t* chosen;  // the piece, or NULL: `piece`
  const float* part_o;
  const float2* part_ml;
};
constexpr int kPreJoinWarps = 8;

template <int D, bool F16>
__global__ void __launch_bounds__(32 * kPreJoinWarps) paged_prefill_join_kernel(const PrefillJoinParams p) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  griddep_wait();
  const int index = blockIdx.x * kPreJoinWarps + (threadIdx.x >> 5);
  const int row = index / p.heads, h = index - row * p.heads;
  if (row >= p.tokens) return;
  const int piece = p.chosen != nullptr ? *p.chosen : p.piece;
  const int b = owner_of(p.cu, p.kv.batch, row, lane);
  if (b >= p.kv.batch) return;  // behind the last sequence
  int row0, row_end;
  packed_range(p.cu, b, p.tokens, &row0, &row_end);
  if (row < row0 || row >= row_end) return;
  const int n = row_end - row0;
  bool bad;
  const int len = paged_clamp_len(p.kv.seq_lens[b], p.kv.max_pages, p.kv.page_shift, &bad);
  if (pieces_of((len + kPreKeys - 1) / kPreKeys, piece) == 1) return;  // the row is done
  // Pieces of the row's item.
  const int last = min(((row - row0) / p.block_tokens + 1) * p.block_tokens, n) - 1;
  const int count = ((visible_keys(len, n, last) + kPreKeys - 1) / kPreKeys + piece - 1) / piece;
  const int64_t at = (static_cast<int64_t>(row) * p.heads + h) * p.splits;
  // The maximum of all pieces first, then sums that do not wait for each other.
  float top = -INFINITY;
  for (int s = lane; s < count; s += 32) {
    const float2 ml = p.part_ml[at + s];
    if (ml.y != 0.f) top = fmaxf(top, ml.x);
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, i));
  const float ms = top == -INFINITY ? 0.f : top;
  float l = 0.f, o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = 0.f;
  for (int s0 = 0; s0 < count; s0 += 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (s0 + lane < count) ml = p.part_ml[at + s0 + lane];
    const float f = ml.y == 0.f ? 0.f : exp2_approx(ml.x - ms);
    l += ml.y * f;
    const float2* src = reinterpret_cast<const float2*>(p.part_o + (at + s0) * D + lane * kPer);
    const int most = min(32, count - s0);
#pragma unroll 8
    for (int s = 0; s < most; ++s) {
      const float fs = __shfl_sync(0xFFFFFFFFu, f, s);
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) {
        float2 v = src[s * (D / 2) + i];
        if (fs == 0.f) v = make_float2(0.f, 0.f);  // the row saw nothing there: its sums were not written
        o[2 * i] += v.x * fs;
        o[2 * i + 1] += v.y * fs;
      }
    }
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, i);
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint16_t* dst = static_cast<uint16_t*>(p.out) + row * p.ot + h * p.oh + lane * kPer;
#pragma unroll
  for (int i = 0; i < kPer; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack2<F16>(o[i] * inv, o[i + 1] * inv);
}

}  // namespace abft
