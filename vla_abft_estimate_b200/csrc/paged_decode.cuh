// paged_decode.cuh - attention of one new token per sequence over the paged
// cache.
//
//   o_h = sum_j softmax_j(scale q_h . k_j) v_j,   j < length
//
// in one pass with the running maximum m and sum l of the softmax: a tile of
// keys with scores x raises m to m' and scales what was summed by e^(m - m');
// pieces of a sequence carry (m, l, sum e^(x - m) v) and are joined by the
// same rule.
//
// Bound: every key and value is read once, 2 flops per byte and query head of
// its group, so the kernel is bound by HBM. The group's heads share the read:
// they are the N = 8 (or 16) columns of warp-level matrix products
//   S^T [keys x heads] = K Q^T,   O^T [d x heads] += V^T P^T
// whose row side is the keys / the head dimension. This orientation fills
// the instruction's 16 rows with cache data and leaves only the column side
// to padding when a group has fewer than 8 heads; mma.sync suffices, since
// the products need a few per cent of the tensor rate at full HBM speed,
// while one tcgen05 tile would need 128 rows of one operand and a trip of
// the scores through TMEM.
//
// P is rounded to 16 bits for the product, as hi + lo (two products), so
// that the output's own rounding stays the only one that counts: the second
// product hides behind the loads. fp16 ends at 2^-24, and the many keys of a
// long cache may weigh less than that each and still count together: there the
// weights are lifted by 2^15 (the greatest becomes 2^15, within the format), and
// the quotient takes it out again.
//
// Work is one list of 32-key tiles over all (sequence, kv head) segments, cut
// into equal shares for the warps of one CTA per SM: lengths of any mix keep
// every SM reading to the end. (Where lengths differ much a segment takes
// kDecCost places in the list more than it has tiles, for its start and end.) A
// warp's ring of loads runs on across segment boundaries. A segment inside one
// warp's share is finished by that warp; pieces of a segment that crosses warps
// are joined in shared memory, those of one that crosses CTAs by a second, small
// kernel, in a fixed order. (Joined instead by the last CTA to arrive, an atomic
// counter's choice, 37 pieces of 8 heads took one SM 12 us; spread over one block
// per head, launch included, 3 us.)
//
// A cache too small to be worth sharing out so gets a CTA or a cluster of CTAs
// per segment: one launch, and the cluster's pieces are read from each other's
// shared memory (1 sequence of 500 slots and 4 kv heads: 6.5 us, 7.5 by the list).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_append.cuh"
#include "paged_index.cuh"
#include "ptx.cuh"

namespace abft {

__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// 16-byte asynchronous copy; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Transposes an 8x8 block of 16-bit elements held two per lane.
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// D[16 x 8] += A[16 x 16] B[16 x 8], fp32 sums.
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The address of the same place in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(addr), "r"(rank));
  return to;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_f2(uint32_t addr, const float2& v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ void st_cluster_f4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

struct DecodeParams {
  PagedView kv;
  const void* q;
  void* out;
  int64_t qt, qh, ot, oh;  // token and head strides, elements
  int32_t group;           // query heads per kv head
  int32_t head_chunks;     // segments that share a kv head's query heads
  int32_t by_segment;      // CTAs (a cluster) per segment, no pieces in memory, no second kernel; 0: the list
  int32_t cluster_shift;   // log2 of by_segment
  float scale_log2;        // scale * log2(e)
  float* part_o;           // [grid][2][heads of a segment][head_dim]: pieces of segments that cross CTAs
  float2* part_ml;         // [grid][2][heads of a segment] (m, l)
  int4* spill;             // [grid] the segment that starts in this CTA and ends in a later one: (sequence, kv head
                           // and chunk, pieces, -), pieces 0 when there is none
};

// Warps of a CTA and keys of a warp's step. (Eight warps on 16 keys: as fast,
// 128 segments of 2,048 slots 26.1 against 24.6 us, the long list 50.6 against
// 49.5: one SM takes in some 62 GB/s however many warps ask.)
constexpr int kDecWarps = 4;
constexpr int kDecCluster = 8;  // CTAs of a segment at most
constexpr int kDecTile = 32;
// Places in the list that a segment takes for its start and end when the
// longest sequence has over twice the tiles of the shortest: short segments
// would make some shares late (37 sequences of 1 to 4,097 slots: 17.8 us with
// 1, 18.3 with 2, 21.6 with 0). Equal ones divide best without (256 of 2,048
// slots: 44.2 us against 47.9 with 1).
constexpr int kDecCost = 1;
// What the weights are lifted by (a power of 2): fp16's greatest is below 2^16.
template <bool F16>
constexpr float kDecLift = F16 ? 15.f : 0.f;

template <int D, int NT>
struct DecodeCfg {
  static constexpr int kWarps = kDecWarps, kThreads = 32 * kWarps;
  static constexpr int kTile = kDecTile;
  static constexpr int kM = kTile / 16;  // 16-key row blocks of a step
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kRowBytes = D * 2;
  static constexpr int kHalfBytes = kTile * kRowBytes;  // keys of a stage; as much again for values
  static constexpr int kStageBytes = 2 * kHalfBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kHeads = 8 * NT;
  // A piece of a segment: kHeads rows of unnormalised sums (padded against
  // bank conflicts) and (m, l) of each.
  static constexpr int kPitch = D + 4;
  static constexpr int kPieceBytes = kHeads * (kPitch + 2) * 4;
  static_assert(2 * kPieceBytes <= kWarpBytes, "a warp's last piece takes the place of its ring, and the CTA's follows");
  static constexpr int kOffFirst = kWarps * kWarpBytes;  // the warps' first pieces
  static constexpr int kSmemBytes = kOffFirst + kWarps * kPieceBytes;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// A position in the list of tiles.
struct TileIter {
  int u;           // its place in the list
  int b, y;        // sequence; kv head and chunk
  int tile, tiles; // tile within the segment, and the segment's tiles
  int len;
};
constexpr int kNoMore = 0x7FFFFFFF;  // the place behind the last tile

template <int kTile>
__device__ __forceinline__ int tiles_of(const PagedView& kv, int b, int* len, bool* bad) {
  *len = paged_clamp_len(kv.seq_lens[b], kv.max_pages, kv.page_shift, bad);
  return (*len + kTile - 1) / kTile;
}

// The sum of x over this lane and those before it.
__device__ __forceinline__ int warp_scan(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// The next tile; `cost` places lie before a segment's first.
template <int kTile>
__device__ __forceinline__ void advance(TileIter& it, const PagedView& kv, int rows, int cost) {
  if (it.tile + 1 < it.tiles) {
    ++it.tile;
    ++it.u;
    return;
  }
  if (it.y + 1 < rows) {
    ++it.y;
  } else {
    bool bad;
    do {
      if (it.b + 1 >= kv.batch) {
        it.u = kNoMore;
        return;
      }
      ++it.b;
      it.tiles = tiles_of<kTile>(kv, it.b, &it.len, &bad);
    } while (it.tiles == 0);
    it.y = 0;
  }
  it.tile = 0;
  it.u += 1 + cost;
}

template <int D, int NT, bool F16>
__global__ void __launch_bounds__(32 * kDecWarps, 1) paged_decode_kernel(const DecodeParams p) {
  using Cfg = DecodeCfg<D, NT>;
  constexpr int kTile = Cfg::kTile, kWarps = Cfg::kWarps, kM = Cfg::kM;
  extern __shared__ __align__(128) unsigned char smem[];
  // Pieces of segments that cross the warp's share: the first began in an
  // earlier share (0: there is none, 1: the segment ends in this share, 2: it
  // goes on), the last begins here and goes on (0, 2).
  __shared__ int s_first[kWarps], s_last[kWarps];
  __shared__ int s_seg[kWarps][2][2];   // (sequence, kv head and chunk) of first and last
  __shared__ int s_end[kWarps];         // the last's segment: its final tile in the list
  constexpr int kShift = D == 128 ? 7 : 6;
  constexpr int kCpr = D / 8;  // 16-byte pieces of a row
  constexpr int kMt = D / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const PagedView& kv = p.kv;
  const int rows = kv.kv_heads * p.head_chunks;  // segments of a sequence

  griddep_wait();
  griddep_launch();

  // ---- this warp's share ------------------------------------------------------
  TileIter head;
  int total, shares, u0, u1, cost = 0;
  const int rank = static_cast<int>(blockIdx.x) & (p.by_segment - 1);  // of the cluster's CTAs
  if (p.by_segment) {  // the list is one segment, its shares the cluster's warps'
    const int segment = static_cast<int>(blockIdx.x) >> p.cluster_shift;
    head.b = segment / rows;
    head.y = segment - head.b * rows;
    bool bad;
    total = head.tiles = tiles_of<kTile>(kv, head.b, &head.len, &bad);
    if (bad && head.y == 0 && rank == 0 && threadIdx.x == 0 && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_LEN);
    shares = p.by_segment * kWarps;
    u0 = head.u = head.tile = share_start(total, shares, rank * kWarps + warp);
    u1 = share_start(total, shares, rank * kWarps + warp + 1);
  } else {
    // Lane i counts the sequences [i * part, (i + 1) * part): the lane that
    // holds a place is found by one scan, its sequence by another (1,024
    // sequences of up to 700 slots: 58 us, 71 with a scan for each 32).
    const int part = (kv.batch + 31) >> 5;
    int len0 = 0, tiles0 = 0;  // the lane's last sequence: its only one when part is 1
    int sum = 0, held_any = 0, least = kNoMore, most = 0;
#pragma unroll 4
    for (int b = lane * part; b < min(kv.batch, (lane + 1) * part); ++b) {
      bool bad;
      tiles0 = tiles_of<kTile>(kv, b, &len0, &bad);
      if (tiles0 > 0) {
        sum += tiles0;
        ++held_any;
        least = min(least, tiles0);
        most = max(most, tiles0);
      }
      if (bad && blockIdx.x == 0 && warp == 0 && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_LEN);
    }
    least = __reduce_min_sync(0xFFFFFFFFu, least);
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (least < most / 2) cost = kDecCost;
    const int places = sum + cost * held_any;  // of this lane's sequences, for each of their rows
    sum = __reduce_add_sync(0xFFFFFFFFu, places);
    total = sum * rows;  // the host keeps it below 2^31
    shares = gridDim.x * kWarps;
    const int share = blockIdx.x * kWarps + warp;
    u0 = share_start(total, shares, share);
    u1 = share_start(total, shares, share + 1);

    head.u = kNoMore;
    head.b = head.y = head.tile = head.tiles = head.len = 0;
    if (u0 < u1) {  // the sequence that holds place u0
      int upto = warp_scan(places, lane);
      int src = __ffs(__ballot_sync(0xFFFFFFFFu, upto * rows > u0)) - 1;
      int before = __shfl_sync(0xFFFFFFFFu, upto - places, src), from = 0, mine = tiles0, len = len0;
      if (part > 1) {  // which of that lane's sequences
        const int end = min(kv.batch, (src + 1) * part);
        for (from = src * part; from < end; from += 32) {
          bool bad;
          mine = from + lane < end ? tiles_of<kTile>(kv, from + lane, &len, &bad) : 0;
          upto = warp_scan(mine > 0 ? mine + cost : 0, lane);
          const uint32_t past = __ballot_sync(0xFFFFFFFFu, (before + upto) * rows > u0);
          if (past != 0) {
            src = __ffs(past) - 1;
            before += __shfl_sync(0xFFFFFFFFu, upto - (mine > 0 ? mine + cost : 0), src);
            break;
          }
          before += __shfl_sync(0xFFFFFFFFu, upto, 31);
          mine = 0;
        }
      }
      const int tiles = __shfl_sync(0xFFFFFFFFu, mine, src);
      if (tiles > 0) {  // always, unless lengths change under the call
        head.b = from + src;
        head.tiles = tiles;
        head.len = __shfl_sync(0xFFFFFFFFu, len, src);
        const int in = u0 - before * rows;
        head.y = in / (tiles + cost);
        const int off = in - head.y * (tiles + cost);
        head.tile = max(0, off - cost);
        head.u = u0 - off + cost + head.tile;  // the first tile at or behind u0
      }
    }
  }

  const uint32_t ring = smem_u32(smem) + warp * Cfg::kWarpBytes;
  const uint16_t* kbase = static_cast<const uint16_t*>(kv.k_pages);
  const uint16_t* vbase = static_cast<const uint16_t*>(kv.v_pages);

  // Lane i holds the table entry of 16 keys, the i-th from tile `held` on: one
  // load serves 512 keys, and the next 512 are asked for ahead of their use.
  constexpr int kHeld = 32 / kM;  // tiles of a load
  int entry = 0, entry_next = 0, held = 0;
  auto look_up = [&](const TileIter& it, int tile) {
    const int key = tile * kTile + lane * 16;
    return key < it.len ? kv.page_table[it.b * kv.table_stride + (key >> kv.page_shift)] : 0;
  };
  auto entries = [&](const TileIter& it) {  // of a segment that begins
    held = it.tile;
    entry = look_up(it, held);
    entry_next = look_up(it, held + kHeld);
  };
  auto issue = [&](const TileIter& it, int stage) {
    constexpr int kRowsPerOp = 32 / kCpr;  // rows one warp-wide copy covers
    const int sub = lane / kCpr, c = lane % kCpr;
    const int hk = p.head_chunks == 1 ? it.y : it.y / p.head_chunks;
#pragma unroll
    for (int i = 0; i < kM; ++i) {
      const int key0 = it.tile * kTile + i * 16;
      const int page = __shfl_sync(0xFFFFFFFFu, entry, kM * (it.tile - held) + i);
      const bool ok = page >= 0 && page < kv.num_pages;
      if (!ok && lane == 0 && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_PAGE);
      const int slot = key0 & ((1 << kv.page_shift) - 1);
      const int64_t ko = ok ? paged_offset(page, kv.k_page_stride, hk, slot, kv.page_shift, kShift) : 0;
      const int64_t vo = ok ? paged_offset(page, kv.v_page_stride, hk, slot, kv.page_shift, kShift) : 0;
#pragma unroll
      for (int j = 0; j < 16 / kRowsPerOp; ++j) {
        const int r = j * kRowsPerOp + sub;  // row within the half
        const uint32_t bytes = (ok && key0 + r < it.len) ? 16u : 0u;
        const int row = bytes ? r : 0;
        const uint32_t dst = ring + stage * Cfg::kStageBytes + (i * 16 + r) * Cfg::kRowBytes + ((c ^ (r & 7)) << 4);
        cp_async16(dst, kbase + ko + row * D + c * 8, bytes);
        cp_async16(dst + Cfg::kHalfBytes, vbase + vo + row * D + c * 8, bytes);
      }
    }
  };

  float o[kMt][NT][4];
  float m[NT][2], l[NT][2];
  uint32_t qf[NT][D / 16][2];  // Q^T fragments: column g = head, rows = head dimension
  auto load_q = [&](const TileIter& it, uint32_t (&to)[NT][D / 16][2]) {
    const int hk = it.y / p.head_chunks, hc = it.y - hk * p.head_chunks;
    const int nheads = min(Cfg::kHeads, p.group - hc * Cfg::kHeads);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const uint16_t* src =
          static_cast<const uint16_t*>(p.q) + it.b * p.qt + (hk * p.group + hc * Cfg::kHeads + h) * p.qh;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          to[nt][ks][i] = h < nheads ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + i * 8 + tq * 2) : 0u;
    }
  };
  auto begin_segment = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][nt][i] = 0.f;
    }
  };
  // Sums of l over the lanes that hold other keys of the same head.
  auto fold_l = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], 16);
      }
  };
  auto store_piece = [&](unsigned char* at) {
    float* row = reinterpret_cast<float*>(at);
    float2* ml = reinterpret_cast<float2*>(row + Cfg::kHeads * Cfg::kPitch);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = nt * 8 + tq * 2 + e;
        if (g == 0) ml[h] = make_float2(m[nt][e], l[nt][e]);
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) {
          row[h * Cfg::kPitch + mt * 16 + g] = o[mt][nt][e];
          row[h * Cfg::kPitch + mt * 16 + g + 8] = o[mt][nt][2 + e];
        }
      }
  };

  TileIter cur = head;  // consumer; `head` runs kStages - 1 tiles ahead
  if (lane == 0) s_first[warp] = s_last[warp] = 0;
  if (cur.u < u1) {
    entries(head);
    load_q(cur, qf);
    begin_segment();
    bool from_before = cur.tile > 0;  // the segment began in an earlier share
    int stage = 0;
    auto fill = [&](int sn) {
      if (head.u < u1) {
        issue(head, sn);
        advance<kTile>(head, kv, rows, cost);
        if (head.u < u1) {
          if (head.tile == 0) {
            entries(head);
          } else if (head.tile - held == kHeld) {
            held += kHeld;
            entry = entry_next;
            entry_next = look_up(head, held + kHeld);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll 1
    for (int s = 0; s < Cfg::kStages - 1; ++s) fill(s);
    while (true) {
      cp_async_wait<Cfg::kStages - 2>();
      __syncwarp();
      // Refill the stage that the previous step emptied.
      fill(stage == 0 ? Cfg::kStages - 1 : stage - 1);
      // The next segment's query rows are asked for under this one's last step.
      const bool ends = cur.tile + 1 == cur.tiles;
      uint32_t qn[NT][D / 16][2];
      TileIter next = cur;
      advance<kTile>(next, kv, rows, cost);
      const bool stops = next.u >= u1;
      if (ends && !stops) load_q(next, qn);
      const uint32_t ks_base = ring + stage * Cfg::kStageBytes;
      const uint32_t vs_base = ks_base + Cfg::kHalfBytes;

      float s[kM][NT][4];
#pragma unroll
      for (int mt = 0; mt < kM; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mt][nt][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int mt = 0; mt < kM; ++mt) {
          const int r = mt * 16 + (lane & 15);
          const int c = ks * 2 + (lane >> 4);
          uint32_t a[4];
          ldsm_x4(a, ks_base + r * Cfg::kRowBytes + ((c ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<F16>(s[mt][nt], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
      }

      // Scores in units of log2(e); keys behind the length drop out.
      const int key_g = cur.tile * kTile + g;
      const bool ragged = cur.tile * kTile + kTile > cur.len;
      float scale[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < kM; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float& x = s[mt][nt][half * 2 + e];
              x *= p.scale_log2;
              if (ragged && key_g + mt * 16 + half * 8 >= cur.len) x = -INFINITY;
              top = fmaxf(top, x);
            }
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
          const float mn = fmaxf(m[nt][e], top);
          const float ms = mn == -INFINITY ? 0.f : mn;  // nothing but -inf so far: weights 0, not NaN
          const float base = ms - kDecLift<F16>;
          scale[nt][e] = exp2_approx(m[nt][e] - ms);
          m[nt][e] = mn;
          float sum_p = 0.f;
#pragma unroll
          for (int mt = 0; mt < kM; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float& x = s[mt][nt][half * 2 + e];
              x = exp2_approx(x - base);
              sum_p += x;
            }
          l[nt][e] = l[nt][e] * scale[nt][e] + sum_p;
        }
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) {
          o[mt][nt][0] *= scale[nt][0];
          o[mt][nt][1] *= scale[nt][1];
          o[mt][nt][2] *= scale[nt][0];
          o[mt][nt][3] *= scale[nt][1];
        }
      }

      // P^T fragments (column = head), hi and lo terms, by 16 keys.
      uint32_t ph[kM][NT][2], pl[kM][NT][2];
#pragma unroll
      for (int kk = 0; kk < kM; ++kk)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float x = s[kk][nt][half * 2], y = s[kk][nt][half * 2 + 1];
            const uint32_t hi = pack2<F16>(x, y);
            const float2 back = unpack2<F16>(hi);
            ph[kk][nt][half] = movm_t(hi);
            pl[kk][nt][half] = movm_t(pack2<F16>(x - back.x, y - back.y));
          }
#pragma unroll
      for (int kk = 0; kk < kM; ++kk)
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) {
          const int r = kk * 16 + (lane & 7) + ((lane >> 4) << 3);
          const int c = mt * 2 + ((lane >> 3) & 1);
          uint32_t a[4];
          ldsm_x4_t(a, vs_base + r * Cfg::kRowBytes + ((c ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_16816<F16>(o[mt][nt], a, ph[kk][nt][0], ph[kk][nt][1]);
            mma_16816<F16>(o[mt][nt], a, pl[kk][nt][0], pl[kk][nt][1]);
          }
        }
      __syncwarp();  // every lane has read the stage before it is refilled
      if (++stage == Cfg::kStages) stage = 0;

      if (ends || stops) {
        fold_l();
        if (from_before) {
          store_piece(smem + Cfg::kOffFirst + warp * Cfg::kPieceBytes);
          if (lane == 0) {
            s_first[warp] = ends ? 1 : 2;
            s_seg[warp][0][0] = cur.b;
            s_seg[warp][0][1] = cur.y;
          }
        } else if (!ends) {
          cp_async_wait<0>();
          __syncwarp();
          store_piece(smem + warp * Cfg::kWarpBytes);
          if (lane == 0) {
            s_last[warp] = 2;
            s_seg[warp][1][0] = cur.b;
            s_seg[warp][1][1] = cur.y;
            s_end[warp] = cur.u + (cur.tiles - 1 - cur.tile);
          }
        } else {  // the whole segment: its rows are done
          const int hk = cur.y / p.head_chunks, hc = cur.y - hk * p.head_chunks;
          const int nheads = min(Cfg::kHeads, p.group - hc * Cfg::kHeads);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float inv[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
              inv[e] = l[nt][e] > 0.f ? 1.f / l[nt][e] : (l[nt][e] == 0.f ? 0.f : l[nt][e]);
            uint16_t* dst = static_cast<uint16_t*>(p.out) + cur.b * p.ot +
                            (hk * p.group + hc * Cfg::kHeads + nt * 8 + g) * p.oh + tq * 2;
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                // (element g; heads 2tq, 2tq + 1) to (head g; elements 2tq, 2tq + 1)
                const uint32_t x =
                    movm_t(pack2<F16>(o[mt][nt][half * 2] * inv[0], o[mt][nt][half * 2 + 1] * inv[1]));
                if (nt * 8 + g < nheads) *reinterpret_cast<uint32_t*>(dst + mt * 16 + half * 8) = x;
              }
          }
        }
        if (stops) break;
      }
      cur = next;
      if (ends) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) qf[nt][ks][0] = qn[nt][ks][0], qf[nt][ks][1] = qn[nt][ks][1];
        begin_segment();
        from_before = false;
      }
    }
  }
  cp_async_wait<0>();
  // Sequences without tokens: rows of zeros.
  for (int b = blockIdx.x; b < kv.batch; b += gridDim.x) {
    int len;
    bool bad;
    if (tiles_of<kTile>(kv, b, &len, &bad) == 0)
      for (int i = threadIdx.x; i < kv.kv_heads * p.group * kCpr; i += Cfg::kThreads)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + b * p.ot + (i / kCpr) * p.oh + (i % kCpr) * 8) =
            make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();

  // ---- pieces that cross warps ------------------------------------------------
  // A chain is a last piece and the first pieces of the following warps as far
  // as the segment goes; the chain before warp 0 lacks its start (in an earlier
  // CTA). 16 threads take a head, each D / 16 of its elements, and read all
  // pieces at once.
  // The CTA's piece for the others of its cluster.
  float* piece = reinterpret_cast<float*>(smem + Cfg::kPieceBytes);
  float2* piece_ml = reinterpret_cast<float2*>(piece + Cfg::kHeads * Cfg::kPitch);
  if (p.by_segment > 1 && s_first[0] == 0 && s_last[0] == 0 && threadIdx.x < Cfg::kHeads)
    piece_ml[threadIdx.x] = make_float2(-INFINITY, 0.f);  // no share, or the whole segment
  int over = -1;  // warp whose last piece goes on in the next CTA
#pragma unroll 1
  for (int w = -1; w < kWarps; ++w) {
    if (w < 0 ? s_first[0] == 0 : s_last[w] == 0) continue;
    int to = w + 1;
    bool on = true;
    while (to < kWarps && on) on = s_first[to++] == 2;
    const int b = w < 0 ? s_seg[0][0][0] : s_seg[w][1][0], y = w < 0 ? s_seg[0][0][1] : s_seg[w][1][1];
    const int hk = y / p.head_chunks, hc = y - hk * p.head_chunks;
    const int nheads = min(Cfg::kHeads, p.group - hc * Cfg::kHeads);
    const bool whole = w >= 0 && !on;
    if (w >= 0 && on) over = w;
    const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (w < 0 ? 0 : 1)) * Cfg::kHeads;
    constexpr int kPer = D / 16;
    const int d = (threadIdx.x & 15) * kPer;
#pragma unroll 1
    for (int h = threadIdx.x >> 4; h < nheads; h += Cfg::kThreads / 16) {
      const float* at[kWarps + 1];  // the last piece of warp w, the first pieces of warps w + 1 .. to - 1
      float2 ml[kWarps + 1];
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k <= kWarps; ++k) {
        const bool used = k == 0 ? w >= 0 : (k - 1 > w && k - 1 < to);
        at[k] = reinterpret_cast<const float*>(k == 0 ? smem + max(w, 0) * Cfg::kWarpBytes
                                                      : smem + Cfg::kOffFirst + (k - 1) * Cfg::kPieceBytes);
        ml[k] = make_float2(-INFINITY, 0.f);
        if (used) ml[k] = reinterpret_cast<const float2*>(at[k] + Cfg::kHeads * Cfg::kPitch)[h];
        if (!used) at[k] = nullptr;
        top = fmaxf(top, ml[k].x);
      }
      const float ms = top == -INFINITY ? 0.f : top;
      float l_sum = 0.f, x[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = 0.f;
#pragma unroll
      for (int k = 0; k <= kWarps; ++k) {
        if (at[k] == nullptr) continue;
        const float f = exp2_approx(ml[k].x - ms);
        l_sum += ml[k].y * f;
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(at[k] + h * Cfg::kPitch + d + i);
          x[i] += v.x * f;
          x[i + 1] += v.y * f;
          x[i + 2] += v.z * f;
          x[i + 3] += v.w * f;
        }
      }
      if (whole) {
        const float inv = l_sum > 0.f ? 1.f / l_sum : (l_sum == 0.f ? 0.f : l_sum);
        uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.ot + (hk * p.group + hc * Cfg::kHeads + h) * p.oh + d;
#pragma unroll
        for (int i = 0; i < kPer; i += 4)
          *reinterpret_cast<uint2*>(dst + i) =
              make_uint2(pack2<F16>(x[i] * inv, x[i + 1] * inv), pack2<F16>(x[i + 2] * inv, x[i + 3] * inv));
      } else {
        float* dst = p.by_segment ? piece + h * Cfg::kPitch + d : p.part_o + (slot + h) * D + d;
#pragma unroll
        for (int i = 0; i < kPer; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        if (d == 0) (p.by_segment ? piece_ml + h : p.part_ml + slot + h)[0] = make_float2(top, l_sum);
      }
    }
  }
  if (p.by_segment) {
    if (p.by_segment == 1) return;
    // The cluster's pieces, in the order of its CTAs; each CTA joins every
    // by_segment-th head, D / 2 threads a head.
    cluster_barrier();
    const bool in_first = share_start(total, shares, kWarps) >= total;  // joined already
    const int b = blockIdx.x / (rows << p.cluster_shift), y = (blockIdx.x >> p.cluster_shift) - b * rows;
    const int hk = y / p.head_chunks, hc = y - hk * p.head_chunks;
    const int nheads = in_first ? 0 : min(Cfg::kHeads, p.group - hc * Cfg::kHeads);
    const int d = (threadIdx.x % (D / 2)) * 2;
    for (int h = rank + (threadIdx.x / (D / 2) << p.cluster_shift); h < nheads;
         h += (Cfg::kThreads / (D / 2)) << p.cluster_shift) {
      const uint32_t at = smem_u32(piece + h * Cfg::kPitch + d), at_ml = smem_u32(piece_ml + h);
      float2 ml[kDecCluster], v[kDecCluster];
      float top = -INFINITY;
#pragma unroll
      for (int r = 0; r < kDecCluster; ++r) {
        ml[r] = make_float2(-INFINITY, 0.f);
        if (r < p.by_segment) {
          ml[r] = ld_cluster_f2(map_rank(at_ml, r));
          v[r] = ld_cluster_f2(map_rank(at, r));
        }
        top = fmaxf(top, ml[r].x);
      }
      const float ms = top == -INFINITY ? 0.f : top;
      float l_sum = 0.f, x = 0.f, z = 0.f;
#pragma unroll
      for (int r = 0; r < kDecCluster; ++r) {
        if (ml[r].y == 0.f) continue;  // no piece: v was not written
        const float f = exp2_approx(ml[r].x - ms);
        l_sum += ml[r].y * f;
        x += v[r].x * f;
        z += v[r].y * f;
      }
      const float inv = l_sum > 0.f ? 1.f / l_sum : (l_sum == 0.f ? 0.f : l_sum);
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + b * p.ot + (hk * p.group + hc * Cfg::kHeads + h) * p.oh +
                                   d) = pack2<F16>(x * inv, z * inv);
    }
    cluster_barrier();  // shared memory stays until it has been read
    return;
  }
  if (threadIdx.x == 0) {
    int4 spill = make_int4(0, 0, 0, 0);
    if (over >= 0)
      spill = make_int4(s_seg[over][1][0], s_seg[over][1][1],
                        share_of(total, shares, s_end[over]) / kWarps - static_cast<int>(blockIdx.x) + 1, 0);
    p.spill[blockIdx.x] = spill;
  }
}

// Joins the segments that cross CTAs: block (c, h) takes head h of the
// segment that starts in CTA c and ends in a later one; its pieces are CTA
// c's second slot and the following CTAs' first ones. Each warp takes every
// eighth piece.
struct JoinParams {
  void* out;
  int64_t ot, oh;
  int32_t group, head_chunks;
  const float* part_o;
  const float2* part_ml;
  const int4* spill;
};
constexpr int kJoinWarps = 8;

template <int D, int NT, bool F16>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_kernel(const JoinParams p) {
  constexpr int kHeads = DecodeCfg<D, NT>::kHeads;
  constexpr int kPer = D / 32;
  __shared__ float so[kJoinWarps][D];
  __shared__ float2 sml[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x, h = blockIdx.y;
  griddep_wait();
  griddep_launch();
  const int4 seg = p.spill[c];
  if (seg.z == 0) return;
  const int hk = seg.y / p.head_chunks, hc = seg.y - hk * p.head_chunks;
  if (hc * kHeads + h >= p.group) return;
  float m = -INFINITY, l = 0.f, o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = 0.f;
  // Five pieces at a time, all asked for before the first is used.
  constexpr int kAtOnce = 5;
#pragma unroll 1
  for (int s0 = warp; s0 < seg.z; s0 += kAtOnce * kJoinWarps) {
    float2 ml[kAtOnce], v[kAtOnce][kPer / 2];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int s = s0 + k * kJoinWarps;
      const int64_t at = (static_cast<int64_t>(c + s) * 2 + (s == 0 ? 1 : 0)) * kHeads + h;
      const bool in = s < seg.z;
      ml[k] = in ? p.part_ml[at] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i)
        v[k][i] = in ? reinterpret_cast<const float2*>(p.part_o + at * D + lane * kPer)[i] : make_float2(0.f, 0.f);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) mn = fmaxf(mn, ml[k].x);
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float f0 = exp2_approx(m - ms);
    m = mn;
    l *= f0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] *= f0;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float f = exp2_approx(ml[k].x - ms);
      l += ml[k].y * f;
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) {
        o[2 * i] += v[k][i].x * f;
        o[2 * i + 1] += v[k][i].y * f;
      }
    }
  }
  if (lane == 0) sml[warp] = make_float2(m, l);
#pragma unroll
  for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = o[i];
  __syncthreads();
  if (threadIdx.x < D / 2) {
    const int d = threadIdx.x * 2;
    float top = sml[0].x;
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) top = fmaxf(top, sml[w].x);
    const float ms = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      const float f = exp2_approx(sml[w].x - ms);
      sum += sml[w].y * f;
      x += so[w][d] * f;
      y += so[w][d + 1] * f;
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + seg.x * p.ot +
                                 (hk * p.group + hc * kHeads + h) * p.oh + d) = pack2<F16>(x * inv, y * inv);
  }
}

}  // namespace abft
