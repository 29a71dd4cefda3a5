// paged_append.cuh - new tokens' keys and values into the paged cache, with
// the rotation by position applied on the way to q and k.
//
// For token t of sequence b at position p, angle pairs (c_j, s_j) = rope[p][j]:
//   x'[j] = x[j] c_j - x[j + D/2] s_j,   x'[j + D/2] = x[j + D/2] c_j + x[j] s_j
// in fp32, rounded once to the element type. The rows are read once and
// written once; there is nothing to reuse, so the kernel is bound by memory
// traffic (large calls) or by its chain of dependent loads (small ones).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/abft_b200.h"
#include "paged_index.cuh"
#include "ptx.cuh"

namespace abft {

// Two packed 16-bit elements <-> two floats.
template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&x));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr int kMostAxes = 4;

struct AppendParams {
  PagedView kv;
  const void *q, *k, *v;
  void* q_out;
  int64_t qt, qh, kt, kh, vt, vh, ot, oh;  // token and head strides, elements
  const int32_t* cu;
  const float* rope;
  int64_t max_positions;
  int64_t tokens;
  int32_t heads;
  int32_t warps_shift;  // log2 of the warps that share a token
};
// With positions of the caller's.
struct AppendAtParams : AppendParams {
  const int32_t* positions;  // [axes][position_stride]: what a token is rotated by, where that is not its slot's place
  int64_t position_stride;
  int32_t axes;
  int32_t axis_end[kMostAxes];  // pairs [axis_end[a - 1], axis_end[a]) turn by axis a
};

// Sequence that owns packed token t: the number of boundaries cu[1..batch]
// at or below t, counted by a whole warp (independent loads instead of a
// chain of a binary search; boundaries do not decrease). Many boundaries are
// first narrowed to the 32nd part that holds t (4 tokens for each of 1,024
// sequences: 10.5 us, 14.9 without). batch when the row is behind the last
// sequence.
constexpr int kOwnerCount = 128;  // boundaries that are counted without narrowing

__device__ __forceinline__ int owner_of(const int32_t* cu, int batch, int64_t t, int lane) {
  int lo = 0, end = batch;  // the answer lies in [lo, end] (in [0, batch] whatever cu holds)
  while (end - lo > kOwnerCount) {
    const int part = (end - lo + 31) / 32, last = lo + lane * part + part - 1;
    const bool below = last < end && cu[1 + last] <= t;
    lo += __popc(__ballot_sync(0xFFFFFFFFu, below)) * part;
    end = min(end, lo + part);
  }
  int n = lo;
  for (int i = lo; i < end; i += 32) {
    const bool below = i + lane < end && cu[1 + i + lane] <= t;
    n += __popc(__ballot_sync(0xFFFFFFFFu, below));
  }
  return n;
}

// One warp of a launch looks at all boundaries; they start at 0, do not fall
// and end within the rows.
__device__ __forceinline__ void check_boundaries(const int32_t* cu, int batch, int64_t tokens, int lane, uint32_t* status) {
  bool bad = false;
  for (int b = lane; b < batch; b += 32) {
    const int lo = cu[b], hi = cu[b + 1];
    bad = bad || hi < lo || hi > tokens || (b == 0 && lo != 0);
  }
  if (bad && status != nullptr) atomicOr(status, ABFT_PAGED_BAD_ROWS);
}

// One thread owns chunk c of a row's pairs: elements [8c, 8c + 8) and their
// partners [D/2 + 8c, D/2 + 8c + 8). D / 16 threads cover a row, a warp 512 / D
// rows of one token. `warps` warps share a token's rows (q's heads, then k's,
// then v's): one when there are tokens enough to fill the SMs, so that the
// angles are read once per token and lane, eight when there are few and the
// chain of dependent loads is what counts.
constexpr int kAppendWarps = 8;
constexpr int kAppendThreads = 32 * kAppendWarps;

// AppendAtParams: the rotation goes by positions of the caller's, of several axes (images
// and video: time, height, width) or one (a drafted token's depth), each for its
// share of the pairs:  (c_j, s_j) = rope[positions[axis of j][t]][j]. They are
// asked for before the chain (sequence, length, page) begins. (Bound by HBM in large
// calls: 10,400 tokens of 36 heads on three axes 34.9 us, 5.6 TB/s, with four CTAs an
// SM; 35.6 with three.)
template <int D, bool F16, typename Params>
__global__ void __launch_bounds__(kAppendThreads, sizeof(Params) > sizeof(AppendParams) ? 4 : 3)
    kv_append_kernel(const Params p) {
  constexpr bool kAxes = sizeof(Params) > sizeof(AppendParams);
  constexpr int kChunks = D / 16;  // threads per row
  griddep_wait();
  constexpr int kRows = 32 / kChunks;  // rows a warp covers at once
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kAppendWarps + (threadIdx.x >> 5);
  const int64_t t = w >> p.warps_shift;
  const int sub = static_cast<int>(w) & ((1 << p.warps_shift) - 1);
  const PagedView& kv = p.kv;
  if (t >= p.tokens) {
    // With boundaries the last block has no row: its first warp checks them.
    if (p.cu != nullptr && blockIdx.x == gridDim.x - 1 && threadIdx.x < 32)
      check_boundaries(p.cu, kv.batch, p.tokens, lane, kv.status);
    return;
  }
  int turn_by[kMostAxes];
  if constexpr (kAxes) {
#pragma unroll
    for (int a = 0; a < kMostAxes; ++a) turn_by[a] = p.positions[(a < p.axes ? a : 0) * p.position_stride + t];
  }
  int b, pos, place = 0, n = 1;
  if (p.cu != nullptr) {
    b = owner_of(p.cu, kv.batch, t, lane);
    if (b >= kv.batch) return;  // behind the last sequence
    int begin, end;
    packed_range(p.cu, b, static_cast<int>(p.tokens), &begin, &end);
    if (t < begin || t >= end) return;  // bad boundaries: the row is no sequence's, or two claim it
    n = end - begin;
    place = static_cast<int>(t) - begin;
  } else {
    b = static_cast<int>(t);
  }
  const int len = kv.seq_lens[b];
  if (p.cu == nullptr && len == 0) return;  // a slot without a sequence
  const int64_t pos64 = static_cast<int64_t>(len) - n + place;
  uint32_t bad = 0;
  if (pos64 < 0 || pos64 >= (static_cast<int64_t>(kv.max_pages) << kv.page_shift)) bad = ABFT_PAGED_BAD_LEN;
  pos = static_cast<int>(pos64);
  if constexpr (kAxes) {
#pragma unroll
    for (int a = 0; a < kMostAxes; ++a)
      if (bad == 0 && (turn_by[a] < 0 || turn_by[a] >= p.max_positions)) bad = ABFT_PAGED_BAD_ANGLE;
  } else {
    if (bad == 0 && p.rope != nullptr && pos >= p.max_positions) bad = ABFT_PAGED_BAD_ANGLE;
  }
  int page = 0;
  if (bad == 0) {
    page = kv.page_table[b * kv.table_stride + (pos >> kv.page_shift)];
    if (page < 0 || page >= kv.num_pages) bad = ABFT_PAGED_BAD_PAGE;
  }
  if (bad != 0) {
    if (lane == 0 && sub == 0 && kv.status != nullptr) atomicOr(kv.status, bad);
    return;
  }
  const int c = lane % kChunks;
  const int slot = pos & ((1 << kv.page_shift) - 1);
  constexpr int kShift = D == 128 ? 7 : 6;
  float cs[16];  // this chunk's (cos, sin) pairs
  if constexpr (kAxes) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pair = 8 * c + i;
      int by = turn_by[0];
#pragma unroll
      for (int a = 1; a < kMostAxes; ++a) by = pair >= p.axis_end[a - 1] ? turn_by[a] : by;
      const float2 x = __ldg(reinterpret_cast<const float2*>(p.rope + static_cast<int64_t>(by) * D) + pair);
      cs[2 * i] = x.x, cs[2 * i + 1] = x.y;
    }
  } else if (p.rope != nullptr) {
    const float4* r = reinterpret_cast<const float4*>(p.rope + static_cast<int64_t>(pos) * D) + c * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = __ldg(r + i);
      cs[4 * i] = x.x, cs[4 * i + 1] = x.y, cs[4 * i + 2] = x.z, cs[4 * i + 3] = x.w;
    }
  }
  // kBatch rows are asked for before the first is written (q_out may be q, so
  // the compiler must not move a load over a store; each thread reads and
  // writes its own elements only). 10,240 tokens of 36 heads of 128: batches of
  // 1 / 2 / 3 / 5: 38.0 / 35.6 / 33.3 / 34.8 us, 5.8 TB/s at 3.
  constexpr int kBatch = 3;
  const int rows = p.heads + 2 * kv.kv_heads;
  const int step = kRows << p.warps_shift;
  for (int r0 = sub * kRows + lane / kChunks; r0 < rows; r0 += kBatch * step) {
    uint4 lo[kBatch], hi[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = r0 + k * step;
      if (r >= rows) break;
      const uint16_t* src;
      if (r < p.heads)
        src = static_cast<const uint16_t*>(p.q) + t * p.qt + r * p.qh;
      else if (r < p.heads + kv.kv_heads)
        src = static_cast<const uint16_t*>(p.k) + t * p.kt + (r - p.heads) * p.kh;
      else
        src = static_cast<const uint16_t*>(p.v) + t * p.vt + (r - p.heads - kv.kv_heads) * p.vh;
      lo[k] = *reinterpret_cast<const uint4*>(src + 8 * c);
      hi[k] = *reinterpret_cast<const uint4*>(src + D / 2 + 8 * c);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = r0 + k * step;
      if (r >= rows) break;
      uint16_t* dst;
      if (r < p.heads)
        dst = static_cast<uint16_t*>(p.q_out) + t * p.ot + r * p.oh;
      else if (r < p.heads + kv.kv_heads)
        dst = static_cast<uint16_t*>(kv.k_pages) +
              paged_offset(page, kv.k_page_stride, r - p.heads, slot, kv.page_shift, kShift);
      else
        dst = static_cast<uint16_t*>(kv.v_pages) +
              paged_offset(page, kv.v_page_stride, r - p.heads - kv.kv_heads, slot, kv.page_shift, kShift);
      if ((kAxes || p.rope != nullptr) && r < p.heads + kv.kv_heads) {
        uint32_t* a = reinterpret_cast<uint32_t*>(&lo[k]);
        uint32_t* z = reinterpret_cast<uint32_t*>(&hi[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = unpack2<F16>(a[i]), y = unpack2<F16>(z[i]);
          const float c0 = cs[4 * i], s0 = cs[4 * i + 1], c1 = cs[4 * i + 2], s1 = cs[4 * i + 3];
          a[i] = pack2<F16>(x.x * c0 - y.x * s0, x.y * c1 - y.y * s1);
          z[i] = pack2<F16>(y.x * c0 + x.x * s0, y.y * c1 + x.y * s1);
        }
      }
      *reinterpret_cast<uint4*>(dst + 8 * c) = lo[k];
      *reinterpret_cast<uint4*>(dst + D / 2 + 8 * c) = hi[k];
    }
  }
}

}  // namespace abft
