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
// product hides behind the loads.
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

struct DecodeParams {
  PagedView kv;
  const void* q;
  void* out;
  int64_t qt, qh, ot, oh;  // token and head strides, elements
  int32_t group;           // query heads per kv head
  int32_t head_chunks;     // CTAs that share a kv head's query heads
  int32_t splits;
  float scale_log2;        // scale * log2(e)
  float* part_o;           // [batch * heads][splits][head_dim]
  float2* part_ml;         // [batch * heads][splits] (m, l)
};

constexpr int kDecTile = 32;  // keys of one warp step

template <int D, int NT>
struct DecodeCfg {
  static constexpr int kWarps = 4;
  static constexpr int kStages = 3;
  static constexpr int kRowBytes = D * 2;
  static constexpr int kHalfBytes = kDecTile * kRowBytes;  // keys of a stage; as much again for values
  static constexpr int kStageBytes = 2 * kHalfBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kHeads = 8 * NT;
  static constexpr int kJoinPitch = D + 4;  // floats of one head's row when the warps join
  static constexpr int kRingBytes = kWarps * kWarpBytes;
  static constexpr int kJoinBytes = kWarps * kHeads * (kJoinPitch + 2) * 4;
  static constexpr int kSmemBytes = (kRingBytes > kJoinBytes ? kRingBytes : kJoinBytes);
};

// Grid: (splits, kv_heads * head_chunks, batch). A warp owns every fourth
// 32-key tile of its CTA's piece, with a private ring of cp.async stages:
// no block-wide barrier before the warps join.
template <int D, int NT, bool F16>
__global__ void __launch_bounds__(128) paged_decode_kernel(const DecodeParams p) {
  using Cfg = DecodeCfg<D, NT>;
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int kShift = D == 128 ? 7 : 6;
  constexpr int kCpr = D / 8;  // 16-byte pieces of a row
  constexpr int kMt = D / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const PagedView& kv = p.kv;
  const int b = blockIdx.z, split = blockIdx.x;
  const int hk = blockIdx.y / p.head_chunks, hc = blockIdx.y - hk * p.head_chunks;
  const int heads = kv.kv_heads * p.group;
  const int head0 = hk * p.group + hc * Cfg::kHeads;
  const int nheads = min(Cfg::kHeads, p.group - hc * Cfg::kHeads);

  griddep_wait();
  griddep_launch();
  bool bad_len;
  const int len = paged_clamp_len(kv.seq_lens[b], kv.max_pages, kv.page_shift, &bad_len);
  if (bad_len && threadIdx.x == 0 && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_LEN);
  const int tiles = (len + kDecTile - 1) / kDecTile;
  int t0, t1;
  split_tiles(tiles, p.splits, split, &t0, &t1);
  if (t0 >= t1 && (p.splits > 1 || tiles > 0)) return;

  // Q^T fragments: column g = head, rows = head dimension.
  uint32_t qf[NT][D / 16][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + g;
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + b * p.qt + (head0 + h) * p.qh;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qf[nt][ks][i] = h < nheads ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + i * 8 + tq * 2) : 0u;
  }

  const uint32_t ring = smem_u32(smem) + warp * Cfg::kWarpBytes;
  const int32_t* table = kv.page_table + b * kv.table_stride;
  const uint16_t* kbase = static_cast<const uint16_t*>(kv.k_pages);
  const uint16_t* vbase = static_cast<const uint16_t*>(kv.v_pages);

  // Table entries of the two 16-key halves of tile t (-1: nothing to read).
  auto entries = [&](int t, int (&pg)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = t * kDecTile + i * 16;
      pg[i] = (t < t1 && key < len) ? table[key >> kv.page_shift] : -1;
    }
  };
  auto issue = [&](int t, int stage, const int (&pg)[2]) {
    constexpr int kRowsPerOp = 32 / kCpr;  // rows one warp-wide copy covers
    const int sub = lane / kCpr, c = lane % kCpr;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key0 = t * kDecTile + i * 16;
      bool ok = pg[i] >= 0 && pg[i] < kv.num_pages;
      if (!ok && t < t1 && key0 < len && lane == 0 && kv.status != nullptr) atomicOr(kv.status, ABFT_PAGED_BAD_PAGE);
      const int slot = key0 & ((1 << kv.page_shift) - 1);
      const int64_t ko = ok ? paged_offset(pg[i], kv.k_page_stride, hk, slot, kv.page_shift, kShift) : 0;
      const int64_t vo = ok ? paged_offset(pg[i], kv.v_page_stride, hk, slot, kv.page_shift, kShift) : 0;
#pragma unroll
      for (int j = 0; j < 16 / kRowsPerOp; ++j) {
        const int r = j * kRowsPerOp + sub;  // row within the half
        const uint32_t bytes = (ok && key0 + r < len) ? 16u : 0u;
        const int row = bytes ? r : 0;
        const uint32_t dst = ring + stage * Cfg::kStageBytes + (i * 16 + r) * Cfg::kRowBytes + ((c ^ (r & 7)) << 4);
        cp_async16(dst, kbase + ko + row * D + c * 8, bytes);
        cp_async16(dst + Cfg::kHalfBytes, vbase + vo + row * D + c * 8, bytes);
      }
    }
  };

  float o[kMt][NT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[mt][nt][i] = 0.f;
  }

  int pg[2];
  const int first = t0 + warp;
#pragma unroll
  for (int s = 0; s < Cfg::kStages - 1; ++s) {
    const int t = first + s * Cfg::kWarps;
    entries(t, pg);
    if (t < t1) issue(t, s, pg);
    cp_async_commit();
  }
  entries(first + (Cfg::kStages - 1) * Cfg::kWarps, pg);

  int stage = 0;
  for (int t = first; t < t1; t += Cfg::kWarps) {
    cp_async_wait<Cfg::kStages - 2>();
    __syncwarp();
    // Refill the stage that the previous step emptied.
    {
      const int tn = t + (Cfg::kStages - 1) * Cfg::kWarps;
      int sn = stage + Cfg::kStages - 1;
      if (sn >= Cfg::kStages) sn -= Cfg::kStages;
      if (tn < t1) issue(tn, sn, pg);
      cp_async_commit();
      entries(tn + Cfg::kWarps, pg);
    }
    const uint32_t ks_base = ring + stage * Cfg::kStageBytes;
    const uint32_t vs_base = ks_base + Cfg::kHalfBytes;

    float s[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[mt][nt][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int r = mt * 16 + (lane & 15);
        const int c = ks * 2 + (lane >> 4);
        uint32_t a[4];
        ldsm_x4(a, ks_base + r * Cfg::kRowBytes + ((c ^ (r & 7)) << 4));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816<F16>(s[mt][nt], a, qf[nt][ks][0], qf[nt][ks][1]);
      }
    }

    // Scores in units of log2(e); keys behind the length drop out.
    const int key_g = t * kDecTile + g;
    const bool ragged = t * kDecTile + kDecTile > len;
    float scale[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float& x = s[mt][nt][half * 2 + e];
            x *= p.scale_log2;
            if (ragged && key_g + mt * 16 + half * 8 >= len) x = -INFINITY;
            top = fmaxf(top, x);
          }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
        const float mn = fmaxf(m[nt][e], top);
        const float ms = mn == -INFINITY ? 0.f : mn;  // nothing but -inf so far: weights 0, not NaN
        scale[nt][e] = exp2_approx(m[nt][e] - ms);
        m[nt][e] = mn;
        float sum = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float& x = s[mt][nt][half * 2 + e];
            x = exp2_approx(x - ms);
            sum += x;
          }
        l[nt][e] = l[nt][e] * scale[nt][e] + sum;
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
    uint32_t ph[2][NT][2], pl[2][NT][2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
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
    for (int kk = 0; kk < 2; ++kk)
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
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings become the join area

  float* jo = reinterpret_cast<float*>(smem);                       // [warp][head][pitch]
  float2* jml = reinterpret_cast<float2*>(jo + Cfg::kWarps * Cfg::kHeads * Cfg::kJoinPitch);  // [warp][head]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[nt][e];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
      const int h = nt * 8 + tq * 2 + e;
      if (g == 0) jml[warp * Cfg::kHeads + h] = make_float2(m[nt][e], sum);
      float* row = jo + (warp * Cfg::kHeads + h) * Cfg::kJoinPitch;
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) {
        row[mt * 16 + g] = o[mt][nt][e];
        row[mt * 16 + g + 8] = o[mt][nt][2 + e];
      }
    }
  __syncthreads();
  // Two elements per thread and step.
  for (int i = threadIdx.x; i < nheads * (D / 2); i += 128) {
    const int h = i / (D / 2), d = (i % (D / 2)) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < Cfg::kWarps; ++w) top = fmaxf(top, jml[w * Cfg::kHeads + h].x);
    const float ms = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < Cfg::kWarps; ++w) {
      const float2 ml = jml[w * Cfg::kHeads + h];
      const float f = exp2_approx(ml.x - ms);
      sum += ml.y * f;
      const float2 v = *reinterpret_cast<const float2*>(jo + (w * Cfg::kHeads + h) * Cfg::kJoinPitch + d);
      x += v.x * f;
      y += v.y * f;
    }
    if (p.splits == 1) {
      const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.ot + (head0 + h) * p.oh + d;
      *reinterpret_cast<uint32_t*>(dst) = pack2<F16>(x * inv, y * inv);
    } else {
      const int64_t row = (static_cast<int64_t>(b) * heads + head0 + h) * p.splits + split;
      *reinterpret_cast<float2*>(p.part_o + row * D + d) = make_float2(x, y);
      if (d == 0) p.part_ml[row] = make_float2(top, sum);
    }
  }
}

// Joins the pieces of each (sequence, head): grid (heads, batch), one warp
// per fourth of the pieces, four head-dimension elements (two for D = 64) per
// lane.
struct JoinParams {
  const int32_t* seq_lens;
  void* out;
  int64_t ot, oh;
  int32_t heads, splits, max_pages, page_shift;
  const float* part_o;
  const float2* part_ml;
};

template <int D, bool F16>
__global__ void __launch_bounds__(128) paged_join_kernel(const JoinParams p) {
  constexpr int kPer = D / 32;
  __shared__ float so[4][D];
  __shared__ float2 sml[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x, b = blockIdx.y;
  griddep_wait();
  griddep_launch();
  bool bad;
  const int len = paged_clamp_len(p.seq_lens[b], p.max_pages, p.page_shift, &bad);
  const int count = split_count((len + kDecTile - 1) / kDecTile, p.splits);
  const int64_t row0 = (static_cast<int64_t>(b) * p.heads + h) * p.splits;
  float m = -INFINITY, l = 0.f, o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int s = warp; s < count; s += 4) {
    const float2 ml = p.part_ml[row0 + s];
    const float* src = p.part_o + (row0 + s) * D + lane * kPer;
    const float mn = fmaxf(m, ml.x);
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float f0 = exp2_approx(m - ms), f1 = exp2_approx(ml.x - ms);
    m = mn;
    l = l * f0 + ml.y * f1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * f0 + src[i] * f1;
  }
  if (lane == 0) sml[warp] = make_float2(m, l);
#pragma unroll
  for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = o[i];
  __syncthreads();
  if (threadIdx.x < D / 2) {
    const int d = threadIdx.x * 2;
    const float top = fmaxf(fmaxf(sml[0].x, sml[1].x), fmaxf(sml[2].x, sml[3].x));
    const float ms = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2_approx(sml[w].x - ms);
      sum += sml[w].y * f;
      x += so[w][d] * f;
      y += so[w][d + 1] * f;
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.ot + h * p.oh + d;
    *reinterpret_cast<uint32_t*>(dst) = pack2<F16>(x * inv, y * inv);
  }
}

}  // namespace abft
