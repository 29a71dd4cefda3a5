// paged_api.cu - the extern "C" entry points of the paged key-value cache:
// argument validation, workspace layout and launches. Declarations are in
// include/abft_b200.h.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>

#include <mutex>

#include "paged_append.cuh"
#include "paged_decode.cuh"
#include "paged_prefill.cuh"

using namespace abft;

namespace {

constexpr int kMaxDevices = 64;
struct DeviceInfo {
  bool init, ok;
  int sms;
  bool smem_set[16];  // decode instances 0-7, prefill instances 8-15
};
DeviceInfo g_paged_dev[kMaxDevices];
std::mutex g_paged_mu;

int paged_device(int* dev_out, int* sms) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return ABFT_ERR_NO_DEVICE;
  }
  std::lock_guard<std::mutex> lk(g_paged_mu);
  DeviceInfo& d = g_paged_dev[dev];
  if (!d.init) {
    int major = 0, minor = 0, n = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cudaGetLastError();
    d.ok = major == 10 && minor == 0;
    d.sms = n;
    d.init = true;
  }
  if (!d.ok) return ABFT_ERR_NO_DEVICE;
  *dev_out = dev;
  *sms = d.sms;
  return ABFT_OK;
}

// Raises a kernel's dynamic shared-memory limit once per device.
template <typename K>
int raise_smem(int dev, int slot, K kernel, int bytes) {
  std::lock_guard<std::mutex> lk(g_paged_mu);
  bool& set = g_paged_dev[dev].smem_set[slot];
  if (set) return ABFT_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return ABFT_ERR_CUDA;
  }
  set = true;
  return ABFT_OK;
}

inline int launch_result() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ABFT_OK : ABFT_ERR_CUDA;
}

inline bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
inline bool off8el(int64_t s) { return (s & 7) != 0; }

// Launch with programmatic serialization: the kernel waits
// (griddepcontrol.wait) before any global access.
template <typename K, typename... P>
int launch_clusters(int cluster, K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t s, const P&... p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p...) != cudaSuccess) {
    cudaGetLastError();
    return ABFT_ERR_CUDA;
  }
  return launch_result();
}

template <typename K, typename... P>
int launch(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t s, const P&... p) {
  return launch_clusters(1, kernel, grid, block, smem, s, p...);
}

int check_kv(const abft_paged_kv& c) {
  if (c.batch < 0 || c.num_pages < 0 || c.max_pages < 0 || c.kv_heads <= 0) return ABFT_ERR_INVALID_ARG;
  if (c.dtype != ABFT_DTYPE_BF16 && c.dtype != ABFT_DTYPE_F16)
    return c.dtype == ABFT_DTYPE_F32 ? ABFT_ERR_UNSUPPORTED : ABFT_ERR_INVALID_ARG;
  if (c.head_dim != 64 && c.head_dim != 128) return ABFT_ERR_UNSUPPORTED;
  if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128) return ABFT_ERR_UNSUPPORTED;
  if (c.batch == 0) return ABFT_OK;
  if (c.k_pages == nullptr || c.v_pages == nullptr || c.page_table == nullptr || c.seq_lens == nullptr ||
      c.max_pages == 0 || c.num_pages == 0)
    return ABFT_ERR_INVALID_ARG;
  if (c.batch > 65535 || c.kv_heads > 4096) return ABFT_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(c.max_pages) * c.page_size >= (int64_t{1} << 30)) return ABFT_ERR_UNSUPPORTED;
  if (c.table_stride < (c.batch > 1 ? c.max_pages : 0)) return ABFT_ERR_INVALID_ARG;
  const int64_t page = static_cast<int64_t>(c.kv_heads) * c.page_size * c.head_dim;
  if (c.num_pages > 1 && (c.k_page_stride < page || c.v_page_stride < page)) return ABFT_ERR_INVALID_ARG;
  if (off16(c.k_pages) || off16(c.v_pages) || off8el(c.k_page_stride) || off8el(c.v_page_stride))
    return ABFT_ERR_ALIGNMENT;
  return ABFT_OK;
}

int check_heads(int heads, int kv_heads) {
  if (heads <= 0 || heads % kv_heads != 0) return ABFT_ERR_INVALID_ARG;
  return heads / kv_heads > 64 ? ABFT_ERR_UNSUPPORTED : ABFT_OK;
}

PagedView view_of(const abft_paged_kv& c) {
  PagedView v;
  v.k_pages = c.k_pages;
  v.v_pages = c.v_pages;
  v.k_page_stride = c.k_page_stride;
  v.v_page_stride = c.v_page_stride;
  v.page_table = c.page_table;
  v.table_stride = c.table_stride;
  v.seq_lens = c.seq_lens;
  v.status = c.status;
  v.num_pages = c.num_pages;
  v.page_shift = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : c.page_size == 64 ? 6 : 7;
  v.kv_heads = c.kv_heads;
  v.batch = c.batch;
  v.max_pages = c.max_pages;
  return v;
}

template <int D, bool F16>
int launch_append(AppendParams p, int sms, cudaStream_t s) {
  // Halve the warps of a token while a full set of the SMs' blocks is left.
  p.warps_shift = 3;
  while (p.warps_shift > 0 && (p.tokens << (p.warps_shift - 1)) >= int64_t{16} * sms) --p.warps_shift;
  const int64_t blocks = ((p.tokens << p.warps_shift) + kAppendWarps - 1) / kAppendWarps + (p.cu != nullptr);
  return launch(kv_append_kernel<D, F16>, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0, s, p);
}

// ---- decode -------------------------------------------------------------------
// Query heads of a group that one CTA takes: one 8-column product, or two
// (16) for larger groups; beyond 16, several CTAs read the same keys.
inline int decode_nt(int group) { return group > 8 ? 2 : 1; }

// Segments (sequence, kv head, chunk of its query heads) and the tiles of one
// in a full cache.
int64_t decode_segments(const abft_paged_attn_args* a) {
  const int group = a->heads / a->kv.kv_heads;
  const int chunks = (group + 8 * decode_nt(group) - 1) / (8 * decode_nt(group));
  return static_cast<int64_t>(a->kv.batch) * a->kv.kv_heads * chunks;
}
int64_t decode_segment_tiles(const abft_paged_attn_args* a) {
  return (static_cast<int64_t>(a->kv.max_pages) * a->kv.page_size + kDecTile - 1) / kDecTile;
}

constexpr int kMostSms = 4096;  // more than any device has: scratch grows with it

int attn_check(const abft_paged_attn_args* a, bool decode) {
  if (a == nullptr) return ABFT_ERR_INVALID_ARG;
  int rc = check_kv(a->kv);
  if (rc != ABFT_OK) return rc;
  if (a->tokens < 0 || a->num_splits < 0 || a->num_sms < 0 || !isfinite(a->scale)) return ABFT_ERR_INVALID_ARG;
  if (a->num_sms > kMostSms) return ABFT_ERR_UNSUPPORTED;
  if ((rc = check_heads(a->heads, a->kv.kv_heads)) != ABFT_OK) return rc;
  if (decode && a->tokens != a->kv.batch) return ABFT_ERR_INVALID_ARG;
  if (a->tokens == 0 || a->kv.batch == 0) return ABFT_OK;
  // The list of tiles is counted in 32 bits.
  if (decode && decode_segments(a) * (decode_segment_tiles(a) + kDecCost) >= (int64_t{1} << 31)) return ABFT_ERR_UNSUPPORTED;
  // Grids (blocks x kv heads, rows x heads for the join) stay below 2^31.
  if (a->tokens >= (int64_t{1} << 30) / a->heads) return ABFT_ERR_UNSUPPORTED;
  if (a->q == nullptr || a->out == nullptr || (!decode && a->cu_seqlens == nullptr)) return ABFT_ERR_INVALID_ARG;
  if (off16(a->q) || off16(a->out) || off8el(a->q_token_stride) || off8el(a->q_head_stride) ||
      off8el(a->o_token_stride) || off8el(a->o_head_stride))
    return ABFT_ERR_ALIGNMENT;
  return ABFT_OK;
}

// CTAs per segment (a cluster of them), or 0: equal shares of the list. When
// the SMs hold all segments and they are short, sharing out costs more (a
// second launch and pieces through memory) than it saves. Measured (equal
// lengths, group 7 of 128; one CTA / a cluster / the list): 4 segments, clusters
// of 8: 190 slots 5.9 / 6.3 / -, 310 slots 7.1 / 6.4 / -, 500 slots - / 6.5 /
// 7.5, 2,000 slots - / 7.8 / 8.0; 32 segments, clusters of 4: 500 slots - / 6.9 /
// 8.3, 1,000 slots - / 8.0 / 9.6; 64 segments, clusters of 2: 370 slots 7.7 / 8.0 /
// -, 500 slots - / 8.2 / 9.7; 128 segments of 512 / 1,280 slots: 9.2 / 17.3 us
// against the list's 11.7 / 21.8. Longer ones are shared out all the same, since
// lengths may differ by more than that. (The lengths are on the device: what is
// known here, and decides, is the width of the table, which is measured where the
// caches fill it. 500 slots in a table of 32,768 go by the list.) Clusters have to fit the device's groups
// of SMs: 15 of 8 and 33 of 4 run at once, a second wave costs 4 us.
int decode_by_segment(const abft_paged_attn_args* a, int sms) {
  const int64_t segments = decode_segments(a), slots = static_cast<int64_t>(a->kv.max_pages) * a->kv.page_size;
  if (segments > sms) return 0;
  if (2 * segments > sms) return slots <= 1280 ? 1 : 0;
  const int c = 8 * segments <= sms * 3 / 4 ? 8 : 4 * segments <= sms * 7 / 8 ? 4 : 2;
  if (slots <= (c == 2 ? 384 : 256)) return 1;
  return slots <= 256 * c ? c : 0;
}

// CTAs of a decode launch: those of the segments' clusters, or one per SM, fewer when the
// cache cannot hold a tile for each of their warps. Of the last fifth of the
// SMs some are left out if the segments then divide evenly among the rest:
// those of equal length do not cross CTAs (256 segments of 8,192 slots: 128
// CTAs 160 us, 148 170; of 2,048: 44 and 48), others lose nothing, since four
// fifths of the SMs already read at full speed (120 CTAs: 168 and 49).
int decode_grid(const abft_paged_attn_args* a, int sms) {
  const int64_t segments = decode_segments(a);
  if (const int c = decode_by_segment(a, sms)) return static_cast<int>(segments) * c;
  const int64_t ctas = (segments * decode_segment_tiles(a) + kDecWarps - 1) / kDecWarps;
  if (ctas <= sms) return static_cast<int>(ctas);
  for (int g = sms; 5 * g >= 4 * sms; --g)
    if (segments % g == 0 || g % segments == 0) return g;
  return sms;
}

// Scratch: two pieces of 8 or 16 heads and one spill record per CTA.
size_t decode_bytes(const abft_paged_attn_args* a, int sms) {
  if (decode_by_segment(a, sms)) return 0;
  const int grid = decode_grid(a, sms);
  const size_t rows = static_cast<size_t>(grid) * 2 * 8 * decode_nt(a->heads / a->kv.kv_heads);
  return rows * (a->kv.head_dim * sizeof(float) + sizeof(float2)) + grid * sizeof(int4);
}

template <int D, int NT, bool F16>
int launch_decode(int dev, int slot, const DecodeParams& p, int grid, cudaStream_t s) {
  using Cfg = DecodeCfg<D, NT>;
  int rc = raise_smem(dev, slot, paged_decode_kernel<D, NT, F16>, Cfg::kSmemBytes);
  if (rc != ABFT_OK) return rc;
  rc = launch_clusters(p.by_segment, paged_decode_kernel<D, NT, F16>, dim3(grid), dim3(Cfg::kThreads), Cfg::kSmemBytes, s, p);
  if (rc != ABFT_OK || p.by_segment) return rc;
  JoinParams j;
  j.out = p.out;
  j.ot = p.ot;
  j.oh = p.oh;
  j.group = p.group;
  j.head_chunks = p.head_chunks;
  j.part_o = p.part_o;
  j.part_ml = p.part_ml;
  j.spill = p.spill;
  const int heads = p.group < Cfg::kHeads ? p.group : Cfg::kHeads;
  return launch(paged_join_kernel<D, NT, F16>, dim3(grid, heads), dim3(32 * kJoinWarps), 0, s, j);
}

// ---- prefill ------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn tile_encoder() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
    else
      cudaGetLastError();
  });
  return fn;
}

// Map of a page pool: [page][group of 8 slots of a head][64-column block][slot
// of the group][64 columns]; a box is one page's slots of one head, whole rows,
// 128-byte swizzled.
int page_map(CUtensorMap* m, const abft_paged_kv& c, const void* pages, int64_t stride) {
  EncodeTiledFn enc = tile_encoder();
  if (enc == nullptr) return ABFT_ERR_DRIVER;
  const int64_t dense = static_cast<int64_t>(c.kv_heads) * c.page_size * c.head_dim;
  if (c.num_pages <= 1) stride = dense;
  const cuuint64_t row = static_cast<cuuint64_t>(c.head_dim) * 2;
  cuuint64_t dims[5] = {64, 8, static_cast<cuuint64_t>(c.head_dim / 64),
                        static_cast<cuuint64_t>(c.kv_heads) * c.page_size / 8, static_cast<cuuint64_t>(c.num_pages)};
  cuuint64_t strides[4] = {row, 128, 8 * row, static_cast<cuuint64_t>(stride) * 2};
  cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(c.head_dim / 64), static_cast<cuuint32_t>(c.page_size / 8), 1};
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType type =
      c.dtype == ABFT_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = enc(m, type, 5, const_cast<void*>(pages), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ABFT_OK : ABFT_ERR_ALIGNMENT;
}

// How a prefill call is cut: items of one or two tiles of query rows and one
// kv head, their keys in pieces of `piece` steps.
struct PrefillPlan {
  int tile_tokens, block_tokens, splits, piece;
  bool choose;    // the kernel chooses the piece, for `splits` pieces at most
  int64_t items;  // blocks of the grid
};

PrefillPlan prefill_plan(const abft_paged_attn_args* a, int sms) {
  PrefillPlan r;
  r.tile_tokens = kPreRows / (a->heads / a->kv.kv_heads);
  // Two tiles an item keep the tensor core at work on one while the other's
  // rows are exponentiated; a call that has an SM for each tile takes one.
  r.block_tokens = 2 * r.tile_tokens;
  const auto blocks = [&](int per) { return (a->tokens / per + a->kv.batch) * a->kv.kv_heads; };
  if (blocks(r.tile_tokens) <= sms) r.block_tokens = r.tile_tokens;
  const int64_t base = blocks(r.block_tokens);
  const int64_t steps = (static_cast<int64_t>(a->kv.max_pages) * a->kv.page_size + kPreKeys - 1) / kPreKeys;
  // Without a number of pieces given, the kernel chooses their length for the
  // sequences it finds (scan_work); here their number is bounded: room for each
  // SM to have one, for several sequences, whose lengths may differ, four. One
  // where the blocks alone fill the SMs. (One sequence, 64 tokens on 16,384
  // slots: 1 piece 159 us, 8 pieces 34, 16 40; 512 tokens on 8,192, 116 items: 1
  // piece 81, 2 pieces 96, for the sums that go through memory. Nine sequences of
  // 5 tokens, 36 items, on up to 7,777 slots: 4 pieces 29, 8 21, 16 18; on 7,777
  // each: 4 pieces 36, 8 37, 16 46. Chosen in the kernel: 36, 79, 19, 38; in tables
  // of 32,768 slots 64 tokens on 4,000 22 us, 46 in pieces of the table's width.)
  int64_t n = a->num_splits;
  if (n == 0) {
    int64_t least = (a->tokens + r.block_tokens - 1) / r.block_tokens;
    if (least < a->kv.batch) least = a->kv.batch;
    n = sms / (least * a->kv.kv_heads);
    if (a->kv.batch > 1) n *= 4;
    if (n > (steps + kPreLeast - 1) / kPreLeast) n = (steps + kPreLeast - 1) / kPreLeast;
  }
  if (n > steps) n = steps;
  if (n < 1) n = 1;
  r.choose = a->num_splits == 0 && n > 1;
  r.piece = static_cast<int>((steps + n - 1) / n);
  r.splits = static_cast<int>((steps + r.piece - 1) / r.piece);
  r.items = r.choose ? (base > sms ? base : sms) : base * r.splits;
  return r;
}

size_t prefill_bytes(const abft_paged_attn_args* a, const PrefillPlan& plan) {
  if (plan.splits <= 1) return 0;
  const size_t rows = static_cast<size_t>(a->tokens) * a->heads * plan.splits;
  return rows * (a->kv.head_dim * sizeof(float) + sizeof(float2)) + (plan.choose ? 16 : 0);
}

template <int D, bool F16, bool kShared>
int launch_prefill(int dev, int slot, const abft_paged_attn_args* a, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                   const PrefillParams& p, int64_t items, cudaStream_t s) {
  using Cfg = PrefillCfg<D>;
  int rc = raise_smem(dev, slot, paged_prefill_kernel<D, F16, kShared>, Cfg::kSmemBytes);
  if (rc != ABFT_OK) return rc;
  rc = launch(paged_prefill_kernel<D, F16, kShared>, dim3(static_cast<unsigned>(items)), dim3(kPreThreads), Cfg::kSmemBytes, s,
              tm_k, tm_v, p);
  if (rc != ABFT_OK || p.splits == 1) return rc;
  PrefillJoinParams j;
  j.kv = p.kv;
  j.cu = p.cu;
  j.out = p.out;
  j.ot = p.ot;
  j.oh = p.oh;
  j.tokens = p.tokens;
  j.heads = a->heads;
  j.splits = p.splits;
  j.piece = p.piece;
  j.chosen = p.chosen;
  j.block_tokens = p.block_tokens;
  j.part_o = p.part_o;
  j.part_ml = p.part_ml;
  const unsigned rows = static_cast<unsigned>(p.tokens) * a->heads;
  return launch(paged_prefill_join_kernel<D, F16>, dim3((rows + kPreJoinWarps - 1) / kPreJoinWarps),
                dim3(32 * kPreJoinWarps), 0, s, j);
}

}  // namespace

extern "C" {

int abft_kv_append(const abft_kv_append_args* a, void* stream) {
  if (a == nullptr) return ABFT_ERR_INVALID_ARG;
  int rc = check_kv(a->kv);
  if (rc != ABFT_OK) return rc;
  if (a->tokens < 0 || a->heads < 0 || a->max_positions < 0) return ABFT_ERR_INVALID_ARG;
  if (a->heads > 0 && (rc = check_heads(a->heads, a->kv.kv_heads)) != ABFT_OK) return rc;
  if (a->cu_seqlens == nullptr && a->tokens != a->kv.batch) return ABFT_ERR_INVALID_ARG;
  if (a->tokens == 0 || a->kv.batch == 0) return ABFT_OK;
  if (a->tokens >= (int64_t{1} << 31)) return ABFT_ERR_UNSUPPORTED;
  if (a->k == nullptr || a->v == nullptr || (a->heads > 0 && (a->q == nullptr || a->q_out == nullptr)))
    return ABFT_ERR_INVALID_ARG;
  if (off16(a->k) || off16(a->v) || off16(a->rope) || off8el(a->k_token_stride) || off8el(a->k_head_stride) ||
      off8el(a->v_token_stride) || off8el(a->v_head_stride))
    return ABFT_ERR_ALIGNMENT;
  if (a->heads > 0 && (off16(a->q) || off16(a->q_out) || off8el(a->q_token_stride) || off8el(a->q_head_stride) ||
                       off8el(a->o_token_stride) || off8el(a->o_head_stride)))
    return ABFT_ERR_ALIGNMENT;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  AppendParams p;
  p.kv = view_of(a->kv);
  p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out;
  p.qt = a->q_token_stride, p.qh = a->q_head_stride;
  p.kt = a->k_token_stride, p.kh = a->k_head_stride;
  p.vt = a->v_token_stride, p.vh = a->v_head_stride;
  p.ot = a->o_token_stride, p.oh = a->o_head_stride;
  p.cu = a->cu_seqlens;
  p.rope = a->rope;
  p.max_positions = a->max_positions;
  p.tokens = a->tokens;
  p.heads = a->heads;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = a->kv.dtype == ABFT_DTYPE_F16;
  if (a->kv.head_dim == 128) return f16 ? launch_append<128, true>(p, sms, s) : launch_append<128, false>(p, sms, s);
  return f16 ? launch_append<64, true>(p, sms, s) : launch_append<64, false>(p, sms, s);
}

size_t abft_paged_decode_workspace_bytes(const abft_paged_attn_args* a) {
  if (attn_check(a, true) != ABFT_OK || a->kv.batch == 0) return 0;
  int dev = 0, sms = a->num_sms;
  if (sms == 0 && paged_device(&dev, &sms) != ABFT_OK) sms = 148;
  return decode_bytes(a, sms);
}

int abft_paged_decode(const abft_paged_attn_args* a, void* stream) {
  int rc = attn_check(a, true);
  if (rc != ABFT_OK || a->kv.batch == 0) return rc;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  if (a->num_sms > 0) sms = a->num_sms;
  DecodeParams p;
  p.kv = view_of(a->kv);
  p.q = a->q, p.out = a->out;
  p.qt = a->q_token_stride, p.qh = a->q_head_stride;
  p.ot = a->o_token_stride, p.oh = a->o_head_stride;
  p.group = a->heads / a->kv.kv_heads;
  const int nt = decode_nt(p.group);
  p.head_chunks = (p.group + 8 * nt - 1) / (8 * nt);
  p.scale_log2 = a->scale * 1.44269504088896340736f;
  const int grid = decode_grid(a, sms);
  p.by_segment = decode_by_segment(a, sms);
  for (p.cluster_shift = 0; 1 << (p.cluster_shift + 1) <= p.by_segment;) ++p.cluster_shift;
  const size_t need = decode_bytes(a, sms);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return ABFT_ERR_WORKSPACE;
  if (need > 0 && off16(a->workspace)) return ABFT_ERR_ALIGNMENT;
  const size_t rows = static_cast<size_t>(grid) * 2 * 8 * nt;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + rows * a->kv.head_dim);
  p.spill = reinterpret_cast<int4*>(p.part_ml + rows);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = a->kv.dtype == ABFT_DTYPE_F16;
  const int slot = (a->kv.head_dim == 128 ? 4 : 0) + (nt == 2 ? 2 : 0) + (f16 ? 1 : 0);
  switch (slot) {
    case 0: return launch_decode<64, 1, false>(dev, slot, p, grid, s);
    case 1: return launch_decode<64, 1, true>(dev, slot, p, grid, s);
    case 2: return launch_decode<64, 2, false>(dev, slot, p, grid, s);
    case 3: return launch_decode<64, 2, true>(dev, slot, p, grid, s);
    case 4: return launch_decode<128, 1, false>(dev, slot, p, grid, s);
    case 5: return launch_decode<128, 1, true>(dev, slot, p, grid, s);
    case 6: return launch_decode<128, 2, false>(dev, slot, p, grid, s);
    default: return launch_decode<128, 2, true>(dev, slot, p, grid, s);
  }
}

size_t abft_paged_prefill_workspace_bytes(const abft_paged_attn_args* a) {
  if (attn_check(a, false) != ABFT_OK || a->kv.batch == 0 || a->tokens == 0) return 0;
  int dev = 0, sms = a->num_sms;
  if (sms == 0 && paged_device(&dev, &sms) != ABFT_OK) sms = 148;
  return prefill_bytes(a, prefill_plan(a, sms));
}

int abft_paged_prefill(const abft_paged_attn_args* a, void* stream) {
  int rc = attn_check(a, false);
  if (rc != ABFT_OK || a->kv.batch == 0 || a->tokens == 0) return rc;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  if (a->num_sms > 0) sms = a->num_sms;
  PrefillParams p;
  p.kv = view_of(a->kv);
  p.q = a->q, p.out = a->out;
  p.qt = a->q_token_stride, p.qh = a->q_head_stride;
  p.ot = a->o_token_stride, p.oh = a->o_head_stride;
  p.cu = a->cu_seqlens;
  p.tokens = static_cast<int32_t>(a->tokens);
  p.group = a->heads / a->kv.kv_heads;
  const PrefillPlan plan = prefill_plan(a, sms);
  if (plan.items >= (int64_t{1} << 31)) return ABFT_ERR_UNSUPPORTED;
  p.tile_tokens = plan.tile_tokens;
  p.block_tokens = plan.block_tokens;
  p.splits = plan.splits;
  p.piece = plan.choose ? 0 : plan.piece;
  p.sms = sms;
  const float s2 = fabsf(a->scale) * 1.44269504088896340736f;
  p.scale_log2 = s2 > 1e-30f ? s2 : 1e-30f;  // scale 0: every visible weight 2^0, masked scores still -inf
  p.negate = a->scale < 0.f;
  p.group_inv = (65536u + p.group - 1) / p.group;
  const size_t need = prefill_bytes(a, plan);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return ABFT_ERR_WORKSPACE;
  if (need > 0 && off16(a->workspace)) return ABFT_ERR_ALIGNMENT;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float2*>(
      p.part_o + static_cast<size_t>(a->tokens) * a->heads * p.splits * a->kv.head_dim);
  p.chosen = plan.choose ? reinterpret_cast<int32_t*>(p.part_ml + static_cast<size_t>(a->tokens) * a->heads * p.splits)
                         : nullptr;
  CUtensorMap tm_k, tm_v;
  if ((rc = page_map(&tm_k, a->kv, a->kv.k_pages, a->kv.k_page_stride)) != ABFT_OK) return rc;
  if ((rc = page_map(&tm_v, a->kv, a->kv.v_pages, a->kv.v_page_stride)) != ABFT_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = a->kv.dtype == ABFT_DTYPE_F16;
  const bool shared = plan.block_tokens == plan.tile_tokens;
  const int slot = 8 + (a->kv.head_dim == 128 ? 4 : 0) + (f16 ? 2 : 0) + (shared ? 1 : 0);
  const int64_t items = plan.items;
  switch (slot - 8) {
    case 0: return launch_prefill<64, false, false>(dev, slot, a, tm_k, tm_v, p, items, s);
    case 1: return launch_prefill<64, false, true>(dev, slot, a, tm_k, tm_v, p, items, s);
    case 2: return launch_prefill<64, true, false>(dev, slot, a, tm_k, tm_v, p, items, s);
    case 3: return launch_prefill<64, true, true>(dev, slot, a, tm_k, tm_v, p, items, s);
    case 4: return launch_prefill<128, false, false>(dev, slot, a, tm_k, tm_v, p, items, s);
    case 5: return launch_prefill<128, false, true>(dev, slot, a, tm_k, tm_v, p, items, s);
    case 6: return launch_prefill<128, true, false>(dev, slot, a, tm_k, tm_v, p, items, s);
    default: return launch_prefill<128, true, true>(dev, slot, a, tm_k, tm_v, p, items, s);
  }
}

}  // extern "C"
