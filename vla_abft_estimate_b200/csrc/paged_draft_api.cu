// paged_draft_api.cu - the extern "C" entry points for drafted trees and forks
// over the paged cache: append by given positions, tree attention, accept, keep
// and fork. Declarations are in include/abft_b200.h.
#include "paged_draft.cuh"
#include "paged_launch.cuh"
#include "paged_tree.cuh"

using namespace abft;

namespace {

int check_layers(const abft_paged_kv& kv, void* const* pools, int32_t layers) {
  if (layers < 1 || (pools == nullptr && layers != 1)) return ABFT_ERR_INVALID_ARG;
  if (layers > kMostLayers) return ABFT_ERR_UNSUPPORTED;
  const int rc = check_kv(kv);
  if (rc != ABFT_OK || pools == nullptr || kv.batch == 0) return rc;
  for (int i = 0; i < 2 * layers; ++i) {
    if (pools[i] == nullptr) return ABFT_ERR_INVALID_ARG;
    if (off16(pools[i])) return ABFT_ERR_ALIGNMENT;
  }
  return ABFT_OK;
}

template <int kLayers>
LayerPools<kLayers> layer_pools(const abft_paged_kv& kv, void* const* pools, int32_t layers) {
  LayerPools<kLayers> r;
  r.layers = layers;
  for (int i = 0; i < 2 * layers; ++i)
    r.pools[i] = static_cast<uint16_t*>(pools != nullptr ? pools[i] : i == 0 ? kv.k_pages : kv.v_pages);
  return r;
}

// How a tree call is cut: segments of a tile of query rows and one kv head, dealt by
// the list or to clusters.
struct TreePlan {
  int tile_tokens;
  int cluster;  // CTAs of a segment, or 0: the list
  int grid;
};

// The list, or a CTA per segment, or a cluster of up to 8 as long as all clusters run
// at once (two CTAs an SM; 8 x 30 and 4 x 65 fit the device's groups of SMs): whichever
// takes least, counted in steps (0.85 us). The list evens out what sequences of unlike
// length take, but its second launch and the pieces' way through memory cost 13; a
// cluster's pieces go through the SMs' network, which is slow (25 GB/s an SM): 1 step
// while 64 CTAs use it at once (one cluster of 8 in each group of SMs), above that 6, or
// 3 with heads of 64. No more than 12 steps for a CTA: the lengths are on the device, what
// is known here is the width of the table, and it is the longest sequence that the
// others then wait for (16 steps: 32 trees of 8 on 2,000 slots each 30 us, by the list 37,
// but on up to 2,000, most far below, 21 and 14). Measured (us; 1, 2, 4, 8 CTAs / list; 28/4 heads of 128):
//   1 tree of 16 tokens on 1,000 slots  18.3 13.9 10.6 9.2 / 10.7, 8,000  104 57 31.9 19.8 / 16.0
//   4 of 16 on 1,000  18.4 14.2 11.1 13.1 / 14.0, 2,000  31.0 20.6 14.1 14.7 / 16.3, 4,000  57 33.7 20.9 18.4 / 21.2
//   16 of 16 on 500  14.0 15.8 15.8 - / 16.9, 2,000  34.1 27.4 22.4 - / 25.3
//   32 of 8 on 300  10.9 11.6 - - / 16.3, 1,250  26.1 21.8 - - / 28.4, on up to 1,200  20.8 16.0 - - / 14.0
//   8 of 16, heads of 64, on 500  11.7 10.1 10.8 12.7 / 13.8, 2,000  29.0 18.4 15.2 15.3 / 15.2
constexpr int kTreeListSteps = 13, kTreeQuiet = 64, kTreeMostSteps = 12;

int tree_plan(const abft_paged_attn_args* a, int sms, TreePlan* r) {
  r->tile_tokens = kTreeRows / (a->heads / a->kv.kv_heads);
  // Segments at most (the boundaries are on the device), and as many as they are when
  // all sequences have equally many rows.
  const int64_t mean = a->kv.batch > 0 ? (a->tokens + a->kv.batch - 1) / a->kv.batch : 0;
  auto most = [&](int tile) { return a->kv.kv_heads * (a->kv.batch == 1 ? (a->tokens + tile - 1) / tile : a->tokens / tile + a->kv.batch); };
  auto likely = [&](int tile) { return a->kv.kv_heads * a->kv.batch * ((mean + tile - 1) / tile); };
  const int64_t segments = likely(r->tile_tokens);
  const int64_t slots = static_cast<int64_t>(a->kv.max_pages) * a->kv.page_size;
  const int64_t steps = slots > kTreeKeys ? (slots + kTreeKeys - 1) / kTreeKeys : 1;
  if (most(r->tile_tokens) * (steps + kTreeCost) >= (int64_t{1} << 31)) return ABFT_ERR_UNSUPPORTED;  // the list is counted in 32 bits
  const int ctas = 2 * sms;
  r->cluster = 0;
  int64_t least = kTreeListSteps + segments * steps / ctas;
  for (int c = 1; c <= 8 && c * segments <= ctas * (c == 8 ? 13 : c == 4 ? 14 : 16) / 16 && (c == 1 || c / 2 < steps); c *= 2) {
    const int64_t per = (steps + c - 1) / c;
    const int64_t time = per + (c == 1 ? 0 : c * segments <= kTreeQuiet ? 1 : a->kv.head_dim == 128 ? 6 : 3);
    if (per <= kTreeMostSteps && time < least) {
      least = time;
      r->cluster = c;
    }
  }
  if (r->cluster == 0) {
    const int64_t places = most(r->tile_tokens) * steps;
    r->grid = static_cast<int>(places < ctas ? places : ctas);
    return ABFT_OK;
  }
  // Clusters of 8 with CTAs to spare take smaller tiles, of which less goes to and fro
  // (1 tree of 16 tokens on 1,000 slots: 9.2 -> 8.3 us).
  for (int half; r->cluster == 8 && r->tile_tokens > 1; r->tile_tokens = half) {
    half = (r->tile_tokens + 1) / 2;
    if (8 * likely(half) > kTreeQuiet) break;
  }
  r->grid = static_cast<int>(most(r->tile_tokens)) * r->cluster;  // those without a segment end at once
  return ABFT_OK;
}

size_t tree_bytes(const abft_paged_attn_args* a, const TreePlan& plan) {
  if (plan.cluster > 0) return 0;
  const size_t rows = static_cast<size_t>(plan.grid) * 2 * kTreeRows;
  return rows * (a->kv.head_dim * sizeof(float) + sizeof(float2)) + plan.grid * (sizeof(int2) + sizeof(int32_t));
}

// Map of the query rows: [token][head][head_dim]; a box is the (token, head) rows of a
// tile and 64 columns, 128-byte swizzled.
int query_map(CUtensorMap* m, const abft_paged_attn_args* a, int tile_tokens) {
  EncodeTiledFn enc = tile_encoder();
  if (enc == nullptr) return ABFT_ERR_DRIVER;
  const cuuint64_t row = static_cast<cuuint64_t>(a->kv.head_dim) * 2;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(a->kv.head_dim), static_cast<cuuint64_t>(a->heads),
                        static_cast<cuuint64_t>(a->tokens)};
  // (The stride of a dimension of one is not used, but has to be a valid one.)
  cuuint64_t strides[2] = {a->heads > 1 ? static_cast<cuuint64_t>(a->q_head_stride) * 2 : row,
                           a->tokens > 1 ? static_cast<cuuint64_t>(a->q_token_stride) * 2 : row};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a->heads / a->kv.kv_heads), static_cast<cuuint32_t>(tile_tokens)};
  cuuint32_t es[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      a->kv.dtype == ABFT_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = enc(m, type, 3, const_cast<void*>(a->q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ABFT_OK : ABFT_ERR_ALIGNMENT;
}

template <int D, bool F16>
int launch_tree(int dev, int slot, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const CUtensorMap& tm_q,
                const TreeParams& p, const TreePlan& plan, int sms, cudaStream_t s) {
  using Cfg = TreeCfg<D>;
  int rc = raise_smem(dev, slot, paged_tree_kernel<D, F16>, Cfg::kSmemBytes);
  if (rc != ABFT_OK) return rc;
  rc = launch_clusters(p.work.cluster, paged_tree_kernel<D, F16>, dim3(plan.grid), dim3(kTreeThreads), Cfg::kSmemBytes, s, tm_k,
                       tm_v, tm_q, p);
  if (rc != ABFT_OK || p.work.cluster > 0) return rc;
  return launch(paged_tree_join_kernel<D, F16>, dim3(4 * sms), dim3(kTreeJoinThreads), 0, s, p, plan.grid);
}

int tree_call(const abft_paged_tree_args* t, void* stream) {
  const abft_paged_attn_args* a = &t->attn;
  int rc = attn_check(a, false);
  if (rc != ABFT_OK || a->kv.batch == 0 || a->tokens == 0) return rc;
  if (t->parents == nullptr) return ABFT_ERR_INVALID_ARG;
  // Query rows come as boxes of a tensor, whose strides are above 0.
  if ((a->heads > 1 && a->q_head_stride <= 0) || (a->tokens > 1 && a->q_token_stride <= 0)) return ABFT_ERR_INVALID_ARG;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  if (a->num_sms > 0) sms = a->num_sms;
  TreePlan plan;
  if ((rc = tree_plan(a, sms, &plan)) != ABFT_OK) return rc;
  const size_t need = tree_bytes(a, plan);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return ABFT_ERR_WORKSPACE;
  if (need > 0 && off16(a->workspace)) return ABFT_ERR_ALIGNMENT;
  TreeParams p = {};
  p.kv = view_of(a->kv);
  p.q = a->q, p.out = a->out;
  p.qt = a->q_token_stride, p.qh = a->q_head_stride;
  p.ot = a->o_token_stride, p.oh = a->o_head_stride;
  p.cu = a->cu_seqlens;
  p.tokens = static_cast<int32_t>(a->tokens);
  p.group = a->heads / a->kv.kv_heads;
  p.tile_tokens = plan.tile_tokens;
  const float s2 = fabsf(a->scale) * 1.44269504088896340736f;
  p.scale_log2 = s2 > 1e-30f ? s2 : 1e-30f;  // scale 0: every visible weight 2^0, masked scores still -inf
  p.negate = a->scale < 0.f;
  p.group_inv = (65536u + p.group - 1) / p.group;
  p.work.parents = t->parents;
  p.work.cluster = plan.cluster;
  while (1 << (p.work.cluster_shift + 1) <= plan.cluster) ++p.work.cluster_shift;
  const size_t rows = static_cast<size_t>(plan.grid) * 2 * kTreeRows;
  p.work.part = static_cast<float4*>(a->workspace);
  p.work.part_ml = reinterpret_cast<float2*>(p.work.part + rows * (a->kv.head_dim / 4));
  p.work.spill = reinterpret_cast<int2*>(p.work.part_ml + rows);
  p.work.pieces = reinterpret_cast<int32_t*>(p.work.spill + plan.grid);
  CUtensorMap tm_k, tm_v, tm_q;
  if ((rc = query_map(&tm_q, a, plan.tile_tokens)) != ABFT_OK) return rc;
  if ((rc = page_map(&tm_k, a->kv, a->kv.k_pages, a->kv.k_page_stride, kTreeKeys)) != ABFT_OK) return rc;
  if ((rc = page_map(&tm_v, a->kv, a->kv.v_pages, a->kv.v_page_stride, kTreeKeys)) != ABFT_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = a->kv.dtype == ABFT_DTYPE_F16;
  if (a->kv.head_dim == 128)
    return f16 ? launch_tree<128, true>(dev, 19, tm_k, tm_v, tm_q, p, plan, sms, s)
               : launch_tree<128, false>(dev, 18, tm_k, tm_v, tm_q, p, plan, sms, s);
  return f16 ? launch_tree<64, true>(dev, 17, tm_k, tm_v, tm_q, p, plan, sms, s)
             : launch_tree<64, false>(dev, 16, tm_k, tm_v, tm_q, p, plan, sms, s);
}

// An array of a call, as memory: what one sequence's or pair's CTAs write must not be
// what another's read.
struct Span {
  uintptr_t at;
  size_t bytes;
  Span(const void* p, int64_t items, size_t size = sizeof(int32_t))
      : at(reinterpret_cast<uintptr_t>(p)), bytes(static_cast<size_t>(items) * size) {}
  bool meets(const Span& o) const { return bytes > 0 && o.bytes > 0 && at < o.at + o.bytes && o.at < at + bytes; }
};

// Some row of the table (what lies between its rows is not its own).
bool meets_table(const Span& x, const abft_paged_kv& kv) {
  const Span whole(kv.page_table, (kv.batch - 1) * kv.table_stride + kv.max_pages);
  if (!x.meets(whole)) return false;
  if (kv.batch == 1 || x.at <= whole.at) return true;
  // The first row that ends behind x's start.
  const int64_t pitch = kv.table_stride * 4, row = kv.max_pages * int64_t{4}, from = static_cast<int64_t>(x.at - whole.at);
  const int64_t first = from < row ? 0 : (from - row) / pitch + 1;
  return first * pitch < from + static_cast<int64_t>(x.bytes);
}

template <int kLayers>
int keep_call(const abft_kv_keep_args* a, int sms, cudaStream_t s) {
  KeepParams<kLayers> p;
  p.kv = view_of(a->kv);
  p.layers = layer_pools<kLayers>(a->kv, a->pools, a->layers);
  p.cu = a->cu_seqlens, p.kept = a->kept, p.counts = a->counts;
  p.lens_out = a->lens_out;
  p.tokens = static_cast<int32_t>(a->tokens);
  // A thread for each 16 bytes of a slot in all layers, as far as a cluster has them;
  // half as many where that makes more CTAs than run at once (28 layers, CTAs of 512 /
  // 256 threads: 1 sequence 3.4 / 3.9 us, 64 sequences 7.4 / 5.6).
  const int64_t columns = int64_t{2} * a->layers * a->kv.kv_heads * a->kv.head_dim / 8;
  for (p.cluster = 1; p.cluster < kKeepCluster && int64_t{p.cluster} * kKeepThreads < columns;) p.cluster *= 2;
  const dim3 grid(a->kv.batch * p.cluster), block(int64_t{a->kv.batch} * p.cluster > 3 * sms ? kKeepThreads / 2 : kKeepThreads);
  return a->kv.head_dim == 128 ? launch_clusters(p.cluster, kv_keep_kernel<128, kLayers>, grid, block, 0, s, p)
                               : launch_clusters(p.cluster, kv_keep_kernel<64, kLayers>, grid, block, 0, s, p);
}

template <int kLayers>
int fork_call(const abft_kv_fork_args* a, cudaStream_t s) {
  ForkParams<kLayers> p;
  p.kv = view_of(a->kv);
  p.layers = layer_pools<kLayers>(a->kv, a->pools, a->layers);
  p.src = a->src, p.dst = a->dst, p.pages = a->pages;
  p.pairs = a->pairs;
  const int64_t items = int64_t{2} * a->layers * a->kv.kv_heads;
  // 1, 2 or 4 warps to a head, so that each has work when the page is full (32 forks,
  // pages of 128: 35.4 us with 1, 32.2 with 2, 30.5 with 4, 33.3 with 8).
  p.shift = a->kv.page_size == 16 ? 0 : a->kv.page_size == 32 ? 1 : 2;
  p.per_pair = static_cast<int32_t>(((items << p.shift) + kForkWarps - 1) / kForkWarps);
  const int64_t blocks = int64_t{p.per_pair} * a->pairs;
  if (blocks >= (int64_t{1} << 31)) return ABFT_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks)), block(32 * kForkWarps);
  return a->kv.head_dim == 128 ? launch(kv_fork_kernel<128, kLayers>, grid, block, 0, s, p)
                               : launch(kv_fork_kernel<64, kLayers>, grid, block, 0, s, p);
}

}  // namespace

extern "C" {

int abft_kv_append_at(const abft_kv_append_at_args* a, void* stream) {
  if (a == nullptr) return ABFT_ERR_INVALID_ARG;
  int rc = append_check(&a->append);
  if (rc != ABFT_OK) return rc;
  if (a->axes < 1 || a->axes > kMostAxes) return a->axes < 1 ? ABFT_ERR_INVALID_ARG : ABFT_ERR_UNSUPPORTED;
  int64_t pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->sections[i] < 0) return ABFT_ERR_INVALID_ARG;
    pairs += a->sections[i];
  }
  if (pairs * 2 != a->append.kv.head_dim) return ABFT_ERR_INVALID_ARG;
  if (a->append.tokens == 0 || a->append.kv.batch == 0) return ABFT_OK;
  if (a->append.rope == nullptr || a->positions == nullptr || a->append.max_positions == 0 || a->position_stride < 0)
    return ABFT_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(a->positions) & 3u) != 0) return ABFT_ERR_ALIGNMENT;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  AppendAtParams p;
  append_params(&a->append, &p);
  p.positions = a->positions;
  p.position_stride = a->position_stride;
  p.axes = a->axes;
  for (int i = 0, end = 0; i < kMostAxes; ++i) {
    if (i < a->axes) end += a->sections[i];
    p.axis_end[i] = end;
  }
  return append_call(p, a->append.kv, sms, stream);
}

size_t abft_paged_tree_workspace_bytes(const abft_paged_tree_args* t) {
  if (t == nullptr) return 0;
  const abft_paged_attn_args* a = &t->attn;
  if (attn_check(a, false) != ABFT_OK || a->kv.batch == 0 || a->tokens == 0) return 0;
  int dev = 0, sms = a->num_sms;
  if (sms == 0 && paged_device(&dev, &sms) != ABFT_OK) sms = 148;
  TreePlan plan;
  return tree_plan(a, sms, &plan) == ABFT_OK ? tree_bytes(a, plan) : 0;
}

int abft_paged_tree(const abft_paged_tree_args* t, void* stream) {
  return t == nullptr ? ABFT_ERR_INVALID_ARG : tree_call(t, stream);
}

int abft_draft_accept(const abft_draft_accept_args* a, void* stream) {
  if (a == nullptr || a->batch < 0 || a->tokens < 0) return ABFT_ERR_INVALID_ARG;
  if (a->id_bytes != 4 && a->id_bytes != 8) return ABFT_ERR_INVALID_ARG;
  if (a->batch > 65535 || a->tokens >= (int64_t{1} << 30)) return ABFT_ERR_UNSUPPORTED;
  if (a->batch == 0 && a->tokens == 0) return ABFT_OK;
  if (a->batch > 0 && (a->cu_seqlens == nullptr || a->counts == nullptr || a->next == nullptr)) return ABFT_ERR_INVALID_ARG;
  if (a->tokens > 0 && (a->parents == nullptr || a->ids == nullptr || a->answers == nullptr || a->kept == nullptr))
    return ABFT_ERR_INVALID_ARG;
  const uintptr_t ids = reinterpret_cast<uintptr_t>(a->ids) | reinterpret_cast<uintptr_t>(a->answers) |
                        reinterpret_cast<uintptr_t>(a->next);
  if ((ids & static_cast<uintptr_t>(a->id_bytes - 1)) != 0) return ABFT_ERR_ALIGNMENT;
  // What is read is read by any thread at any time.
  const Span kept(a->kept, a->tokens), counts(a->counts, a->batch), next(a->next, a->batch, a->id_bytes);
  const Span read[] = {Span(a->cu_seqlens, int64_t{a->batch} + 1), Span(a->parents, a->tokens), Span(a->ids, a->tokens, a->id_bytes),
                       Span(a->answers, a->tokens, a->id_bytes)};
  for (const Span& x : read)
    if (kept.meets(x) || counts.meets(x) || next.meets(x)) return ABFT_ERR_INVALID_ARG;
  if (kept.meets(counts) || kept.meets(next) || counts.meets(next)) return ABFT_ERR_INVALID_ARG;
  int dev = 0, sms = 0;
  const int rc = paged_device(&dev, &sms);
  if (rc != ABFT_OK) return rc;
  AcceptParams p;
  p.cu = a->cu_seqlens;
  p.parents = a->parents;
  p.ids = a->ids, p.answers = a->answers;
  p.kept = a->kept;
  p.counts = a->counts;
  p.next = a->next;
  p.status = a->status;
  p.tokens = static_cast<int32_t>(a->tokens);
  p.batch = a->batch;
  const dim3 grid(a->batch + 1), block(kAcceptThreads);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->id_bytes == 8 ? launch(draft_accept_kernel<int64_t>, grid, block, 0, s, p)
                          : launch(draft_accept_kernel<int32_t>, grid, block, 0, s, p);
}

int abft_kv_keep(const abft_kv_keep_args* a, void* stream) {
  if (a == nullptr) return ABFT_ERR_INVALID_ARG;
  int rc = check_layers(a->kv, a->pools, a->layers);
  if (rc != ABFT_OK) return rc;
  if (a->tokens < 0) return ABFT_ERR_INVALID_ARG;
  if (a->tokens >= (int64_t{1} << 30)) return ABFT_ERR_UNSUPPORTED;
  if (a->kv.batch == 0) return ABFT_OK;
  if (a->cu_seqlens == nullptr || a->counts == nullptr || a->lens_out == nullptr || (a->tokens > 0 && a->kept == nullptr))
    return ABFT_ERR_INVALID_ARG;
  // The lengths themselves, or an array of its own: not a part of them, nor of what other
  // sequences still read. (A sequence's count is read before its length is written.)
  const Span out(a->lens_out, a->kv.batch), lens(a->kv.seq_lens, a->kv.batch), counts(a->counts, a->kv.batch);
  if ((out.at != lens.at && out.meets(lens)) || (out.at != counts.at && out.meets(counts)) ||
      out.meets(Span(a->cu_seqlens, a->kv.batch + 1)) || out.meets(Span(a->kept, a->tokens)) || meets_table(out, a->kv))
    return ABFT_ERR_INVALID_ARG;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->layers <= kFewLayers ? keep_call<kFewLayers>(a, sms, s) : keep_call<kMostLayers>(a, sms, s);
}

int abft_kv_fork(const abft_kv_fork_args* a, void* stream) {
  if (a == nullptr) return ABFT_ERR_INVALID_ARG;
  int rc = check_layers(a->kv, a->pools, a->layers);
  if (rc != ABFT_OK) return rc;
  if (a->pairs < 0) return ABFT_ERR_INVALID_ARG;
  if (a->pairs > 65535) return ABFT_ERR_UNSUPPORTED;
  if (a->pairs == 0 || a->kv.batch == 0) return ABFT_OK;
  if (a->src == nullptr || a->dst == nullptr || a->pages == nullptr) return ABFT_ERR_INVALID_ARG;
  // Table and lengths are written: not the lists of the pairs.
  for (const int32_t* list : {a->src, a->dst, a->pages}) {
    const Span pairs(list, a->pairs);
    if (meets_table(pairs, a->kv) || pairs.meets(Span(a->kv.seq_lens, a->kv.batch))) return ABFT_ERR_INVALID_ARG;
  }
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->layers <= kFewLayers ? fork_call<kFewLayers>(a, s) : fork_call<kMostLayers>(a, s);
}

}  // extern "C"
