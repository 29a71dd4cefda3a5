// paged_draft_api.cu - the extern "C" entry points for drafted trees and forks
// over the paged cache: append by given positions, tree attention, accept, keep
// and fork. Declarations are in include/abft_b200.h.
#include "paged_draft.cuh"
#include "paged_launch.cuh"

using namespace abft;

namespace {

int check_layers(const abft_paged_kv& kv, const void* const* pools, int32_t layers) {
  if (layers < 1 || (pools == nullptr && layers != 1)) return ABFT_ERR_INVALID_ARG;
  if (layers > 4096) return ABFT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(pools) & 7u) != 0) return ABFT_ERR_ALIGNMENT;
  return check_kv(kv);
}

bool overlap(const void* a, const void* b, size_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + bytes && y < x + bytes;
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
  AppendParams p = append_params(&a->append);
  p.positions = a->positions;
  p.position_stride = a->position_stride;
  p.axes = a->axes;
  for (int i = 0, end = 0; i < kMostAxes; ++i) {
    if (i < a->axes) end += a->sections[i];
    p.axis_end[i] = end;
  }
  return append_call<true>(p, a->append.kv, sms, stream);
}

size_t abft_paged_tree_workspace_bytes(const abft_paged_tree_args* a) {
  return a == nullptr ? 0 : abft_paged_prefill_workspace_bytes(&a->attn);
}

int abft_paged_tree(const abft_paged_tree_args* a, void* stream) {
  return a == nullptr ? ABFT_ERR_INVALID_ARG : prefill_call<true>(&a->attn, a->parents, stream);
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
  // The lengths themselves, or an array of its own: not a part of them.
  if (a->lens_out != a->kv.seq_lens && overlap(a->lens_out, a->kv.seq_lens, a->kv.batch * sizeof(int32_t)))
    return ABFT_ERR_INVALID_ARG;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  KeepParams p;
  p.kv = view_of(a->kv);
  p.layers.pools = a->pools;
  p.layers.layers = a->layers;
  p.cu = a->cu_seqlens, p.kept = a->kept, p.counts = a->counts;
  p.lens_out = a->lens_out;
  p.tokens = static_cast<int32_t>(a->tokens);
  // A thread for each 16 bytes of a slot in all layers, as far as a cluster has them.
  const int64_t columns = int64_t{2} * a->layers * a->kv.kv_heads * a->kv.head_dim / 8;
  for (p.cluster = 1; p.cluster < kKeepCluster && int64_t{p.cluster} * kKeepThreads < columns;) p.cluster *= 2;
  const dim3 grid(a->kv.batch * p.cluster), block(kKeepThreads);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->kv.head_dim == 128 ? launch_clusters(p.cluster, kv_keep_kernel<128>, grid, block, 0, s, p)
                               : launch_clusters(p.cluster, kv_keep_kernel<64>, grid, block, 0, s, p);
}

int abft_kv_fork(const abft_kv_fork_args* a, void* stream) {
  if (a == nullptr) return ABFT_ERR_INVALID_ARG;
  int rc = check_layers(a->kv, a->pools, a->layers);
  if (rc != ABFT_OK) return rc;
  if (a->pairs < 0) return ABFT_ERR_INVALID_ARG;
  if (a->pairs > 65535) return ABFT_ERR_UNSUPPORTED;
  if (a->pairs == 0 || a->kv.batch == 0) return ABFT_OK;
  if (a->src == nullptr || a->dst == nullptr || a->pages == nullptr) return ABFT_ERR_INVALID_ARG;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  ForkParams p;
  p.kv = view_of(a->kv);
  p.layers.pools = a->pools;
  p.layers.layers = a->layers;
  p.src = a->src, p.dst = a->dst, p.pages = a->pages;
  p.pairs = a->pairs;
  const int64_t items = int64_t{2} * a->layers * a->kv.kv_heads;
  p.per_pair = static_cast<int32_t>((items + kForkWarps - 1) / kForkWarps);
  const int64_t blocks = int64_t{p.per_pair} * a->pairs;
  if (blocks >= (int64_t{1} << 31)) return ABFT_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks)), block(32 * kForkWarps);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->kv.head_dim == 128 ? launch(kv_fork_kernel<128>, grid, block, 0, s, p)
                               : launch(kv_fork_kernel<64>, grid, block, 0, s, p);
}

}  // extern "C"
