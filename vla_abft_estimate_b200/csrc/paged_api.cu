// paged_api.cu - the extern "C" entry points of the paged key-value cache:
// argument validation, workspace layout and launches. Declarations are in
// include/abft_b200.h.
#include "paged_launch.cuh"

using namespace abft;

namespace {

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

}  // namespace

extern "C" {

int abft_kv_append(const abft_kv_append_args* a, void* stream) {
  int rc = append_check(a);
  if (rc != ABFT_OK || a->tokens == 0 || a->kv.batch == 0) return rc;
  int dev = 0, sms = 0;
  if ((rc = paged_device(&dev, &sms)) != ABFT_OK) return rc;
  AppendParams p;
  append_params(a, &p);
  return append_call(p, a->kv, sms, stream);
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
