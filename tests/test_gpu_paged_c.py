"""The paged cache's C entries where Python never calls them so."""
import ctypes

import pytest
import torch

from vla_abft_estimate_b200 import _native as N

from .test_gpu_paged_run import decode_state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefill", [False, True])
def test_scratch_that_a_call_does_not_need_is_not_looked_at(cuda_device, prefill):
    """Short caches need none: a pointer that is given all the same, whatever its
    alignment, is no reason to refuse. Where scratch is needed it is one."""
    cache, q, *_ = decode_state(cuda_device)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda_device)
    want = cache.prefill(q, cu, num_splits=1) if prefill else cache.decode(q)
    space = torch.zeros(1 << 20, dtype=torch.uint8, device=cuda_device)
    out = torch.empty_like(q)
    a = N.PagedAttnArgs()
    a.kv, a.q, a.out, a.tokens, a.heads, a.scale = cache._kv, q.data_ptr(), out.data_ptr(), 3, 28, 128 ** -0.5
    a.q_token_stride, a.q_head_stride, _ = q.stride()
    a.o_token_stride, a.o_head_stride, _ = out.stride()
    a.cu_seqlens, a.num_splits = cu.data_ptr(), 1
    L = N.lib()
    call = L.abft_paged_prefill if prefill else L.abft_paged_decode
    size = L.abft_paged_prefill_workspace_bytes if prefill else L.abft_paged_decode_workspace_bytes
    assert size(ctypes.byref(a)) == 0
    a.workspace, a.workspace_bytes = space.data_ptr() + 4, 64
    stream = torch.cuda.current_stream().cuda_stream
    assert call(ctypes.byref(a), stream) == 0
    assert torch.equal(out, want)
    a.num_splits, a.num_sms = (2, 0) if prefill else (1, 2)  # pieces, or the list
    need = size(ctypes.byref(a))
    assert 0 < need < space.numel() - 16
    a.workspace_bytes = need - 1
    assert call(ctypes.byref(a), stream) == -4
    a.workspace_bytes = need
    assert call(ctypes.byref(a), stream) == -2
