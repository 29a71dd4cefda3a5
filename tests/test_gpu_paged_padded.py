"""The decoder over paged caches with rows behind the last sequence, as a batch of
fixed size has them."""
import pytest
import torch

from vla_abft_estimate_b200.abft import AbftConfig, AbftInjector, AbftStatsCollector, CheapSumChecker
from vla_abft_estimate_b200.workloads import build_qwen2

from .test_gpu_paged import BF16
from .test_gpu_paged_run import TINY

pytestmark = pytest.mark.gpu


def poison(dev, rows):
    """Freed memory of a layer's sizes holds NaN: what a kernel leaves unwritten shows."""
    for cols in (TINY["hidden"], TINY["hidden"] * 2, TINY["inter"] * 2):
        held = [torch.full((rows, cols), float("nan"), dtype=BF16, device=dev) for _ in range(40)]
        del held


def test_rows_behind_the_last_sequence_disturb_nothing(cuda_device):
    """Logits of the sequences' rows as without the padding, of the padding
    finite, and no checked linear reports a fault."""
    dev = cuda_device
    model = build_qwen2(TINY, dev, seed=0)
    ids = torch.randint(0, 512, (187 + 69,), generator=torch.Generator().manual_seed(2)).to(dev)
    cu = torch.tensor([0, 37, 187], dtype=torch.int32, device=dev)
    cfg = AbftConfig(enable=True, checker_backend="b200", detect_only=False)
    stats = AbftStatsCollector()
    injector = AbftInjector(cfg, CheapSumChecker(cfg), stats, defer_reports=True)

    def logits(rows):
        caches = model.new_paged_caches(2, 160)
        caches.lens.copy_(torch.tensor([37, 150], dtype=torch.int32))
        poison(dev, rows)
        got = model.forward_paged(ids[:rows], caches, cu)
        for c in caches.layers:
            c.check_status()
        return got

    with torch.no_grad():
        plain = logits(256)
        with injector:
            checked = logits(256)
            injector.flush()
        want = logits(187)
    for got in (plain, checked):
        assert torch.isfinite(got).all()
        # other row counts may take other tiles in the linears: a few roundings
        assert (got[:187] - want).float().norm() <= 0.09 * want.float().norm()
    assert stats.export_summary()["abft"]["faults"]["detected_total"] == 0
