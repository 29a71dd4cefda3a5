"""The decoder of several rotation axes over drafted trees."""
import pytest
import torch

from vla_abft_estimate_b200.workloads import build_qwen2

from .draft_reference import i32, packed, random_tree
from .test_gpu_draft_run import SMALL, depth_of

pytestmark = pytest.mark.gpu


def test_a_depth_is_every_axis_position(cuda_device):
    """Positions [tokens] or [1, tokens], a drafted token's depth, on a model with three axes: bit for bit what the same
    number on every axis gives, and what the model without axes gives."""
    dev = cuda_device
    trees = [random_tree(13, 1), random_tree(1, 2), random_tree(9, 3)]
    cu, parents = packed(trees)
    past = [17, 40, 3]
    depths = i32([p + d for p, t in zip(past, trees) for d in depth_of(t)], dev)
    g = torch.Generator().manual_seed(6)
    prompt = torch.randint(0, 211, (sum(past),), generator=g).to(dev)
    ids = torch.randint(0, 211, (cu[-1],), generator=g).to(dev)
    out = []
    with torch.no_grad():
        for sections, positions in (((8, 12, 12), depths), ((8, 12, 12), depths[None]), ((8, 12, 12), depths.repeat(3, 1)),
                                    (None, depths), ((32,), depths[None])):
            model = build_qwen2(dict(SMALL, rope_sections=sections) if sections else SMALL, dev, seed=3)
            caches = model.new_paged_caches(3, 100)
            caches.lens.copy_(i32(past))
            model.forward_paged(prompt, caches, i32([0, 17, 57, 60], dev))
            caches.lens.add_(i32([len(t) for t in trees], dev))
            out.append(model.forward_paged(ids, caches, i32(cu, dev), i32(parents, dev), positions))
            caches.together.check_status()
        assert all(torch.equal(x, out[0]) for x in out[1:])
        # one token for each sequence, at a depth of its own
        model = build_qwen2(dict(SMALL, rope_sections=(8, 12, 12)), dev, seed=3)
        steps = []
        for positions in (i32([17, 40, 3], dev), None, i32([[17, 40, 3]] * 3, dev)):
            caches = model.new_paged_caches(3, 100)
            caches.lens.copy_(i32(past))
            model.forward_paged(prompt, caches, i32([0, 17, 57, 60], dev))
            caches.lens.add_(1)
            steps.append(model.forward_paged(ids[:3], caches, positions=positions))
        assert all(torch.equal(x, steps[0]) for x in steps[1:])
        with pytest.raises(ValueError, match="section"):
            model.forward_paged(ids[:3], caches, positions=i32([[17, 40, 3]] * 2, dev))
