"""What autograd and tracers are told of the paged cache operators."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from .test_gpu_paged_run import decode_state

pytestmark = pytest.mark.gpu


def misaligned(t):
    """The same rows where the kernels cannot read them in place: the call goes the long way."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


def calls(cache, q, k, v, rope, cu):
    return {"append": lambda x=q: cache.append(x, k, v, rope), "decode": lambda x=q: cache.decode(x),
            "prefill": lambda x=q: cache.prefill(x, cu)}


@pytest.fixture
def state(cuda_device):
    cache, q, k, v, rope = decode_state(cuda_device)
    return cache, q, k, v, rope, torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda_device)


@pytest.mark.parametrize("which", ["k_pages", "v_pages"])
def test_pages_that_require_a_gradient_are_refused(state, which):
    cache = state[0]
    ops = calls(*state)
    want = {name: call().clone() for name, call in ops.items()}
    getattr(cache, which).requires_grad_()
    for name, call in ops.items():
        with pytest.raises(ValueError, match=which):
            call()
        with torch.no_grad():
            assert torch.equal(call(), want[name])


def test_a_rotation_table_that_requires_a_gradient_is_refused(state):
    cache, q, k, v, rope, _ = state
    learned = rope.clone().requires_grad_()
    with pytest.raises(ValueError, match="rope"):
        cache.append(q, k, v, learned)
    with torch.no_grad():
        assert torch.equal(cache.append(q, k, v, learned), cache.append(q, k, v, rope))


def test_tangents_are_refused(state):
    cache, q, k, v, rope, cu = state
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for call in calls(*state).values():
            with pytest.raises(ValueError, match="tangent"):
                call(dual)
        with pytest.raises(ValueError, match="tangent"):
            cache.append(q, fwd.make_dual(k, torch.ones_like(k)), v, rope)
        with pytest.raises(ValueError, match="tangent"):
            cache.append(q, k, v, fwd.make_dual(rope, torch.ones_like(rope)))
        for call in calls(*state).values():
            call()  # no dual among these


def test_calls_under_a_tracer_are_refused(state):
    cache, q, *_, cu = state
    for call in (lambda x: cache.decode(x), lambda x: cache.prefill(x, cu)):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, (q,), check_trace=False)
    assert cache.decode(q).shape == q.shape


@pytest.mark.parametrize("long_way", [False, True])
def test_what_a_call_writes_counts_as_modified(state, long_way):
    cache, q, k, v, rope, cu = state
    x = misaligned(q) if long_way else q

    def versions():
        return cache.k_pages._version, cache.v_pages._version, out._version

    out = torch.empty_like(q)
    before = versions()
    cache.append(x, k, v, rope, q_out=out)
    assert all(now > was for now, was in zip(versions(), before))
    for call in (lambda: cache.decode(x, out=out), lambda: cache.prefill(x, cu, out=out)):
        before = versions()
        call()
        now = versions()
        assert now[:2] == before[:2] and now[2] > before[2]
    # a tensor that autograd has saved
    w = torch.ones_like(q, requires_grad=True)
    y = (w * out).sum()
    cache.decode(x, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors(state):
    """Tensors made in inference mode count no versions; calls take them."""
    cache, q, k, v, rope, cu = state
    want = cache.decode(q)
    with torch.inference_mode():
        x, out = q.clone(), torch.empty_like(q)
        assert out.is_inference()
        assert torch.equal(cache.decode(x, out=out), want)
        assert torch.equal(cache.decode(misaligned(q), out=out), want)
        other = decode_state(q.device)[0]
        assert other.k_pages.is_inference()
        other.append(x, k, v, rope)
        other.append(None, k, v, rope)
