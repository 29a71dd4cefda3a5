"""The library builds without what only the paged cache's extension needs."""
import pytest

from vla_abft_estimate_b200 import _build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Builds into an empty folder; commands are recorded and leave their output."""
    monkeypatch.setattr(_build, "LIB_DIR", tmp_path)
    monkeypatch.setattr(_build, "OBJ_DIR", tmp_path / "obj")
    monkeypatch.setattr(_build, "LIB_PATH", tmp_path / "libabft_b200.so")
    monkeypatch.setattr(_build, "_nvcc", lambda: "/opt/cuda/bin/nvcc")
    ran, broken = [], set()

    def run(cmd, verbose):
        ran.append(cmd)
        if cmd[0] in broken:
            raise RuntimeError(f"{cmd[0]} failed")
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(_build, "_run", run)
    return ran, broken


def test_a_failing_extension_leaves_the_library(tree):
    ran, broken = tree
    broken.add("g++")
    with pytest.warns(UserWarning, match="not built"):
        assert _build.build() == _build.LIB_PATH
    assert _build.LIB_PATH.exists() and not _build.host_path().exists()
    broken.clear()
    before = len(ran)
    _build.build()  # the extension alone
    assert _build.host_path().exists() and [c[0] for c in ran[before:]] == ["g++"]


def test_without_torch_the_library_is_all(tree, monkeypatch):
    ran, _ = tree
    monkeypatch.setattr(_build, "_torch_version", lambda: None)
    assert _build.build() == _build.LIB_PATH and _build.LIB_PATH.exists()
    assert all(c[0] != "g++" for c in ran) and not _build.is_stale()


def test_a_failing_source_is_an_error(tree):
    _, broken = tree
    broken.add("/opt/cuda/bin/nvcc")
    with pytest.raises(RuntimeError):
        _build.build()
    assert not _build.LIB_PATH.exists()


def test_another_torch_has_another_extension(tree, monkeypatch):
    ran, _ = tree
    _build.build()
    assert not _build.is_stale()
    first, before = _build.host_path(), len(ran)
    monkeypatch.setattr(_build, "_torch_version", lambda: "99.0")
    assert _build.host_path() != first and _build.is_stale()
    _build.build()
    assert [c[0] for c in ran[before:]] == ["g++"] and first.exists() and _build.host_path().exists()


def test_a_cache_without_the_extension_takes_the_long_way(tree, monkeypatch):
    from vla_abft_estimate_b200 import paged

    monkeypatch.setattr(paged, "_HOST", None)
    with pytest.warns(UserWarning, match="missing"):
        calls = paged._host().Calls(b"", 0, 0, 0, 0, 0, 0)
    assert calls.append(None, None, None, None, None, None) is None
    assert calls.attend(False, None, None, None, None, 0, 0) is None


@pytest.mark.gpu
def test_the_long_way_gives_the_same(cuda_device, monkeypatch):
    import torch

    from vla_abft_estimate_b200 import paged

    from .test_gpu_paged_run import decode_state

    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda_device)

    def outputs():
        cache, q, k, v, rope = decode_state(cuda_device)
        x = cache.append(q, k, v, rope)
        cache.append(None, k, v, rope, cu_seqlens=cu)
        got = x, cache.decode(x), cache.prefill(x, cu), cache.prefill(x, cu, num_splits=3, scale=0.5)
        cache.check_status()
        return got

    want = outputs()
    monkeypatch.setattr(paged, "_HOST", paged._LongWay)
    for a, b in zip(outputs(), want):
        assert torch.equal(a, b)
