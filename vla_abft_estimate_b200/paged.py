"""Paged key-value cache: appending with rotation, and the attention over it.

The cache of one decoder layer, next to the checked linears of a decode step
(``ops.abft_linear``, ``AbftInjector``): pages of token slots that sequences
of unlike length share, where a dense cache reserves the longest length for
each. PyTorch supplies memory and streams, every computation runs in
libabft_b200.so; tensors are CUDA bf16 or fp16 on an sm_100 device.

    cache = PagedKVCache(k_pages, v_pages, page_table, seq_lens)
    # each step: seq_lens counts the step's tokens already
    q = cache.append(q, k, v, rope, cu_seqlens=cu)   # rotate q and k, store k and v
    o = cache.prefill(q, cu)                         # causal, several tokens per sequence
    q = cache.append(q, k, v, rope)                  # one token per sequence
    o = cache.decode(q)

Drafted tokens, several continuations of a sequence at once, form trees: row i
of a sequence's new tokens has the row ``parents[i]`` above it (-1: none).

    layers = PagedLayers(caches)                     # every decoder layer's
    # in each layer: rotated by depth, not by slot; each row sees its ancestors
    q = cache.append(q, k, v, rope, cu_seqlens=cu, positions=positions)
    o = cache.tree(q, cu, parents)
    # once per step, for all layers: the path the model confirms, moved up
    kept, counts, token = layers.accept(cu, parents, ids, answers)
    layers.keep(cu, kept, counts)
    layers.fork(src, dst, pages)                     # samples or beams of one prompt

``page_table`` and ``seq_lens`` stay on the device and are read by the
kernels, so a captured step (``torch.cuda.graph``) replays with the lengths
and pages of the moment. Bad entries never lead outside the tensors; they set
bits that ``check_status`` turns into an error. Calls are queued on the
current stream of the cache's device; results and workspaces are allocated
there, per call. No derivatives: tensors that require a gradient (under grad
mode) or have a tangent are refused, and so are calls under a tracer; what a
call writes counts as modified in place.
"""
from __future__ import annotations

import ctypes
import importlib.util
import math
import warnings
from typing import Optional, Sequence, Tuple

import torch

from . import _build
from . import _native as N

_DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


def rope_table(positions: int, head_dim: int, theta: float = 1e6, device=None) -> torch.Tensor:
    """(cos, sin) of position p and pair j, angle p * theta^(-2j / head_dim):
    fp32 [positions, head_dim / 2, 2], computed in 64 bits (a 32-bit product
    of a far position loses the angle's fraction) and rounded once."""
    if head_dim % 2 or positions < 0:
        raise ValueError(f"rope_table takes an even head_dim and positions >= 0, got {head_dim} and {positions}")
    inv = float(theta) ** (-torch.arange(0, head_dim, 2, device=device, dtype=torch.float64) / head_dim)
    ang = torch.outer(torch.arange(positions, device=device, dtype=torch.float64), inv)
    return torch.stack((ang.cos(), ang.sin()), dim=-1).float()


def _i32(name: str, t: torch.Tensor, dim: int, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim or t.device != device:
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name} must be a {dim}-D int32 tensor on {device}, got {got}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride in its last dimension")


_HOST = None


class _LongWay:
    """In the place of the extension: every call goes through the checks below."""

    class Calls:
        def __init__(self, *cache_and_entries):
            pass

        def hold(self, k_pages, v_pages):
            pass

        def append(self, *args):
            return None

        def attend(self, *args):
            return None

        def drafts(self, *entries):
            pass

        def tree(self, *args):
            return None

    class Layers:
        def __init__(self, *caches_and_entries):
            pass

        def accept(self, *args):
            return None

        def keep(self, *args):
            return None

        def fork(self, *args):
            return None


def _host():
    """The extension of csrc/paged_host.cpp, built next to the library for the
    torch that is installed. Without it calls go through ctypes to the same
    kernels, which takes about 5 us longer."""
    global _HOST
    if _HOST is None:
        path = _build.host_path()
        if path.exists():
            spec = importlib.util.spec_from_file_location("_paged_host", path)
            _HOST = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(_HOST)
        if not hasattr(_HOST, "Layers"):
            warnings.warn(f"{path} is missing or of another build: calls of the paged cache take longer on the host; build it with "
                          "`python -m vla_abft_estimate_b200._build`")
            _HOST = _LongWay
    return _HOST


def _addresses(*names: str) -> list:
    return [ctypes.cast(getattr(N.lib(), name), ctypes.c_void_p).value for name in names]


def _derivative_free(name: str, t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which the paged cache operators do not give: call them under "
                         "torch.no_grad()")
    if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a tangent, which the paged cache operators do not carry on")


def _not_traced() -> None:
    if torch._C._get_tracing_state() is not None:
        raise ValueError("the paged cache operators cannot be traced: a trace would hold their results as constants")


def _mark_written(*tensors: Optional[torch.Tensor]) -> None:
    """Autograd learns that the tensors have been written."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _raise_status(bits: int) -> None:
    said = [text for bit, text in ((N.PAGED_BAD_PAGE, "a page_table entry outside the pool, or a page to fork into that is"),
                                   (N.PAGED_BAD_LEN, "a length below 0, beyond the table or below the new tokens"),
                                   (N.PAGED_BAD_ANGLE, "a position beyond the rotation table"),
                                   (N.PAGED_BAD_ROWS, "cu_seqlens that does not start at 0, falls or passes the rows"),
                                   (N.PAGED_TIMEOUT, "a bounded device wait gave up"),
                                   (N.PAGED_BAD_DRAFT, "a tree's parent that does not come before its child, or rows to keep "
                                                       "that do not rise within the new ones"),
                                   (N.PAGED_BAD_FORK, "a fork from or to a sequence outside the batch, to one that another "
                                                      "fork names, or into a page that another needs")) if bits & bit]
    raise ValueError("paged cache: " + "; ".join(said))


class PagedKVCache:
    """Pages, page table and lengths of one layer's cache.

    ``k_pages``, ``v_pages``: [num_pages, kv_heads, page_size, head_dim],
    dense within a page (the page stride is free, so both may be views of one
    [num_pages, 2, ...] pool), page_size 16, 32, 64 or 128, head_dim 64 or
    128. ``page_table``: int32 [batch, max_pages]; ``seq_lens``: int32
    [batch], the tokens of each sequence including the current step's. The
    object holds references: write new entries into the tensors in place.
    Sequences may share pages that neither appends to; tokens appended by one
    call must go to distinct slots. Slots at or behind a sequence's length
    may hold anything; keys and values below it are taken as finite numbers
    (a non-finite value of a slot may reach every query of its sequence that
    ``prefill`` or ``tree`` answers in the same call).
    """

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, *, status: Optional[torch.Tensor] = None):
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dim() != 4:
                raise ValueError(f"{name} must be [num_pages, kv_heads, page_size, head_dim], got {tuple(t.shape)}")
            if t.dtype not in _DTYPES:
                raise ValueError(f"{name} must be bfloat16 or float16, got {t.dtype}")
        if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != k_pages.device:
            raise ValueError("k_pages and v_pages must have one shape, type and device")
        num_pages, kv_heads, page_size, head_dim = k_pages.shape
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}, got "
                             f"{page_size} and {head_dim}")
        if kv_heads == 0:
            raise ValueError("k_pages has no heads")
        if not k_pages.is_cuda:
            raise ValueError("k_pages must be a CUDA tensor (the library has no CPU path)")
        dense = (page_size * head_dim, head_dim, 1)
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            inner = [(s, d) for s, d, n in zip(t.stride()[1:], dense, t.shape[1:]) if n > 1]
            if any(s != d for s, d in inner) or (num_pages > 1 and (t.stride(0) < kv_heads * dense[0] or t.stride(0) % 8)):
                raise ValueError(f"{name} must be dense within a page, pages a multiple of 8 elements apart; strides "
                                 f"{t.stride()} of shape {tuple(t.shape)}")
        dev = k_pages.device
        _i32("page_table", page_table, 2, dev)
        _i32("seq_lens", seq_lens, 1, dev)
        batch, max_pages = page_table.shape
        if seq_lens.shape[0] != batch:
            raise ValueError(f"seq_lens has {seq_lens.shape[0]} entries, page_table {batch} rows")
        if batch > 1 and page_table.stride(0) < max_pages:
            raise ValueError("page_table rows must not overlap")
        if batch and (num_pages == 0 or max_pages == 0):
            raise ValueError("a cache with sequences needs at least one page and one table column")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=dev)
        else:
            _i32("status", status, 1, dev)
            if status.shape[0] < 1:
                raise ValueError("status needs one entry")
        self._tensors = k_pages, v_pages, page_table, seq_lens, status
        self.batch, self.max_pages, self.num_pages = batch, max_pages, num_pages
        self.kv_heads, self.page_size, self.head_dim = kv_heads, page_size, head_dim
        self.dtype, self.device = k_pages.dtype, dev
        kv = N.PagedKv()
        kv.k_pages, kv.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
        kv.k_page_stride, kv.v_page_stride = k_pages.stride(0), v_pages.stride(0)
        kv.page_table, kv.table_stride, kv.seq_lens = page_table.data_ptr(), page_table.stride(0), seq_lens.data_ptr()
        kv.status = status.data_ptr()
        kv.num_pages, kv.page_size, kv.kv_heads, kv.head_dim = num_pages, page_size, kv_heads, head_dim
        kv.batch, kv.max_pages, kv.dtype = batch, max_pages, _DTYPES[k_pages.dtype]
        self._kv = kv
        self._index = dev.index
        entry = _addresses("abft_kv_append", "abft_paged_decode", "abft_paged_decode_workspace_bytes",
                           "abft_paged_prefill", "abft_paged_prefill_workspace_bytes")
        self._fast = _host().Calls(bytes(kv), dev.index, *entry)
        self._fast.hold(k_pages, v_pages)
        self._fast.drafts(*_addresses("abft_kv_append_at", "abft_paged_tree", "abft_paged_tree_workspace_bytes"))

    # The kernels hold the addresses: the tensors are written in place, not
    # replaced.
    k_pages = property(lambda self: self._tensors[0])
    v_pages = property(lambda self: self._tensors[1])
    page_table = property(lambda self: self._tensors[2])
    seq_lens = property(lambda self: self._tensors[3])
    status = property(lambda self: self._tensors[4])

    # ---- argument checks ------------------------------------------------------
    # A call whose arguments are all in order goes to the library through
    # _paged_host (csrc/paged_host.cpp), which returns None for any other; the
    # checks below then copy what has to be copied or say what is wrong.
    def _rows(self, name: str, t: torch.Tensor, tokens: Optional[int], heads: Optional[int]) -> torch.Tensor:
        """Checks [tokens, heads, head_dim] rows; returns them as the kernels
        can read them (16-byte pieces): themselves, or a dense copy."""
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
        shape = t.shape
        if (t.dtype != self.dtype or t.device != self.device or len(shape) != 3 or shape[2] != self.head_dim
                or (tokens is not None and shape[0] != tokens) or (heads is not None and shape[1] != heads)):
            raise ValueError(f"{name} must be a {self.dtype} tensor [{'tokens' if tokens is None else tokens}, "
                             f"{'heads' if heads is None else heads}, {self.head_dim}] on {self.device}, got {t.dtype} "
                             f"{tuple(shape)} on {t.device}")
        self._no_derivative(name, t)
        if not self._in_place(t):
            return t.clone(memory_format=torch.contiguous_format)
        return t

    _no_derivative = staticmethod(_derivative_free)
    _written = staticmethod(_mark_written)

    def _callable(self) -> None:
        _not_traced()
        self._no_derivative("k_pages", self.k_pages)
        self._no_derivative("v_pages", self.v_pages)

    @staticmethod
    def _in_place(t: torch.Tensor) -> bool:
        s = t.stride()
        return s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and t.data_ptr() % 16 == 0

    def _group(self, heads: int) -> None:
        if heads == 0 or heads % self.kv_heads or heads // self.kv_heads > 64:
            raise ValueError(f"q has {heads} heads: a multiple of the cache's {self.kv_heads} kv heads, at most 64 "
                             "for each, is needed")

    def _result(self, name: str, out: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
        if out is None:
            return torch.empty_like(like, memory_format=torch.contiguous_format)
        if self._rows(name, out, like.shape[0], like.shape[1]) is not out:
            raise ValueError(f"{name} must be 16-byte aligned, with strides a multiple of 8 and unit stride in its last "
                             "dimension")
        if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
            raise ValueError(f"{name} must not repeat memory")
        return out

    def _boundaries(self, cu: torch.Tensor) -> None:
        _i32("cu_seqlens", cu, 1, self.device)
        if cu.shape[0] != self.batch + 1:
            raise ValueError(f"cu_seqlens must have {self.batch + 1} entries, got {cu.shape[0]}")

    def _call(self, name: str, args) -> None:
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        N.check(name, getattr(N.lib(), name)(ctypes.byref(args), stream))

    # ---- operators --------------------------------------------------------------
    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, rope: Optional[torch.Tensor] = None, *,
               cu_seqlens: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               positions: Optional[torch.Tensor] = None,
               sections: Optional[Sequence[int]] = None) -> Optional[torch.Tensor]:
        """Stores the new tokens' keys and values and returns the rotated q.

        ``q`` [tokens, heads, head_dim], ``k`` and ``v`` [tokens, kv_heads,
        head_dim] (parts of one fused projection are read in place; rows that
        are not 16-byte aligned are copied first). ``cu_seqlens`` int32
        [batch + 1]: rows cu[b] to cu[b + 1] are the last tokens of sequence
        b, rows behind cu[batch] belong to none; without it row b is the
        newest token of sequence b, none where seq_lens[b] is 0. ``rope``:
        fp32 [positions, head_dim / 2, 2] (``rope_table``) rotates q and k by
        position, in fp32, rounded once; None stores k as it is. ``q_out``
        (may be ``q``, but not overlap it otherwise) receives q; rows of no
        sequence are left as they were (undefined without ``q_out``). q None
        stores k and v only.

        ``positions``: int32 [tokens] or [axes, tokens] (up to 4 axes), what the
        rotation goes by in place of the slots' places, which stay those of the
        lengths: a drafted token's depth behind the cache, an image patch's
        time, height and width. With several axes ``sections`` says how many
        pairs turn by each, in their order, head_dim / 2 in all.
        """
        if positions is None and sections is None:
            done = self._fast.append(q, k, v, rope, cu_seqlens, q_out)
            if done is not None:
                return done if type(done) is not int else N.check("abft_kv_append", done)
        elif positions is None:
            raise ValueError("sections without positions")
        else:
            positions, sections = self._axes(positions, sections)
            done = self._fast.append(q, k, v, rope, cu_seqlens, q_out, positions, sections)
            if done is not None:
                return done if type(done) is not int else N.check("abft_kv_append_at", done)
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                return self.append(q, k, v, rope, cu_seqlens=cu_seqlens, q_out=q_out, positions=positions, sections=sections)
        self._callable()
        by = N.KvAppendAtArgs()
        args = by.append
        args.kv = self._kv
        k = self._rows("k", k, None, self.kv_heads)
        tokens = k.shape[0]
        v = self._rows("v", v, tokens, self.kv_heads)
        if cu_seqlens is not None:
            self._boundaries(cu_seqlens)
            args.cu_seqlens = cu_seqlens.data_ptr()
        elif tokens != self.batch:
            raise ValueError(f"without cu_seqlens k must have one row for each of the {self.batch} sequences, got {tokens}")
        if rope is not None:
            if (not isinstance(rope, torch.Tensor) or rope.dtype != torch.float32 or rope.dim() != 3
                    or rope.shape[1] * 2 != self.head_dim or rope.shape[2] != 2 or rope.device != self.device
                    or not rope.is_contiguous() or rope.shape[0] == 0 or rope.data_ptr() % 16):
                raise ValueError(f"rope must be a contiguous, 16-byte aligned float32 [positions, {self.head_dim // 2}, 2] "
                                 f"tensor on {self.device}")
            self._no_derivative("rope", rope)
            args.rope, args.max_positions = rope.data_ptr(), rope.shape[0]
        if q is not None:
            self._group(q.shape[1] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0)
            q = self._rows("q", q, tokens, None)
            q_out = self._result("q_out", q_out, q)
            args.q, args.q_out, args.heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
            args.q_token_stride, args.q_head_stride, _ = q.stride()
            args.o_token_stride, args.o_head_stride, _ = q_out.stride()
        elif q_out is not None:
            raise ValueError("q_out without q")
        args.k, args.v, args.tokens = k.data_ptr(), v.data_ptr(), tokens
        args.k_token_stride, args.k_head_stride, _ = k.stride()
        args.v_token_stride, args.v_head_stride, _ = v.stride()
        if positions is not None:
            if rope is None:
                raise ValueError("positions without rope")
            _i32("positions", positions, 2, self.device)
            if positions.shape[1] != tokens or len(sections) != positions.shape[0]:
                raise ValueError(f"positions must be [tokens] or [axes, tokens] with a section for each axis, got "
                                 f"{tuple(positions.shape)} for {tokens} tokens and sections {sections}")
            if (not 1 <= len(sections) <= N.MOST_AXES or any(type(x) is not int or x < 0 for x in sections)
                    or sum(sections) * 2 != self.head_dim):
                raise ValueError(f"sections must be 1 to {N.MOST_AXES} whole numbers, {self.head_dim // 2} in all, got {sections}")
            by.positions, by.position_stride, by.axes = positions.data_ptr(), positions.stride(0), len(sections)
            for i, x in enumerate(sections):
                by.sections[i] = x
            self._call("abft_kv_append_at", by)
        else:
            self._call("abft_kv_append", args)
        self._written(self.k_pages, self.v_pages, q_out)
        return q_out

    def _axes(self, positions, sections):
        """positions as [axes, tokens], sections as a tuple."""
        if not isinstance(positions, torch.Tensor):
            raise TypeError(f"positions must be a torch.Tensor, got {type(positions).__name__}")
        if sections is None:
            sections = (self.head_dim // 2,)
        elif type(sections) is not tuple:
            sections = tuple(sections)
        return (positions[None] if positions.dim() == 1 else positions), sections

    def decode(self, q: torch.Tensor, *, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               num_sms: int = 0) -> torch.Tensor:
        """Attention of each sequence's newest token over its cache: ``q``
        [batch, heads, head_dim], returns the same shape. ``scale`` defaults
        to head_dim^-0.5. A sequence of length 0 gives zeros. ``out`` may be
        ``q``. ``num_sms``: SMs the caches are shared out to (0: all)."""
        return self._attention(False, q, None, scale, out, 0, num_sms)

    def prefill(self, q: torch.Tensor, cu_seqlens: torch.Tensor, *, scale: Optional[float] = None,
                out: Optional[torch.Tensor] = None, num_splits: int = 0) -> torch.Tensor:
        """Causal attention of the newest tokens of each sequence over its
        cache: rows cu[b] to cu[b + 1] of ``q`` [tokens, heads, head_dim] are
        the last tokens of sequence b (``append`` has stored their keys), and
        row i of n sees the slots up to seq_lens[b] - n + i. Chunks of any
        length, 0 and 1 included; rows behind cu[batch] are left as they were
        in ``out`` (undefined without one), which may be ``q``.
        ``num_splits``: pieces the keys of
        a block of query rows are cut into (0: chosen on the device for the
        sequences' lengths)."""
        return self._attention(True, q, cu_seqlens, scale, out, num_splits, 0)

    def tree(self, q: torch.Tensor, cu_seqlens: torch.Tensor, parents: torch.Tensor, *, scale: Optional[float] = None,
             out: Optional[torch.Tensor] = None, num_sms: int = 0) -> torch.Tensor:
        """Attention of a tree of drafted tokens for each sequence: rows as in
        ``prefill``, but row i of n sees the slots before the n new ones, its
        own and its ancestors'. ``parents`` int32 [tokens]: the place of row
        i's parent among its sequence's new rows, below i, or -1 for none (a row
        that follows the cached tokens directly; there may be several). Trees of
        any size, one row included. Everything else is as in ``prefill``;
        ``num_sms`` as in ``decode``."""
        return self._attention(True, q, cu_seqlens, scale, out, 0, num_sms, parents, True)

    def _attention(self, prefill, q, cu, scale, out, num_splits, num_sms, parents=None, tree=False):
        if tree:
            done = self._fast.tree(q, cu, parents, scale, out, num_splits, num_sms)
        else:
            done = self._fast.attend(prefill, q, cu, scale, out, num_splits, num_sms)
        name = "abft_paged_tree" if tree else "abft_paged_prefill" if prefill else "abft_paged_decode"
        if done is not None:
            return done if type(done) is not int else N.check(name, done)
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                return self._attention(prefill, q, cu, scale, out, num_splits, num_sms, parents, tree)
        self._callable()
        call = N.PagedTreeArgs()
        args = call.attn
        args.kv = self._kv
        if prefill:
            self._boundaries(cu)
            args.cu_seqlens = cu.data_ptr()
        if not isinstance(q, torch.Tensor):
            raise TypeError(f"q must be a torch.Tensor, got {type(q).__name__}")
        self._group(q.shape[1] if q.dim() == 3 else 0)
        q = self._rows("q", q, None if prefill else self.batch, None)
        if tree:
            _i32("parents", parents, 1, self.device)
            if parents.shape[0] != q.shape[0]:
                raise ValueError(f"parents must have an entry for each of the {q.shape[0]} rows, got {parents.shape[0]}")
            call.parents = parents.data_ptr()
            if any(st == 0 and size > 1 for st, size in zip(q.stride(), q.shape)):
                q = q.clone(memory_format=torch.contiguous_format)  # read as boxes of a tensor that does not repeat itself
        out = self._result("out", out, q)
        args.q, args.out, args.tokens, args.heads = q.data_ptr(), out.data_ptr(), q.shape[0], q.shape[1]
        args.q_token_stride, args.q_head_stride, _ = q.stride()
        args.o_token_stride, args.o_head_stride, _ = out.stride()
        args.scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if int(num_splits) < 0 or int(num_sms) < 0 or not math.isfinite(args.scale):
            raise ValueError(f"scale must be finite, num_splits and num_sms at least 0, got {scale}, {num_splits}, {num_sms}")
        args.num_splits, args.num_sms = int(num_splits), int(num_sms)
        given = call if tree else args
        need = int(getattr(N.lib(), name + "_workspace_bytes")(ctypes.byref(given)))
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)  # of this call alone
            args.workspace, args.workspace_bytes = ws.data_ptr(), need
        self._call(name, given)
        self._written(out)
        return out

    def check_status(self) -> None:
        """Raises ValueError when a call since the last check met a bad page
        entry, length, position or boundary on the device (which it skipped),
        and clears the record. Synchronises with the current stream: work queued on
        others is waited for by the caller."""
        bits = int(self.status.cpu()[0])
        if not bits:
            return
        self.status.zero_()
        _raise_status(bits)


class PagedLayers:
    """The caches of a model's layers, for what is done in all of them at once.

    ``layers``: a ``PagedKVCache`` for each (512 at most), with one page table, one
    array of lengths, one type and one geometry, and pools of their own. What the
    status tells of these calls is in the first layer's.
    """

    def __init__(self, layers: Sequence[PagedKVCache]):
        layers = tuple(layers)
        if not layers or not all(isinstance(c, PagedKVCache) for c in layers):
            raise TypeError("layers must be PagedKVCache objects, one at least")
        if len(layers) > N.MOST_LAYERS:
            raise ValueError(f"{len(layers)} layers: at most {N.MOST_LAYERS}")
        first = layers[0]

        def shared(c):
            kv = c._kv
            return (kv.page_table, kv.table_stride, kv.seq_lens, kv.k_page_stride, kv.v_page_stride, c.device, c.dtype,
                    c.batch, c.max_pages, c.num_pages, c.kv_heads, c.page_size, c.head_dim)

        if any(shared(c) != shared(first) for c in layers):
            raise ValueError("layers must share page table, lengths, type, shape and page strides")
        pools = [x for c in layers for x in (c._kv.k_pages or 0, c._kv.v_pages or 0)]
        if first.num_pages and len(set(pools)) != len(pools):
            raise ValueError("layers must have pools of their own, for keys and for values")
        self.layers, self.batch, self.device = layers, first.batch, first.device
        self._kv, self._index = first._kv, first._index
        self._pools = (ctypes.c_void_p * len(pools))(*pools)
        self._pages = tuple(x for c in layers for x in (c.k_pages, c.v_pages))
        self._fast = _host().Layers(bytes(self._kv), self._index, bytes(self._pools),
                                    *_addresses("abft_draft_accept", "abft_kv_keep", "abft_kv_fork"),
                                    self._pages, first.page_table, first.seq_lens)

    page_table = property(lambda self: self.layers[0].page_table)
    seq_lens = property(lambda self: self.layers[0].seq_lens)

    def _list(self, name: str, t: torch.Tensor, size: int) -> None:
        _i32(name, t, 1, self.device)
        if t.shape[0] != size:
            raise ValueError(f"{name} must have {size} entries, got {t.shape[0]}")

    def _callable(self) -> None:
        _not_traced()
        for c in self.layers:
            c._callable()

    def _call(self, name: str, args) -> None:
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        N.check(name, getattr(N.lib(), name)(ctypes.byref(args), stream))

    def accept(self, cu_seqlens: torch.Tensor, parents: torch.Tensor, ids: torch.Tensor,
               answers: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Which rows of each sequence's tree the model confirms: (kept,
        counts, token). ``ids`` int32 or int64 [tokens], the drafted tokens;
        ``answers`` of the same type, the token that the model gives behind each
        row. A row is confirmed when it has no parent (it was sampled already),
        or its parent is confirmed and ``answers[parent] == ids[row]``. ``kept``
        int32 [tokens]: for each sequence the path to its deepest confirmed row
        (the lowest of equals), as places among its new rows, then -1;
        ``counts`` int32 [batch] its length; ``token`` [batch] the last row's
        answer, -1 for a sequence without rows."""
        done = self._fast.accept(cu_seqlens, parents, ids, answers)
        if done is not None:
            return done if type(done) is not int else N.check("abft_draft_accept", done)
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                return self.accept(cu_seqlens, parents, ids, answers)
        _not_traced()
        self._list("cu_seqlens", cu_seqlens, self.batch + 1)
        for name, t in (("ids", ids), ("answers", answers)):
            if (not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64) or t.dim() != 1
                    or t.device != self.device or t.dtype != ids.dtype or t.shape != ids.shape):
                raise ValueError(f"{name} must be a 1-D int32 or int64 tensor on {self.device}, ids and answers alike")
        self._list("parents", parents, ids.shape[0])
        ids, answers = ids.contiguous(), answers.contiguous()
        kept = torch.empty(ids.shape, dtype=torch.int32, device=self.device)
        counts = torch.empty(self.batch, dtype=torch.int32, device=self.device)
        token = torch.empty(self.batch, dtype=ids.dtype, device=self.device)
        args = N.DraftAcceptArgs()
        args.cu_seqlens, args.parents = cu_seqlens.data_ptr(), parents.data_ptr()
        args.ids, args.answers = ids.data_ptr(), answers.data_ptr()
        args.kept, args.counts, args.next = kept.data_ptr(), counts.data_ptr(), token.data_ptr()
        args.status, args.tokens, args.batch = self._kv.status, ids.shape[0], self.batch
        args.id_bytes = ids.element_size()
        self._call("abft_draft_accept", args)
        return kept, counts, token

    def keep(self, cu_seqlens: torch.Tensor, kept: torch.Tensor, counts: torch.Tensor, *,
             lens_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Of each sequence's n new tokens (rows cu[b] to cu[b + 1] of the step)
        keeps the rows ``kept[cu[b]]`` to ``kept[cu[b] + counts[b] - 1]``, rising
        places among them: their keys and values move up to the slots behind
        the cache, in all layers, and ``seq_lens[b]`` falls by ``n - counts[b]``.
        ``lens_out``: int32 [batch] that gets the lengths instead (and overlaps
        none of the arrays, but may be ``counts``), ``seq_lens`` stays. Pages behind the new lengths stay in the table, for the caller to
        use again. A sequence with bad rows, boundaries, length or pages is left
        as it was, and the status tells. Returns the array of lengths written."""
        out = self.seq_lens if lens_out is None else lens_out
        done = self._fast.keep(cu_seqlens, kept, counts, out)
        if done is not None:
            N.check("abft_kv_keep", done)
            return out
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                return self.keep(cu_seqlens, kept, counts, lens_out=lens_out)
        self._callable()
        self._list("cu_seqlens", cu_seqlens, self.batch + 1)
        _i32("kept", kept, 1, self.device)
        self._list("counts", counts, self.batch)
        self._list("lens_out", out, self.batch)
        args = N.KvKeepArgs()
        args.kv, args.pools, args.layers = self._kv, ctypes.addressof(self._pools), len(self.layers)
        args.cu_seqlens, args.kept, args.counts = cu_seqlens.data_ptr(), kept.data_ptr(), counts.data_ptr()
        args.lens_out, args.tokens = out.data_ptr(), kept.shape[0]
        self._call("abft_kv_keep", args)
        _mark_written(*self._pages, out)
        return out

    def fork(self, src: torch.Tensor, dst: torch.Tensor, pages: torch.Tensor) -> None:
        """Lets sequences go on from others' caches: for each pair i (int32
        [pairs] each) sequence ``dst[i]`` gets the length and the full pages of
        ``src[i]``, which they share from now on, and, where the length ends
        inside a page, a copy of that page's slots in use, in all layers, in
        page ``pages[i]``, which no sequence may hold and which its row of the
        table names then (not looked at where the length ends with a page). -1
        in ``src`` or ``dst``: no pair. The lists are no part of the table or the
        lengths, which are written. Sources may be named by several pairs;
        a destination that is also a source or named twice, or a page that
        another pair names too or that is another source's last, is refused: the
        pair is left undone, and the status tells."""
        done = self._fast.fork(src, dst, pages)
        if done is not None:
            return N.check("abft_kv_fork", done)
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                return self.fork(src, dst, pages)
        self._callable()
        _i32("src", src, 1, self.device)
        self._list("dst", dst, src.shape[0])
        self._list("pages", pages, src.shape[0])
        args = N.KvForkArgs()
        args.kv, args.pools, args.layers = self._kv, ctypes.addressof(self._pools), len(self.layers)
        args.src, args.dst, args.pages, args.pairs = src.data_ptr(), dst.data_ptr(), pages.data_ptr(), src.shape[0]
        self._call("abft_kv_fork", args)
        _mark_written(*self._pages, self.page_table, self.seq_lens)

    def check_status(self) -> None:
        """``PagedKVCache.check_status`` for all layers at once."""
        words = {c.status.data_ptr(): c.status for c in self.layers}.values()
        bits = 0
        for x in torch.cat([w[:1] for w in words]).tolist():
            bits |= x
        if not bits:
            return
        for w in words:
            w.zero_()
        _raise_status(bits)
