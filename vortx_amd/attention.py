"""A quantized key/value cache in pages, and attention over it.

:class:`KvCache` holds the keys and values of one model layer in blocks of the
GGUF types Q8_0 or Q4_0, :class:`KvAttention` writes rows into it, reads them
back and computes attention over it, for single tokens, prompts and trees of
drafted tokens (``vx_kv_write`` and what follows it in include/vortx_hip.h;
the reference has none of this). What changes from step to step — page table,
lengths, starts — is device memory that the kernels read, so a captured graph
can be replayed on new values::

    cache = vx.KvCache(pages=512, page_tokens=64, heads=8, dim=128, k_type=vx.VX_Q8_0, v_type=vx.VX_Q8_0)
    kv = vx.KvAttention(0)
    plan = kv.plan(cache, table, lens, starts, q_heads=32, max_queries=1, max_len=8192)
    kv.write(cache, k, v, slots)     # this step's keys and values [tokens, 8, 128]
    kv.attend(out, q, plan)          # [tokens, 32, 128]

What goes before it in a step: :class:`KvPages` says which pages the sequences
hold and :meth:`KvAttention.resize` brings it to the step's lengths, with the
slots and positions of the new tokens, all on the device;
:meth:`KvAttention.rotate` norms and rotates queries and keys by position, and
:meth:`KvAttention.write_rotated` does it on their way into the cache::

    pages, step = vx.KvPages(512, 64, seqs=32, cols=128), vx.KvStep(32, tokens=32)
    plan = kv.plan(cache, pages.table, pages.lens, step.starts, q_heads=32, max_queries=1, max_len=8192)
    how = kv.rotation(vx.rotation_freqs(128), norm=True, q_weight=wq, k_weight=wk, eps=1e-6)
    kv.resize(pages, want, step)     # int32 [32]: tokens that each sequence is to hold
    kv.write_rotated(cache, q, q, k, v, step.positions, step.slots, how)
    kv.attend(out, q, plan)
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import vortx_amd as _vx

from . import _ADDR, _ByAddress, _Context, _ffi, _stream, _view_of
from ._ffi import VX_Q8_0, VortxError, check, lib

_WRITE, _READ, _ATTEND, _TREE = (_ADDR[n] for n in ("vx_kv_write", "vx_kv_read", "vx_attention", "vx_attention_tree"))
_ROTATE, _WRITE_ROTATED, _RESIZE = (_ADDR[n] for n in ("vx_rotate", "vx_kv_write_rotated", "vx_kv_resize"))


def _u32(**values) -> None:
    """Refuses what a 32-bit field would hold as another number."""
    for name, v in values.items():
        if not 0 <= v < 2 ** 32:
            raise VortxError(_ffi.VX_ERR_INVALID, f"{name} is {v}: a number from 0 to 2^32 - 1 is expected")


def kv_cache_size(pages: int, page_tokens: int, heads: int, dim: int, k_type: int = VX_Q8_0, v_type: int = VX_Q8_0) -> int:
    """Bytes of such a cache (vx_kv_cache_size)."""
    _u32(pages=pages, page_tokens=page_tokens, heads=heads, dim=dim, k_type=k_type, v_type=v_type)
    n = C.c_uint64()
    check(lib().vx_kv_cache_size(C.byref(_ffi.VxKvCache(None, 0, pages, page_tokens, heads, dim, k_type, v_type)), C.byref(n)))
    return n.value


class KvCache:
    """``pages`` pages of ``page_tokens`` tokens of ``heads`` key/value heads of
    ``dim`` values, K and V quantized as ``k_type`` and ``v_type``. ``data``: the
    memory (a contiguous uint8 GPU tensor of at least :func:`kv_cache_size`
    bytes); by default a new one. Slot ``page * page_tokens + i`` is token i of
    a page; its contents are undefined until it is written."""

    def __init__(self, pages: int, page_tokens: int, heads: int, dim: int, k_type: int = VX_Q8_0, v_type: int = VX_Q8_0,
                 device="cuda:0", data=None):
        import torch
        need = kv_cache_size(pages, page_tokens, heads, dim, k_type, v_type)
        if data is None:
            data = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
        if not (isinstance(data, torch.Tensor) and data.is_cuda and data.is_contiguous()):
            raise TypeError("cache data must be a contiguous GPU tensor")
        have = data.numel() * data.element_size()
        if have < need:
            raise VortxError(_ffi.VX_ERR_INVALID, f"the cache needs {need} bytes, the buffer holds {have}")
        self.pages, self.page_tokens, self.heads, self.dim = pages, page_tokens, heads, dim
        self.k_type, self.v_type, self.data = k_type, v_type, data
        self._c = _ffi.VxKvCache(data.data_ptr(), have, pages, page_tokens, heads, dim, k_type, v_type)
        self._addr = C.addressof(self._c)


def _array(t, name: str, shape, dtype="int32"):
    """Address of a GPU tensor of 4-byte elements; ``shape``: its sizes (None: any)."""
    import torch
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == getattr(torch, dtype)):
        raise TypeError(f"{name} must be an {dtype} tensor on the GPU")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise VortxError(_ffi.VX_ERR_SHAPE, f"{name} is {tuple(t.shape)}, not {shape}")
    if t.numel() and (t.stride(-1) != 1 and t.shape[-1] > 1 or t.dim() == 1 and not t.is_contiguous()):
        raise VortxError(_ffi.VX_ERR_UNSUPPORTED, f"{name} has strided elements")
    if t.dim() == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise VortxError(_ffi.VX_ERR_UNSUPPORTED, f"{name} has overlapping rows")
    return t.data_ptr()


def _ptr(t) -> int:
    return t.data_ptr() or None


def _row_stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _i32_on(device):
    """What torch makes int32 numbers with that kernels can reach."""
    import torch
    if torch.device(device).type != "cuda":
        raise TypeError(f"device is {device}: the GPU is expected")
    return dict(dtype=torch.int32, device=device)


class KvPages(_ByAddress):
    """Which of ``pages`` pages of ``page_tokens`` tokens ``seqs`` sequences
    hold, at most ``cols`` each (vx_kv_pages): int32 GPU tensors ``table``
    [seqs, cols], ``lens`` [seqs], and the stack of free pages, the first
    ``free_count`` [1] of ``free`` [pages]. A new one holds nothing, and page 0
    is on top of the stack. :meth:`KvAttention.resize` changes it."""

    def __init__(self, pages: int, page_tokens: int, seqs: int, cols: int, device="cuda:0"):
        import torch
        _u32(pages=pages, page_tokens=page_tokens, seqs=seqs, cols=cols)
        i32 = _i32_on(device)
        self.pages, self.page_tokens, self.seqs, self.cols = pages, page_tokens, seqs, cols
        self.table, self.lens = torch.zeros(seqs, cols, **i32), torch.zeros(seqs, **i32)
        self.free, self.free_count = torch.arange(pages - 1, -1, -1, **i32), torch.full((1,), pages, **i32)
        self._c = _ffi.VxKvPages(_ptr(self.table), _ptr(self.lens), _ptr(self.free), _ptr(self.free_count), seqs, cols, cols,
                                 page_tokens, pages, 0)
        self._at = C.addressof(self._c)  # (not a cache's address)


class KvStep(_ByAddress):
    """What :meth:`KvAttention.resize` says of a step's new tokens, up to
    ``tokens`` of them: int32 GPU tensors ``starts`` [seqs + 1] (of a batch),
    ``slots`` and ``positions`` [tokens]."""

    def __init__(self, seqs: int, tokens: int, device="cuda:0"):
        import torch
        _u32(seqs=seqs, tokens=tokens)
        i32 = _i32_on(device)
        self.seqs, self.tokens = seqs, tokens
        self.starts = torch.zeros(seqs + 1, **i32)
        self.slots, self.positions = torch.full((tokens,), -1, **i32), torch.zeros(tokens, **i32)
        self._call = (_ptr(self.starts), _ptr(self.slots), _ptr(self.positions), tokens)


def rotation_freqs(rotated: int, base: float = 10000.0, scale: float = 1.0, device="cuda:0"):
    """Radians a position of each of ``rotated`` / 2 pairs of dims, float64:
    scale * base^(-2 i / rotated)."""
    import torch
    return (scale * base ** (-2.0 * torch.arange(rotated // 2, dtype=torch.float64) / max(rotated, 1))).to(device)


@dataclass
class Rotation(_ByAddress):
    """How queries and keys are normed and rotated (:meth:`KvAttention.rotation`).
    It keeps the tensors it was made of alive; their contents may change."""
    dim: int       # of the heads that it is for (0: any that its rotated dims fit into)
    q_heads: int   # of weights of their own for each head (0: any)
    k_heads: int
    keep: tuple
    _c: object     # _ffi.VxRotation

    def __post_init__(self):
        self._call = (C.addressof(self._c), self.dim, self.q_heads, self.k_heads, self._c.rotated)


@dataclass
class AttentionPlan:
    """What attention calls of one batch share (:meth:`KvAttention.plan`): the
    cache, the batch's device arrays, options and a workspace. It keeps the
    tensors it was made of alive; their contents may change between calls.
    Calls that use one plan share its workspace, so they must be ordered.
    ``ws`` and ``ws_bytes`` are the workspace's address (None: none, the keys
    are not split) and size; ``max_queries``, ``seqs`` and ``tokens`` say what
    the plan was made for."""
    cache: KvCache
    q_heads: int
    max_queries: int
    seqs: int
    tokens: int          # most query tokens of a call that the workspace is made for
    first_tokens: object  # length of ``first``, or None
    workspace: object
    keep: tuple
    batch: object        # _ffi.VxAttnBatch
    opts: object         # _ffi.VxAttnOpts

    def __post_init__(self):
        self.workspace = self.workspace

    def __setattr__(self, name, value):
        set_ = object.__setattr__
        set_(self, name, value)
        if "opts" not in self.__dict__:
            return  # (not all there yet)
        if name == "workspace":
            set_(self, "ws", value.data_ptr())
            set_(self, "ws_bytes", value.numel() * value.element_size())
        if "ws_bytes" in self.__dict__:
            # what _pycall.attend takes: the structs' addresses, the workspace, and what q may be
            set_(self, "call", (self.cache._addr, C.addressof(self.batch), C.addressof(self.opts), self.ws or 0, self.ws_bytes, self.q_heads,
                                2 ** 32 - 1 if self.first_tokens is None else self.first_tokens))


def tree_mask(parents, device="cuda:0"):
    """The bit rows of drafted trees: ``parents`` has a list per sequence, the
    parent of each of its drafts (-1: the last cached token; a parent comes
    before its drafts). int32 [drafts in all, words], draft j of a sequence
    having bit i set where draft i is an ancestor of it or itself."""
    import torch
    words = max(1, -(-max((len(p) for p in parents), default=0) // 32))
    rows = []
    for tree in parents:
        seen = []
        for j, p in enumerate(tree):
            if not -1 <= p < j:
                raise VortxError(_ffi.VX_ERR_INVALID, f"draft {j} has parent {p}: one of -1..{j - 1} is expected")
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        rows += [[(m >> 32 * w) & 0xFFFFFFFF for w in range(words)] for m in seen]
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, words).to(torch.int32).to(device)


class KvAttention(_Context):
    """Rows into a :class:`KvCache` and out of it, and attention over it."""

    def write(self, cache: KvCache, k, v, slots, stream=None) -> None:
        """Quantize ``k`` and ``v`` ([tokens, heads, dim] f32 views) into the
        cache's ``slots`` (int32 [tokens]; one outside the cache leaves its
        token out; no slot twice)."""
        st = _vx._pycall.kv_write(_WRITE, self._ctx, stream, cache._addr, k, v, slots)
        if st is not None:
            if st:
                check(st)
            return
        kv, vv = _view_of(k, False), _view_of(v, False)
        check(lib().vx_kv_write(self._h, _stream(stream), C.byref(cache._c), C.byref(kv), C.byref(vv), self._slots(slots, k, v)))

    def read(self, k, v, cache: KvCache, slots, stream=None) -> None:
        """The values of the cache's ``slots`` into ``k`` and ``v`` ([tokens,
        heads, dim] f32 views; None: not that one); zeros for a slot outside
        the cache."""
        st = _vx._pycall.kv_read(_READ, self._ctx, stream, cache._addr, k, v, slots)
        if st is not None:
            if st:
                check(st)
            return
        kv, vv = (None if t is None else C.byref(_view_of(t, True)) for t in (k, v))
        check(lib().vx_kv_read(self._h, _stream(stream), kv, vv, C.byref(cache._c), self._slots(slots, k, v)))

    def resize(self, pages: KvPages, want, step: KvStep, stream=None) -> None:
        """Sequence s is to hold ``want[s]`` tokens (int32 [seqs]; negative: as
        many as it does): shorter ones give pages back, then longer ones take
        the pages that they need, in order, while there are any
        (vx_kv_resize). ``step`` gets the starts, slots and positions of the
        new tokens; a sequence that found too few pages keeps its length, and
        its tokens have slot -1. ``step.tokens`` has to be at least the new
        tokens of all sequences."""
        if step.seqs != pages.seqs:
            raise VortxError(_ffi.VX_ERR_SHAPE, f"the step is for {step.seqs} sequences, the pages for {pages.seqs}")
        st = _vx._pycall.kv_resize(_RESIZE, self._ctx, stream, pages._at, pages.seqs, want, *step._call)
        if st is not None:
            if st:
                check(st)
            return
        at = _array(want, "want", (pages.seqs,)) or None
        check(lib().vx_kv_resize(self._h, _stream(stream), C.byref(pages._c), at, *step._call))

    def rotation(self, freqs, *, pairs: bool = False, norm: bool = False, q_weight=None, k_weight=None, eps: float = 1e-6) -> Rotation:
        """How :meth:`rotate` and :meth:`write_rotated` treat a head (vx_rotation).
        ``freqs``: float64 [rotated / 2], radians a position
        (:func:`rotation_freqs`; None: no rotation) of the dims i and i +
        rotated / 2 or, with ``pairs``, 2 i and 2 i + 1. ``norm``: each head
        is divided by sqrt(mean(x^2) + ``eps``) first, and multiplied by
        ``q_weight`` / ``k_weight``, f32 [dim] or [heads, dim] (None: by nothing)."""
        import torch
        r = _ffi.VxRotation()
        if freqs is not None:
            if not (isinstance(freqs, torch.Tensor) and freqs.is_cuda and freqs.dtype == torch.float64):
                raise TypeError("freqs must be a float64 tensor on the GPU")
            if freqs.dim() != 1 or not freqs.is_contiguous():
                raise VortxError(_ffi.VX_ERR_SHAPE, "freqs is one row of numbers")
            r.freqs, r.rotated = _ptr(freqs), 2 * freqs.numel()
        r.flags = (_ffi.VX_ROTATE_PAIRS if pairs else 0) | (_ffi.VX_ROTATE_NORM if norm else 0)
        r.eps = eps
        dims, heads = set(), [0, 0]
        for i, (n, w) in enumerate((("q", q_weight), ("k", k_weight))):
            if w is None:
                continue
            each = isinstance(w, torch.Tensor) and w.dim() == 2
            setattr(r, n + "_weight", _array(w, n + "_weight", (None, None) if each else (None,), "float32"))
            dims.add(w.shape[-1])
            if each:
                heads[i] = w.shape[0]
                setattr(r, n + "_weight_stride", _row_stride(w))
        if len(dims) > 1:
            raise VortxError(_ffi.VX_ERR_SHAPE, "q_weight and k_weight have different dims")
        return Rotation(dims.pop() if dims else 0, *heads, (freqs, q_weight, k_weight), r)

    @staticmethod
    def _rotation(how, positions, q, k):
        """Address of the positions; what the rotation's tensors do not hold is refused."""
        tokens = None
        for n, v, heads in (("q", q, how.q_heads), ("k", k, how.k_heads)):
            if v is None:
                continue
            l = v.layout
            if l.rank != 3:
                raise VortxError(_ffi.VX_ERR_SHAPE, f"{n} is a [tokens, heads, dim] view")
            tokens = l.size[0]
            if how.dim and l.size[2] != how.dim:
                raise VortxError(_ffi.VX_ERR_SHAPE, f"{n} has {l.size[2]} dims, the norm weights {how.dim}")
            if heads and l.size[1] != heads:
                raise VortxError(_ffi.VX_ERR_SHAPE, f"{n} has {l.size[1]} heads, its norm weights {heads}")
        if positions is None:
            return None
        return _array(positions, "positions", (tokens,))

    def rotate(self, q_out, q, k_out, k, positions, how: Rotation, stream=None) -> None:
        """``q_out`` = ``q`` and ``k_out`` = ``k`` ([tokens, heads, dim] f32
        views; both of the keys' None: queries alone) normed and rotated by
        ``positions`` (int32 [tokens]). An output may be its input itself."""
        st = _vx._pycall.rotate(_ROTATE, self._ctx, stream, q_out, q, k_out, k, positions, *how._call)
        if st is not None:
            if st:
                check(st)
            return
        ov, qv = _view_of(q_out, True), _view_of(q, False)
        kov, kv = (None if t is None else _view_of(t, m) for t, m in ((k_out, True), (k, False)))
        ref = lambda v: None if v is None else C.byref(v)  # noqa: E731
        check(lib().vx_rotate(self._h, _stream(stream), C.byref(ov), C.byref(qv), ref(kov), ref(kv),
                              self._rotation(how, positions, qv, kv), C.byref(how._c)))

    def write_rotated(self, cache: KvCache, q_out, q, k, v, positions, slots, how: Rotation, stream=None) -> None:
        """:meth:`rotate` of ``q`` into ``q_out`` and of ``k``, which goes into
        the cache's ``slots`` with ``v`` as :meth:`write` puts it there, in one
        launch (queries of many tokens in a second; the same bits as the two
        calls). ``q`` and ``q_out`` None: keys alone."""
        st = _vx._pycall.kv_write_rotated(_WRITE_ROTATED, self._ctx, stream, cache._addr, q_out, q, k, v, positions, slots, *how._call)
        if st is not None:
            if st:
                check(st)
            return
        kv, vv = _view_of(k, False), _view_of(v, False)
        ov, qv = (None if t is None else _view_of(t, m) for t, m in ((q_out, True), (q, False)))
        ref = lambda v: None if v is None else C.byref(v)  # noqa: E731
        check(lib().vx_kv_write_rotated(self._h, _stream(stream), C.byref(cache._c), ref(ov), ref(qv), C.byref(kv), C.byref(vv),
                                        self._rotation(how, positions, qv, kv), self._slots(slots, k, v), C.byref(how._c)))

    @staticmethod
    def _slots(slots, *views):
        counts = {t[1].size[0] if isinstance(t, tuple) else t.shape[0] if t.dim() else None for t in views if t is not None}
        if len(counts) != 1:  # the library says what is wrong where the views differ
            counts = {None}
        return _array(slots, "slots", (counts.pop(),))

    def plan(self, cache: KvCache, table, lens, starts, *, q_heads: int, max_queries: int, max_len: int, tokens: int = 0,
             scale: float = 0.0, softcap: float = 0.0, slopes=None, causal: bool = True, window: int = 0, prefix=None,
             first=None) -> AttentionPlan:
        """A batch of sequences and how they attend (vx_attn_batch,
        vx_attn_opts). ``table`` int32 [sequences, pages of the longest],
        ``lens`` int32 [sequences] (keys, the queries' own among them),
        ``starts`` int32 [sequences + 1] (first query token of each, and the
        end). ``max_queries`` and ``max_len`` bound what the arrays hold,
        ``tokens`` the query tokens of a call (0: sequences * max_queries).
        Options: ``scale`` (0: 1 / sqrt(dim)); ``softcap`` c, c tanh(score /
        c); ``slopes`` f32 [q_heads], score - slope |distance|; ``causal``;
        ``window``, keys less than that many positions away; ``prefix`` int32
        [sequences], keys that every query sees; ``first`` int32 [tokens], the
        first key that a query sees."""
        import torch
        _u32(q_heads=q_heads, max_queries=max_queries, max_len=max_len, tokens=tokens, window=window)
        o = _ffi.VxAttnOpts(scale, softcap, None, None, None, _ffi.VX_ATTN_CAUSAL if causal else 0, window)
        seqs = lens.shape[0] if isinstance(lens, torch.Tensor) and lens.dim() == 1 else 0
        b = _ffi.VxAttnBatch(_array(table, "table", (seqs, None)), _array(lens, "lens", (None,)),
                             _array(starts, "starts", (seqs + 1,)), seqs, table.shape[1], _row_stride(table), max_queries, max_len, 0)
        if slopes is not None:
            o.slopes = _array(slopes, "slopes", (q_heads,), "float32")
        if prefix is not None:
            o.prefix = _array(prefix, "prefix", (seqs,))
        if first is not None:
            o.first = _array(first, "first", (None,))
        tokens = tokens or min(seqs * max_queries, 2 ** 32 - 1)
        n = C.c_uint64()
        check(lib().vx_attention_ws_size(self._h, C.byref(cache._c), C.byref(b), C.byref(o), tokens, q_heads, C.byref(n)))
        ws = torch.empty(max(16, n.value), dtype=torch.uint8, device=cache.data.device)
        return AttentionPlan(cache, q_heads, max_queries, seqs, tokens, None if first is None else first.shape[0], ws,
                             (table, lens, starts, slopes, prefix, first), b, o)

    def _views(self, out, q, plan):
        ov, qv = _view_of(out, True), _view_of(q, False)
        l = qv.layout
        if l.rank >= 3 and plan.first_tokens is not None and plan.first_tokens < l.size[l.rank - 3]:
            raise VortxError(_ffi.VX_ERR_SHAPE, "plan has a first key for fewer tokens than q has")
        if l.rank >= 2 and l.size[l.rank - 2] != plan.q_heads:
            raise VortxError(_ffi.VX_ERR_SHAPE, f"q has {l.size[l.rank - 2]} heads, the plan {plan.q_heads}")
        return ov, qv

    def attend(self, out, q, plan: AttentionPlan, stream=None) -> None:
        """out = softmax(q k^T) v over each sequence's cache; ``q`` and ``out``
        are [tokens, q_heads, dim] f32 views. A query that sees no key gives zeros."""
        st = _vx._pycall.attend(_ATTEND, _TREE, self._ctx, stream, out, q, None, *plan.call)
        if st is not None:
            if st:
                check(st)
            return
        ov, qv = self._views(out, q, plan)
        check(lib().vx_attention(self._h, _stream(stream), C.byref(ov), C.byref(qv), C.byref(plan.cache._c), C.byref(plan.batch),
                                 C.byref(plan.opts), plan.ws, plan.ws_bytes))

    def attend_tree(self, out, q, plan: AttentionPlan, tree, stream=None) -> None:
        """The same for drafted tokens, whose keys are the last of each
        sequence: a draft sees the cached keys and the drafts whose bits are
        set in its row of ``tree`` (int32 [tokens, words], :func:`tree_mask`).
        ``causal`` and ``prefix`` of the plan do not apply."""
        if tree is not None:
            st = _vx._pycall.attend(_ATTEND, _TREE, self._ctx, stream, out, q, tree, *plan.call)
            if st is not None:
                if st:
                    check(st)
                return
        ov, qv = self._views(out, q, plan)
        tokens = qv.layout.size[qv.layout.rank - 3] if qv.layout.rank >= 3 else None
        at = _array(tree, "tree", (tokens, None))
        check(lib().vx_attention_tree(self._h, _stream(stream), C.byref(ov), C.byref(qv), C.byref(plan.cache._c),
                                      C.byref(plan.batch), C.byref(plan.opts), at, tree.shape[1], _row_stride(tree), plan.ws,
                                      plan.ws_bytes))
