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
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import vortx_amd as _vx

from . import _ADDR, _Context, _ffi, _stream, _view_of
from ._ffi import VX_Q8_0, VortxError, check, lib

_WRITE, _READ, _ATTEND, _TREE = (_ADDR[n] for n in ("vx_kv_write", "vx_kv_read", "vx_attention", "vx_attention_tree"))


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


def _row_stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


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
