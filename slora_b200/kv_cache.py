"""8-bit paged KV cache: append, attention, read-back, eviction.

The reference keeps KV rows in the pool's 16-bit type (``slora/common/mem_allocator.py:229-234``), one row per token, and
its attention kernels read them there (``slora/models/llama/triton_kernel/token_attention_nopad_att1.py``).  Here a page
holds ``page_tokens`` tokens of every KV head in 8 bits with one scale per (page, KV head): half the bytes that a decode
step reads and half the memory, in buffers of the cache's own.  Pages are rows of a
:class:`~slora_b200.MemoryAllocator` that owns no buffers.

One layer of a step, between ``LoraBatchOps.lora_get_qkv`` and ``lora_get_o``::

    batch = KvBatch(page_table, kv_len, q_start, q_len, max_q_len)      # once per step
    cache.append(layer, batch, k, v, q=q, rope=(table, positions))      # rotate q and k, quantise k and v into the pages
    o = cache.attend(layer, batch, q)
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from .mem_allocator import MemoryAllocator
from .rotary import _positions, _rows

KINDS = {"int8": (torch.int8, _lib.KV_INT8, 127.0), "e4m3": (torch.float8_e4m3fn, _lib.KV_E4M3, 448.0)}


def _table_stride(t):
    """Entries from one row of a page table to the next."""
    if t.dtype != torch.int64 or t.dim() != 2 or (t.size(1) > 1 and t.stride(1) != 1):
        raise RuntimeError("page_table must be an int64 tensor [sequences, pages] with contiguous rows")
    if t.size(0) > 1 and t.stride(0) < t.size(1):
        raise RuntimeError("the rows of page_table overlap (an expanded tensor?)")
    return max(t.stride(0), t.size(1))


def _size(value, name):
    """``value`` as the C interface takes it: an int from 0 to 2^31 - 1."""
    if value < 0:
        raise RuntimeError(f"{name} must not be negative")
    if value > 0x7fffffff:
        raise RuntimeError(f"{name}={value} is 2^31 or more")
    return int(value)


class KvBatch:
    """The sequences of one step, as device tables; made once per step and used by every layer.

    ``page_table`` int64 ``[n, max_pages]`` (entries behind a sequence's last page are not read); ``kv_len`` int32
    ``[n]``: tokens in the cache, the step's new ones included; ``q_start`` / ``q_len`` int32 ``[n]``: the rows of q, k and
    v that are the sequence's new tokens (the reference's ``b_start_loc`` / ``b_seq_len``).  ``max_q_len`` bounds
    ``q_len`` (as ``max_len_in_batch`` does in the reference; it sizes launches), ``max_kv_len``, when given, ``kv_len``
    (up to the end of its page): the table's columns behind it are not looked at, and workspaces are sized by it.

    The kernels check every length and page; what they had to skip is in :meth:`status`.
    """

    def __init__(self, page_table, kv_len, q_start, q_len, max_q_len, max_kv_len=None):
        _lib.require_cuda(page_table, kv_len, q_start, q_len)
        stride = _table_stride(page_table)
        n = page_table.size(0)
        for name, t in (("kv_len", kv_len), ("q_start", q_start), ("q_len", q_len)):
            if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous int32 tensor with one entry per sequence")
            if t.device != page_table.device:
                raise RuntimeError(f"{name} and page_table lie on different devices")
        self.page_table, self.kv_len, self.q_start, self.q_len = page_table, kv_len, q_start, q_len
        self.max_q_len = _size(max_q_len, "max_q_len")
        self.max_kv_len = None if max_kv_len is None else _size(min(max_kv_len, 0x7fffffff), "max_kv_len")
        self._status = torch.zeros((1,), dtype=torch.int32, device=page_table.device)
        self._fields = [page_table.data_ptr(), stride, kv_len.data_ptr(), q_start.data_ptr(), q_len.data_ptr(),
                        self._status.data_ptr(), n, page_table.size(1), self.max_q_len]
        self.n_seq = n
        self._c = {}            # by the cache's page size
        self.workspaces = {}    # bytes that attention over this batch needs, by the call's sizes

    def _ptr(self, page_tokens):
        """The C struct for a cache with that page size (it counts columns of the page table)."""
        c = self._c.get(page_tokens)
        if c is None:
            f = list(self._fields)
            if self.max_kv_len is not None:
                f[7] = min(f[7], -(-self.max_kv_len // page_tokens))
            c = self._c[page_tokens] = _lib.Kv8Batch(*f)
        return ctypes.addressof(c)

    def status(self) -> int:
        """Status bits (``_lib.STATUS_BITS``) of the calls so far -- synchronises the current stream."""
        return int(self._status.item())

    def check(self):
        st = self.status()
        if st:
            what = ", ".join(v for k, v in _lib.STATUS_BITS.items() if st & k)
            raise RuntimeError(f"slora_b200: device reported: {what} (status {st})")


class KvCache8:
    """8-bit paged KV cache of ``layer_num`` layers.

    ``k[l]`` / ``v[l]``: ``[n_pages, kv_heads, page_tokens, head_dim]`` int8 or e4m3; ``k_scale[l]`` / ``v_scale[l]``: FP32
    ``[n_pages, kv_heads]``; ``weights[l]`` (with ``track_weights``): FP32 ``[n_pages, kv_heads, page_tokens]``, the
    attention weight each token has gathered.  ``page_tokens`` 16, 32, 64 or 128; ``head_dim`` 64, 128 or 256.
    """

    def __init__(self, n_pages, page_tokens, kv_heads, head_dim, layer_num=1, kind="int8", track_weights=False,
                 device="cuda"):
        if kind not in KINDS:
            raise RuntimeError(f"cache kind {kind!r} is none of {sorted(KINDS)}")
        shape = (n_pages, kv_heads, page_tokens, head_dim)
        k, v, ks, vs, w = [], [], [], [], [] if track_weights else None
        for _ in range(layer_num):
            k.append(torch.zeros(shape, dtype=torch.uint8, device=device).view(KINDS[kind][0]))
            v.append(torch.zeros(shape, dtype=torch.uint8, device=device).view(KINDS[kind][0]))
            ks.append(torch.zeros(shape[:2], dtype=torch.float32, device=device))
            vs.append(torch.zeros(shape[:2], dtype=torch.float32, device=device))
            if track_weights:
                w.append(torch.zeros(shape[:3], dtype=torch.float32, device=device))
        self._bind(k, v, ks, vs, w)

    @classmethod
    def from_buffers(cls, k, v, k_scale, v_scale, weights=None):
        """A cache over existing tensors (lists with one entry per layer; see the class for shapes)."""
        self = cls.__new__(cls)
        self._bind(list(k), list(v), list(k_scale), list(v_scale), None if weights is None else list(weights))
        return self

    def _bind(self, k, v, ks, vs, w):
        if not k or len({len(x) for x in (k, v, ks, vs)} | ({len(w)} if w is not None else set())) != 1:
            raise RuntimeError("a cache needs one k, v, k_scale and v_scale per layer (and weights for all layers or none)")
        if k[0].dim() != 4:
            raise RuntimeError("k must be [pages, kv_heads, page_tokens, head_dim]")
        kinds = [name for name, (dt, _, _) in KINDS.items() if dt == k[0].dtype]
        if not kinds:
            raise RuntimeError(f"No suitable kernel. cache dtype={k[0].dtype}")
        self.kind = kinds[0]
        self.n_pages, self.kv_heads, self.page_tokens, self.head_dim = k[0].shape
        if self.page_tokens not in (16, 32, 64, 128):
            raise RuntimeError(f"No suitable kernel. page_tokens={self.page_tokens} (16, 32, 64 or 128)")
        if self.head_dim not in (64, 128, 256):
            raise RuntimeError(f"No suitable kernel. head_dim={self.head_dim} (64, 128 or 256)")
        if self.n_pages < 1 or self.kv_heads < 1:
            raise RuntimeError("a cache needs at least one page and one KV head")
        self.device = k[0].device
        for name, ts, dt, dims in (("k", k, k[0].dtype, 4), ("v", v, k[0].dtype, 4), ("k_scale", ks, torch.float32, 2),
                                   ("v_scale", vs, torch.float32, 2), ("weights", w or [], torch.float32, 3)):
            for t in ts:
                if t.dtype != dt or t.shape != k[0].shape[:dims] or not t.is_contiguous() or t.device != self.device:
                    raise RuntimeError(f"{name} must be contiguous {dt} tensors {tuple(k[0].shape[:dims])} on one device")
        self.k, self.v, self.k_scale, self.v_scale, self.weights = k, v, ks, vs, w
        self.layer_num = len(k)
        self.c = [_lib.Kv8Cache(k[i].data_ptr(), v[i].data_ptr(), ks[i].data_ptr(), vs[i].data_ptr(),
                                w[i].data_ptr() if w is not None else 0, self.n_pages, self.page_tokens, self.kv_heads,
                                self.head_dim, KINDS[self.kind][1]) for i in range(self.layer_num)]
        self._ptr = [ctypes.addressof(c) for c in self.c]
        self._key = (self.kv_heads, self.head_dim, self.page_tokens)
        self._pages = None

    # -- pages ------------------------------------------------------------------------------------------
    @property
    def pages(self) -> MemoryAllocator:
        """The allocator of the cache's pages: ``pages.alloc(n)``, ``pages.free(index)``."""
        if self._pages is None:
            self._pages = MemoryAllocator(self.n_pages, 0, torch.uint8, self.kv_heads, self.head_dim, self.layer_num,
                                          device=self.device, allocate_buffers=False)
        return self._pages

    def bytes_per_token(self) -> float:
        """Bytes of all layers that a cached token takes, scales and weights included."""
        per = 2 * self.kv_heads * (self.head_dim + 4.0 / self.page_tokens)
        return self.layer_num * (per + (4 * self.kv_heads if self.weights is not None else 0))

    # -- operators --------------------------------------------------------------------------------------
    def append(self, layer, batch, k, v, q=None, rope=None, q_out=None):
        """Quantise the step's new keys and values (``[T, kv_heads, head_dim]``) into the pages.

        ``rope=(table, positions)`` turns k (which itself is not written) and, when given, q: in place, or into ``q_out``.
        Returns the turned q.  The scale of a (page, head) is the largest value over all its tokens; when a new token
        raises it, the page's older values are rounded to the new scale.  A page that is appended to must belong to one
        sequence only.  Rows of no sequence are left as they are; of a sequence with more new tokens than ``kv_len`` the last
        ``kv_len`` are appended, the others' q is not turned, and the status says so.  C entry ``slora_kv8_append``.
        """
        q_out, call = self._append_call(layer, batch, k, v, q, rope, q_out)
        _lib.call(*call)
        return q_out

    def _append_call(self, layer, batch, k, v, q=None, rope=None, q_out=None):
        """The checks of :meth:`append`, and what is left to do as the arguments of ``_lib.call``."""
        d, dtype = self.head_dim, k.dtype
        table = positions = None
        if rope is not None:
            table, positions = rope
        ctx = _lib.device_of(k, v, self.k[layer], batch.kv_len, q, q_out, positions, None if table is None else table.turns)
        shape, k_stride = _rows(k, "k", d)
        v_shape, v_stride = _rows(v, "v", d)
        if shape[1] != self.kv_heads or v_shape != shape or v.dtype != dtype:
            raise RuntimeError(f"k and v must be [tokens, {self.kv_heads}, {d}] tensors of one dtype")
        pos = turns = rot = layout = 0
        factor = 1.0
        if rope is not None:
            if table.head_dim != d:
                raise RuntimeError(f"the rotary table is for head_dim {table.head_dim}, the cache has {d}")
            _positions(positions, shape[0])
            pos, turns, rot, factor, layout = positions.data_ptr(), table.turns_ptr, table.rotary_dim, table.factor, table.layout_code
        qp = qop = q_heads = q_stride = qo_stride = 0
        if q is not None:
            if rope is None:
                raise RuntimeError("q is only turned: it needs rope=(table, positions)")
            q_shape, q_stride = _rows(q, "q", d)
            if q_out is None:
                q_out, qo_stride = q, q_stride
            else:
                out_shape, qo_stride = _rows(q_out, "q_out", d)
                if out_shape != q_shape or q_out.dtype != dtype:
                    raise RuntimeError("q_out must have q's shape and dtype")
            if q_shape[0] != shape[0] or q.dtype != dtype:
                raise RuntimeError("q must have k's tokens and dtype")
            qp, qop, q_heads = q.data_ptr(), q_out.data_ptr(), q_shape[1]
        elif q_out is not None:
            raise RuntimeError("q_out without q")
        return q_out, (ctx, _lib.lib.slora_kv8_append, self._ptr[layer], batch._ptr(self.page_tokens), k.data_ptr(), v.data_ptr(),
                       k_stride, v_stride, shape[0], qp, qop, q_heads, q_stride, qo_stride, pos, turns, rot, factor, layout,
                       _lib.dtype_code(dtype))

    def read(self, layer, batch, dtype, count, first=None):
        """Tokens ``first[b] .. first[b] + count`` of each sequence (default: from 0) as the 16-bit values they stand for:
        ``(k, v)`` ``[n, count, kv_heads, head_dim]``, zero at and beyond ``kv_len``.  C entry ``slora_kv8_read``."""
        code = _lib.dtype_code(dtype)
        count = _size(count, "count")
        ctx = _lib.device_of(self.k[layer], batch.kv_len, first)
        if first is not None and (first.dtype != torch.int32 or first.numel() != batch.n_seq or not first.is_contiguous()):
            raise RuntimeError("first must be a contiguous int32 tensor with one entry per sequence")
        shape = (batch.n_seq, count, self.kv_heads, self.head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        _lib.call(ctx, _lib.lib.slora_kv8_read, self._ptr[layer], batch._ptr(self.page_tokens), _lib.ptr(first), count,
                  k.data_ptr(), v.data_ptr(), code)
        return k, v

    def attend(self, layer, batch, q, out=None, lse=None, scale=None, window=0, add_weights=False):
        """Causal attention of ``q`` ``[T, heads, head_dim]`` over the cached keys and values; returns ``out``.

        A sequence's new tokens are its last: query ``j`` sees positions up to ``kv_len - q_len + j``, the last ``window``
        of them when ``window`` > 0.  ``heads`` is a multiple of the cache's KV heads.  ``scale`` defaults to
        ``head_dim ** -0.5``; ``lse`` (FP32 ``[T, heads]``) receives the logarithm of the softmax's sum.  A query that sees
        nothing gives 0 and ``-inf``; rows that belong to no sequence are left as they are.  ``out`` may be ``q`` unless
        ``add_weights`` is set, which reads q again.  At head_dim 256 long chunks of prompts are slow: the cache is read once
        per eight rows.

        ``add_weights`` adds every key's attention weight, summed over queries and the heads of its KV head, to
        ``weights[layer]``.  Up to 512 MB of scores are kept for that (by the capacity of the page table, or
        ``max_kv_len``); beyond they are computed again.  On pages that several sequences share their sums arrive in no
        fixed order; all else does not depend on timing.
        C entry ``slora_kv8_attend``.
        """
        d, dtype = self.head_dim, q.dtype
        ctx = _lib.device_of(q, self.k[layer], batch.kv_len, out, lse)
        shape, q_stride = _rows(q, "q", d)
        tokens, heads = shape[0], shape[1]
        if heads % self.kv_heads or heads == 0:
            raise RuntimeError(f"q has {heads} heads, which is no multiple of the cache's {self.kv_heads}")
        if add_weights and self.weights is None:
            raise RuntimeError("add_weights needs a cache with track_weights")
        window = _size(window, "window")
        code = _lib.dtype_code(dtype)
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=q.device)
            o_stride = heads * d
        else:
            out_shape, o_stride = _rows(out, "out", d)
            if out_shape != shape or out.dtype != dtype:
                raise RuntimeError("out must have q's shape and dtype")
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != (tokens, heads) or not lse.is_contiguous()):
            raise RuntimeError("lse must be a contiguous float32 tensor [tokens, heads]")
        if tokens == 0 or batch.n_seq == 0:
            return out
        # the size follows from the sizes in the key (and the device, which is the cache's)
        key = (self._key, tokens, heads, bool(add_weights))
        need = batch.workspaces.get(key)
        if need is None:
            with ctx or contextlib.nullcontext():    # it goes by the device's SMs
                need = batch.workspaces[key] = max(_lib.lib.slora_kv8_attend_workspace_bytes(
                    self._ptr[layer], batch._ptr(self.page_tokens), tokens, heads, int(add_weights)), 16)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        _lib.call(ctx, _lib.lib.slora_kv8_attend, self._ptr[layer], batch._ptr(self.page_tokens), q.data_ptr(), q_stride, tokens,
                  heads, out.data_ptr(), o_stride, _lib.ptr(lse), d ** -0.5 if scale is None else float(scale), window,
                  int(add_weights), ws.data_ptr(), need, code)
        return out

    def evict(self, layer, batch, budget, recent, sink=0, dest=None):
        """Bring sequences longer than ``budget`` tokens back to ``budget``, per KV head by accumulated weight.

        Kept are the first ``sink`` tokens, the last ``recent`` and, of the others, those with the largest ``weights``
        (ties: the lowest position); they move, in order, to the front of the sequence's own pages, or to the pages of
        ``dest`` (a :class:`KvBatch` whose ``page_table`` names pages that no sequence of ``batch`` uses).  In place a page must
        belong to one sequence.  Returns the kept
        positions, int32 ``[n, kv_heads, budget]``, -1 behind the last.  The caller's lengths become
        ``min(kv_len, budget)`` and the pages behind them are free; all layers must be brought back alike.
        C entry ``slora_kv8_evict``.
        """
        if self.weights is None:
            raise RuntimeError("evict needs a cache with track_weights")
        table = batch.page_table if dest is None else dest.page_table
        if table.size(0) != batch.n_seq:
            raise RuntimeError("dest must have one row of pages per sequence")
        budget, recent, sink = _size(budget, "budget"), _size(recent, "recent"), _size(sink, "sink")
        if budget < 1 or recent + sink > budget:
            raise RuntimeError("budget must hold the sink and the recent tokens")
        ctx = _lib.device_of(self.k[layer], batch.kv_len, table)
        kept = torch.empty((batch.n_seq, self.kv_heads, budget), dtype=torch.int32, device=self.device)
        _lib.call(ctx, _lib.lib.slora_kv8_evict, self._ptr[layer], batch._ptr(self.page_tokens), budget, recent,
                  sink, kept.data_ptr(), table.data_ptr(), _table_stride(table), table.size(1))
        return kept
