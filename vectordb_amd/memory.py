"""Keys and values of language-model contexts in 8 bits, in pages: the store that attention reads, over everything or over
the tokens that an index found.

An index over a context's keys (``HierarchicalNSW`` or ``BruteforceSearch`` with the inner-product space, labels = token
numbers) answers which tokens matter for a query; ``KeyValueMemory.attend(select=labels)`` reads those, without ``select``
it reads all of them.  Everything runs on CUDA tensors and on torch's current stream of their device
(include/vdb_index.h, vdb_kv_*)."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import KvBatchStruct, KvMemoryStruct
from .rows4 import dtype_code, no_gradient, on_device


_needs = {}  # bytes of workspace by the sizes of a call
_E4M3, _F32, _I32 = torch.float8_e4m3fn, torch.float32, torch.int32


def _rows(x):
    """x [tokens, heads, dim], or a copy of it, as the kernels read it: heads of contiguous numbers, 16-byte steps; and the
    address and steps of that."""
    a, b, c = x.stride()
    at = x.data_ptr()
    if c != 1 or a % 8 or b % 8 or a < 0 or b < 0 or at % 16:
        x = x.clone(memory_format=torch.contiguous_format)  # (contiguous() may keep the odd stride of a dimension of size 1)
        a, b, c = x.stride()
        at = x.data_ptr()
    return x, at, a, b


class KeyValueMemory:
    """``pages`` pages of ``page_tokens`` tokens of ``kv_heads`` keys and values of ``head_dim`` numbers.

    ``k``, ``v``: float8_e4m3fn [pages, kv_heads, page_tokens, head_dim]; ``k_scale``, ``v_scale``: float32
    [pages, kv_heads].  A stored number is code * scale.  Which page holds what is the caller's: ``table`` [sequences, width]
    int32, token t of sequence b lies in page table[b, t // page_tokens]; a page that several sequences list is not
    appended to.  ``lengths`` [sequences] int32 counts a sequence's
    tokens, the new ones of the call included, for ``append`` and ``attend`` alike.  Neither call has a gradient: tensors that
    require one are refused where torch records operations."""

    def __init__(self, pages: int, page_tokens: int, kv_heads: int, head_dim: int, device="cuda"):
        code = lambda: torch.zeros((pages, kv_heads, page_tokens, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)  # noqa: E731
        scale = lambda: torch.ones((pages, kv_heads), dtype=torch.float32, device=device)  # noqa: E731
        self._take(code(), code(), scale(), scale())

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale) -> "KeyValueMemory":
        """A memory that is these tensors (shared, not copied)."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale)
        return self

    def _take(self, k, v, k_scale, v_scale):
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or k_scale.shape != shape[:2] or v_scale.shape != shape[:2]:
            raise ValueError("expected k, v [pages, kv_heads, page_tokens, head_dim] and k_scale, v_scale [pages, kv_heads]")
        if k.dtype is not _E4M3 or v.dtype is not _E4M3 or k_scale.dtype is not _F32 or v_scale.dtype is not _F32:
            raise ValueError("k, v: float8_e4m3fn; k_scale, v_scale: float32")
        index = k.get_device() if k.is_cuda else -1
        if index < 0 or v.get_device() != index or k_scale.get_device() != index or v_scale.get_device() != index:
            raise ValueError("k, v, k_scale, v_scale: CUDA tensors on one device")
        if k_scale.requires_grad or v_scale.requires_grad:
            no_gradient()
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("k, v, k_scale, v_scale must be contiguous")
        pages, heads, page_tokens, dim = shape
        if page_tokens < 16 or page_tokens > 1024 or page_tokens & (page_tokens - 1):
            raise ValueError("page_tokens must be a power of two in 16..1024")
        if dim < 32 or dim > 256 or dim % 32:
            raise ValueError("head_dim must be a multiple of 32 in 32..256")
        self._l = _lib.lib()
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self._index = k.device, index
        self.kv_heads, self.page_tokens, self.head_dim = heads, page_tokens, dim
        self._m = KvMemoryStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, page_tokens, dim)

    def _batch(self, table, lengths, offsets, max_new, tokens):
        n, index = lengths.shape[0], self._index
        if table.dtype is not _I32 or lengths.dtype is not _I32 or table.dim() != 2 or lengths.dim() != 1 or table.shape[0] != n:
            raise ValueError("table [sequences, width] and lengths [sequences]: int32")
        if table.get_device() != index or lengths.get_device() != index or not (table.is_contiguous() and lengths.is_contiguous()):
            raise ValueError(f"table and lengths: contiguous, on {self.device}")
        width = table.shape[1]
        if n and not width:
            raise ValueError("table: at least one page wide")
        if offsets is None:
            if tokens != n:
                raise ValueError(f"without offsets every sequence has one new token: {tokens} rows for {n} sequences")
            at = None
        elif offsets.dtype is not _I32 or offsets.shape != (n + 1,) or offsets.get_device() != index or not offsets.is_contiguous():
            raise ValueError(f"offsets: contiguous int32 [{n + 1}] on {self.device}")
        else:
            at = offsets.data_ptr()
        return KvBatchStruct(table.data_ptr(), lengths.data_ptr(), at, n, width or 1, tokens, max_new)

    def _check_rows(self, x, heads, what):
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads and shape[1] != heads) or x.get_device() != self._index:
            raise ValueError(f"{what}: expected [tokens, {heads or 'heads'}, {self.head_dim}] on {self.device}, got {tuple(shape)} on {x.device}")
        return shape

    def append(self, k, v, table, lengths, *, offsets=None, max_new=None, queries=None, cos=None, sin=None, interleaved: bool = False):
        """Stores the keys and values k, v [tokens, kv_heads, head_dim] of new tokens.

        Row b is the last token of sequence b, or with ``offsets`` [sequences + 1] int32 rows offsets[b] .. offsets[b + 1] - 1
        are its last ones (at most ``max_new`` of any sequence; by default all rows).  ``cos``, ``sin`` [positions, half]
        float32 turn the first 2 * half numbers of each key by its position's angles, in pairs (d, d + half), or (2 i, 2 i + 1)
        if ``interleaved``.  Returns ``queries`` [tokens, q_heads, head_dim], turned likewise (rows of no
        sequence: copied; None without queries; where nothing turns, ``queries`` itself)."""
        shape = self._check_rows(k, self.kv_heads, "k")
        t, dtype, index = dtype_code(k, "k"), k.dtype, self._index
        if v.shape != shape or v.dtype is not dtype or v.get_device() != index:
            raise ValueError("k and v: one shape, type and device")
        if k.requires_grad or v.requires_grad or (queries is not None and queries.requires_grad):
            no_gradient()
        tokens = shape[0]
        batch = self._batch(table, lengths, offsets, tokens if max_new is None else max_new, tokens)
        rot = positions = 0
        cos_at = sin_at = None
        if cos is not None and sin is not None:
            if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not _F32 or sin.dtype is not _F32:
                raise ValueError("cos and sin: float32 [positions, half]")
            if cos.get_device() != index or sin.get_device() != index or not (cos.is_contiguous() and sin.is_contiguous()):
                raise ValueError(f"cos and sin: contiguous, on {self.device}")
            if cos.requires_grad or sin.requires_grad:
                no_gradient()
            positions, rot = cos.shape
            rot *= 2
            if rot:
                cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
        elif cos is not None or sin is not None:
            raise ValueError("cos and sin go together")
        # (the tensors keep the copies alive until the launch)
        k, k_at, k0, k1 = _rows(k)
        v, v_at, v0, v1 = _rows(v)
        out = queries
        q_at = out_at = None
        q0 = q1 = q_heads = 0
        if queries is not None:
            shape = self._check_rows(queries, None, "queries")
            if shape[0] != tokens or queries.dtype is not dtype:
                raise ValueError(f"queries: [{tokens}, q_heads, {self.head_dim}] {dtype}")
            if rot:
                queries, q_at, q0, q1 = _rows(queries)
                out = torch.empty_like(queries, memory_format=torch.contiguous_format)
                q_heads, out_at = shape[1], out.data_ptr()
        on_device(index, self._l.vdb_kv_append_device, self._m, batch, t, k_at, k0, k1, v_at, v0, v1, cos_at, sin_at, positions, rot, interleaved,
                  q_at, q0, q1, q_heads, out_at)
        return out

    def attend(self, q, table, lengths, *, offsets=None, max_new=None, scale=None, window: int = 0, select=None, return_lse: bool = False):
        """Attention of queries q [tokens, q_heads, head_dim] over the memory: [tokens, q_heads, head_dim] in q's type, and
        with ``return_lse`` the logarithm of the softmax's sum, [tokens, q_heads] float32.

        Rows as in ``append``.  A query sees its own token and those before it, with ``window`` only the last ``window`` of
        them; with ``select`` [sequences, kv_heads, n] int64 (one new token per sequence) it sees the tokens with these
        numbers, each as often as listed; numbers outside the sequence are skipped, as a search's padding is.
        ``scale`` is 1 / sqrt(head_dim) unless given."""
        tokens, q_heads, dim = self._check_rows(q, None, "q")
        t = dtype_code(q, "q")
        if q.requires_grad:
            no_gradient()
        if q_heads == 0 or q_heads % self.kv_heads:
            raise ValueError(f"q: a multiple of {self.kv_heads} heads")
        if window < 0:
            raise ValueError("window must not be negative")
        batch = self._batch(table, lengths, offsets, tokens if max_new is None else max_new, tokens)
        n_select = 0
        if select is not None:
            if offsets is not None or window:
                raise ValueError("select goes with one new token per sequence and no window")
            if select.dtype != torch.int64 or select.dim() != 3 or tuple(select.shape[:2]) != (tokens, self.kv_heads) or select.get_device() != self._index:
                raise ValueError(f"select: int64 [{tokens}, {self.kv_heads}, n] on {self.device}")
            select = select.contiguous()
            n_select = select.shape[2]
            if n_select == 0:  # nothing to see: a list of one number that no sequence has
                select, n_select = torch.full((tokens, self.kv_heads, 1), -1, dtype=torch.int64, device=self.device), 1
        q, q_at, q0, q1 = _rows(q)
        # rows of no sequence are zeros
        device = self.device
        out = (torch.empty_like if offsets is None else torch.zeros_like)(q, memory_format=torch.contiguous_format)
        lse = (torch.empty if offsets is None else torch.zeros)((tokens, q_heads), dtype=_F32, device=device) if return_lse else None
        sizes = (self.kv_heads, self.page_tokens, dim, batch.count, batch.table_width, tokens, batch.max_new, offsets is None, q_heads, window, n_select)
        need = _needs.get(sizes)
        if need is None:
            if len(_needs) > 10000:
                _needs.clear()
            need = _needs[sizes] = self._l.vdb_kv_attend_workspace(self._m, batch, q_heads, window, n_select)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        on_device(self._index, self._l.vdb_kv_attend_device, self._m, batch, t, q_at, q0, q1, q_heads,
                  float(dim) ** -0.5 if scale is None else float(scale), window, None if select is None else select.data_ptr(), n_select,
                  out.data_ptr(), None if lse is None else lse.data_ptr(), None if work is None else work.data_ptr(), need)
        return (out, lse) if return_lse else out
