"""Paged key-value cache on libfanar_b200: what a model reads when it answers from the passages that a search found.

The ids that `search` returns name passages; with each passage's keys and values in pages of a `PagedKV`, they become
rows of a page table (`passage_table`), and the model's next token attends over these pages, then over its own.
`append` stores new tokens' keys and values with the position rotation on the way, `attend` is the attention of one new
token per sequence, `read` gives stored rows back as floating point.  The reference has no counterpart: it ends with
the ids.

Every call runs on the current torch stream, neither synchronises nor reads device memory on the host, and can be
captured into a CUDA graph.  Wrong arguments raise; an index outside its table is skipped on the device and reported by
`check_status()`.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from ._lib import check

HEAD_DIMS = (64, 96, 128, 192, 256)
_CODE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.int8: _lib.I8, torch.float32: _lib.F32T}
_WIDE = (torch.float16, torch.bfloat16)


def _need(cond, what):
    if not cond:
        raise ValueError(what)


class PagedKV:
    """One layer's cache over tensors that the caller owns.

    k, v             : [pages, heads, page, dim] fp16, bf16 or int8 codes, equal strides, each head's row contiguous and
                       16-byte aligned; dim one of HEAD_DIMS
    k_scale, v_scale : fp32 [pages, heads, page], for int8 codes: value = code * scale
    fill             : int32 [pages], the slots of each page that hold a token (default: all of them), e.g. of a
                       passage's last page; the caller keeps it up to date

    A page table is int32 [sequences, wide]: token t of sequence b lies in page table[b, t // page], slot t % page; a
    negative entry is a hole.
    """

    def __init__(self, k, v, k_scale=None, v_scale=None, fill=None):
        _need(k.is_cuda and v.device == k.device, "k and v have to be on one GPU (the library has no CPU path)")
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype, "k and v are [pages, heads, page, dim] of one type")
        _need(k.dtype in (torch.float16, torch.bfloat16, torch.int8), f"cache type {k.dtype}: fp16, bf16 or int8 codes")
        _need(min(k.shape) >= 1 and k.shape[3] in HEAD_DIMS, f"head dim {k.shape[3]}: one of {HEAD_DIMS}")
        _need(k.stride() == v.stride() and k.stride(3) == 1, "k and v need equal strides and contiguous rows")
        per = 16 // k.element_size()
        _need(all(s % per == 0 for s in k.stride()[:3]) and k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0,
              "k and v need 16-byte aligned rows")
        _need(k.stride(2) >= k.shape[3], "slots of a page overlap")
        i8 = k.dtype == torch.int8
        _need(i8 == (k_scale is not None) == (v_scale is not None), "int8 codes need k_scale and v_scale, other types none")
        if i8:
            _need(all(s.dtype == torch.float32 and s.shape == k.shape[:3] and s.device == k.device
                      for s in (k_scale, v_scale)) and k_scale.stride() == v_scale.stride(),
                  "k_scale and v_scale are fp32 [pages, heads, page] with equal strides")
        _need(fill is None or (fill.dtype == torch.int32 and fill.shape == k.shape[:1] and fill.is_contiguous()
                               and fill.device == k.device), "fill is a contiguous int32 [pages]")
        self.k, self.v, self.k_scale, self.v_scale, self.fill = k, v, k_scale, v_scale, fill
        self.pages, self.heads, self.page, self.dim = k.shape
        self.device, self.dtype = k.device, k.dtype
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        p = lambda t: None if t is None else t.data_ptr()
        ss = k_scale.stride() if i8 else (0, 0, 0)
        self._c = _lib.KvCache(p(k), p(v), p(k_scale), p(v_scale), p(fill), p(self.status), *k.stride()[:3], *ss,
                               self.pages, self.heads, self.page, self.dim, _CODE[k.dtype])
        self._ref = C.byref(self._c)
        self._work = {}      # stream -> workspace of attend: addresses, counters held, tensors
        self._captured = []  # workspaces of captured calls
        self.L = _lib.lib()
        self.launches = 0

    @classmethod
    def empty(cls, pages, heads, page, dim, dtype=torch.bfloat16, device="cuda", fill=None):
        """A cache with tensors of its own, rows of zeros (torch.int8: codes with scales)."""
        k, v = (torch.zeros(pages, heads, page, dim, dtype=dtype, device=device) for _ in range(2))
        scales = [torch.zeros(pages, heads, page, device=device) for _ in range(2)] if dtype == torch.int8 else [None] * 2
        return cls(k, v, *scales, fill=fill)

    # ---------------------------------------------------------------- arguments
    def _table(self, table):
        _need(table.dim() == 2 and table.dtype == torch.int32 and table.device == self.device
              and (table.shape[1] <= 1 or table.stride(1) == 1) and table.shape[1] >= 1,
              "the page table is an int32 [sequences, wide] with contiguous rows on the cache's GPU")
        return table.data_ptr(), table.shape[0], table.shape[1], table.stride(0)

    def _ints(self, t, n, what):
        if t is None:
            return None
        _need(t.dtype == torch.int32 and t.shape == (n,) and t.is_contiguous() and t.device == self.device,
              f"{what} is a contiguous int32 [{n}] on the cache's GPU")
        return t.data_ptr()

    def _heads(self, x, n, what, heads=None):
        """address, token stride and head stride of [n, heads, dim]"""
        _need(x.dim() == 3 and x.shape[0] == n and x.shape[2] == self.dim and (heads is None or x.shape[1] == heads)
              and x.device == self.device, f"{what} is [{n}, {heads or 'heads'}, {self.dim}] on the cache's GPU")
        s = x.stride()
        at = x.data_ptr()
        _need(s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and at % 16 == 0,
              f"{what} needs contiguous, 16-byte aligned heads")
        return at, s[0], s[1]

    def _type(self, dtype, what):
        _need(dtype in _WIDE and (self.dtype == torch.int8 or dtype == self.dtype),
              f"{what} is {dtype}: fp16 or bf16, and the cache's own type unless that holds int8 codes")
        return _CODE[dtype]

    # ---------------------------------------------------------------- the operators
    def append(self, k, v, table, idx, seq=None, pos=None, rope=None, pairs="halves", q=None, q_out=None):
        """Stores k, v [n, heads, dim] of n new tokens at logical places idx [n] (negative: not stored) of sequences seq
        [n] (default: token i is sequence i's).  rope: (cos, sin), fp32 [positions, rot / 2]: the first rot elements of the
        heads of k and of q [n, any, dim] are rotated at positions pos [n] (default idx), pairs "halves" (i, i + rot / 2)
        or "neighbours" (2i, 2i + 1).  Returns q_out, the rotated q (contiguous, default a new tensor, may be q; zeros for
        tokens that have no place), or None without q."""
        n = k.shape[0]
        ty = self._type(k.dtype, "k")
        _need(v.dtype == k.dtype and (q is None or q.dtype == k.dtype), "k, v and q need one type")
        ka, va = self._heads(k, n, "k", self.heads), self._heads(v, n, "v", self.heads)
        qa, hq, qo = (None, 0, 0), 0, None
        if q is not None:
            qa, hq = self._heads(q, n, "q"), q.shape[1]
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            _need(q_out.dtype == q.dtype and q_out.shape == q.shape and q_out.is_contiguous()
                  and q_out.device == q.device, "q_out is a contiguous tensor like q")
            qo = q_out.data_ptr()
        cos = sin = None
        positions = rot = 0
        if rope is not None:
            cos, sin = rope
            _need(cos.dtype == sin.dtype == torch.float32 and cos.dim() == 2 and cos.shape == sin.shape
                  and cos.is_contiguous() and sin.is_contiguous() and cos.device == sin.device == self.device,
                  "rope is two contiguous fp32 [positions, rot / 2] on the cache's GPU")
            positions, rot = cos.shape[0], 2 * cos.shape[1]
            _need(rot % 16 == 0 and 0 < rot <= self.dim and positions >= 1, f"rotation of {rot} elements: a multiple of 16, "
                  f"at most {self.dim}")
            cos, sin = cos.data_ptr(), sin.data_ptr()
        _need(pairs in _lib.PAIRS, f"pairs {pairs!r}: one of {sorted(_lib.PAIRS)}")
        _need(seq is not None or n <= table.shape[0], "without seq there is a table row for each token")
        check(self.L.fvs_kv_append(_lib.stream_handle(), self._ref, ty, *ka, *va, *qa, hq, qo, *self._table(table),
                                   self._ints(seq, n, "seq"), self._ints(idx, n, "idx"), self._ints(pos, n, "pos"), n,
                                   cos, sin, positions, rot, _lib.PAIRS[pairs]), "kv_append")
        self.launches += 1
        return q_out if q is not None else None

    def read(self, table, idx, seq=None, dtype=None):
        """The stored rows of tokens idx [n] of sequences seq [n] (default: token i is sequence i's) as (k, v), each
        [n, heads, dim] of `dtype` (fp16, bf16 or fp32; default the cache's, fp32 for int8 codes); zeros for a hole."""
        n = idx.shape[0]
        dtype = dtype or (torch.float32 if self.dtype == torch.int8 else self.dtype)
        _need(dtype in (torch.float16, torch.bfloat16, torch.float32), f"read as {dtype}: fp16, bf16 or fp32")
        _need(seq is not None or n <= table.shape[0], "without seq there is a table row for each token")
        k = torch.empty(n, self.heads, self.dim, dtype=dtype, device=self.device)
        v = torch.empty(n, self.heads, self.dim, dtype=dtype, device=self.device)
        check(self.L.fvs_kv_read(_lib.stream_handle(), self._ref, _CODE[dtype], k.data_ptr(), v.data_ptr(),
                                 *self._table(table), self._ints(seq, n, "seq"), self._ints(idx, n, "idx"), n), "kv_read")
        self.launches += 1
        return k, v

    def attend(self, q, table, lens, scale=None, out=None, lse=None):
        """Attention of one new token per sequence: q [sequences, query heads, dim] over the visible ones of the first
        lens [sequences] logical tokens (no hole, slot < fill); scale defaults to 1 / sqrt(dim); query heads in groups
        share a key head.  Returns (out like q, lse fp32 [sequences, query heads]): zeros and -inf where nothing is
        visible.  lse joins parts that were attended apart (other caches, other GPUs): weights e^(lse - max lse)."""
        n = q.shape[0]
        ty = self._type(q.dtype, "q")
        qa = self._heads(q, n, "q")
        hq = q.shape[1]
        _need(hq >= 1 and hq % self.heads == 0, f"{hq} query heads over {self.heads} key heads")
        _need(table.shape[0] == n, f"the page table has {table.shape[0]} rows for {n} sequences")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _need(out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous() and out.device == q.device,
                  "out is a contiguous tensor like q")
        if lse is None:
            lse = torch.empty(n, hq, device=q.device)
        else:
            _need(lse.dtype == torch.float32 and lse.shape == (n, hq) and lse.is_contiguous()
                  and lse.device == q.device, "lse is a contiguous fp32 [sequences, query heads]")
        if n == 0:
            return out, lse
        stream = _lib.stream_handle()
        work, arrived = self._workspace(stream.value, n * hq)
        check(self.L.fvs_kv_attend(stream, self._ref, ty, *qa, hq, *self._table(table), self._ints(lens, n, "lens"),
                                   1.0 / math.sqrt(self.dim) if scale is None else scale, out.data_ptr(),
                                   lse.data_ptr(), work, arrived), "kv_attend")
        self.launches += 1
        return out, lse

    def _workspace(self, stream, n):
        """Addresses of the partial results and of n arrival counters (zeroed once, left zeroed by every call), one pair for
        each stream; a captured call gets its own, whose counters its graph zeroes, because the graph may be replayed
        beside calls on any stream."""
        capturing = torch.cuda.is_current_stream_capturing()
        held = None if capturing else self._work.get(stream)
        if held is None or held[2] < n:
            need = self.L.fvs_kv_attend_work(self.dim)
            if need < 0:
                check(need, "kv_attend_work")
            work = torch.empty(need, dtype=torch.uint8, device=self.device)
            arrived = torch.zeros(n + 2, dtype=torch.int32, device=self.device)
            held = (work.data_ptr(), arrived.data_ptr(), n, work, arrived)
            if capturing:
                self._captured.append(held)
            else:
                self._work[stream] = held
        return held[:2]

    def check_status(self):
        """Raises if a call since the last check met an index outside its table (synchronises)."""
        if int(self.status.item()) != 0:
            self.status.zero_()
            raise _lib.FvsError("paged cache: an index was outside its table (page, sequence, token or position); "
                                "that access was skipped")


def passage_table(ids, pages_of, own=None):
    """Page table rows for found passages: ids [B, k] as `search` returns them (-1: none), pages_of int32 [N, m] the
    pages of each passage in order (-1 after its last), own int32 [B, w] the pages of each sequence's own tokens ->
    int32 [B, k * m + w].  The own tokens begin at logical token k * m * page."""
    B = ids.shape[0]
    _need(pages_of.dtype == torch.int32 and pages_of.dim() == 2, "pages_of is int32 [passages, pages of each]")
    rows = pages_of[ids.clamp(min=0).long()]
    rows = torch.where((ids >= 0)[..., None], rows, torch.full_like(rows, -1)).reshape(B, -1)
    return rows if own is None else torch.cat([rows, own], 1)
