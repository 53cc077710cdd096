"""Paged key-value cache on libfanar_b200: what a model reads when it answers from the passages that a search found.

The ids that `search` returns name passages; with each passage's keys and values in pages of a `PagedKV`, they become
rows of a page table (`passage_table`), and the model's next token attends over these pages, then over its own.
`append` stores new tokens' keys and values with the position rotation on the way, `attend` is the attention of one new
token per sequence, `read` gives stored rows back as floating point.  The reference has no counterpart: it ends with
the ids.

Every call runs on the current torch stream, neither synchronises nor reads device memory on the host, and can be
captured into a CUDA graph.  The operators have no gradients and refuse inputs that require one.  Wrong arguments raise;
an index outside its table is skipped on the device and reported by `check_status()`.
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
_READ = (torch.float16, torch.bfloat16, torch.float32)
_WORK = {}  # (GPU, stream) -> workspace of attend


def _need(cond, what):
    if not cond:
        raise ValueError(what)


def _no_gradient(x, what):
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, which the cache's operators do not have (torch.no_grad())")


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
        for x, what in ((k, "k"), (v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if x is not None:
                _no_gradient(x, what)
        self.k, self.v, self.k_scale, self.v_scale, self.fill = k, v, k_scale, v_scale, fill
        self.pages, self.heads, self.page, self.dim = k.shape
        self.device, self.dtype = k.device, k.dtype
        self.scale = 1.0 / math.sqrt(self.dim)
        self._index = k.device.index
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        p = lambda t: None if t is None else t.data_ptr()
        ss = k_scale.stride() if i8 else (0, 0, 0)
        self._c = _lib.KvCache(p(k), p(v), p(k_scale), p(v_scale), p(fill), p(self.status), *k.stride()[:3], *ss,
                               self.pages, self.heads, self.page, self.dim, _CODE[k.dtype])
        self._ref = C.byref(self._c)
        self.L = _lib.lib()
        self._append, self._read, self._attend = self.L.fvs_kv_append, self.L.fvs_kv_read, self.L.fvs_kv_attend
        self._work_bytes = self.L.fvs_kv_attend_work(self.dim)
        check(min(self._work_bytes, 0), "kv_attend_work")
        self.launches = 0

    @classmethod
    def empty(cls, pages, heads, page, dim, dtype=torch.bfloat16, device="cuda", fill=None):
        """A cache with tensors of its own, rows of zeros (torch.int8: codes with scales)."""
        k, v = (torch.zeros(pages, heads, page, dim, dtype=dtype, device=device) for _ in range(2))
        scales = [torch.zeros(pages, heads, page, device=device) for _ in range(2)] if dtype == torch.int8 else [None] * 2
        return cls(k, v, *scales, fill=fill)

    # ---------------------------------------------------------------- arguments
    # A decoding step makes these calls for every layer, so each check is one condition and messages are made on failure.
    def _table(self, table):
        shape, stride = table.shape, table.stride()
        if not (len(shape) == 2 and table.dtype is torch.int32 and table.get_device() == self._index and shape[1] >= 1
                and (shape[1] == 1 or stride[1] == 1)):
            raise ValueError("the page table is an int32 [sequences, wide] with contiguous rows on the cache's GPU")
        return table.data_ptr(), shape[0], shape[1], stride[0]

    def _ints(self, t, n, what):
        if t is None:
            return None
        if not (t.dtype is torch.int32 and t.dim() == 1 and t.numel() == n and t.is_contiguous()
                and t.get_device() == self._index):
            raise ValueError(f"{what} is a contiguous int32 [{n}] on the cache's GPU")
        return t.data_ptr()

    def _heads(self, x, n, what, heads=None):
        """address, token stride and head stride of [n, heads, dim]"""
        shape = x.shape
        if not (len(shape) == 3 and shape[0] == n and shape[2] == self.dim and (heads is None or shape[1] == heads)
                and x.get_device() == self._index):
            raise ValueError(f"{what} is [{n}, {heads or 'heads'}, {self.dim}] on the cache's GPU")
        if x.requires_grad:
            _no_gradient(x, what)
        s0, s1, s2 = x.stride()
        at = x.data_ptr()
        if s2 != 1 or s0 % 8 or s1 % 8 or at % 16:
            raise ValueError(f"{what} needs contiguous, 16-byte aligned heads")
        return at, s0, s1

    def _type(self, dtype, what):
        if not (dtype in _WIDE and (self.dtype is torch.int8 or dtype is self.dtype)):
            raise ValueError(f"{what} is {dtype}: fp16 or bf16, and the cache's own type unless that holds int8 codes")
        return _CODE[dtype]

    def _like(self, out, x, what):
        if not (out.dtype is x.dtype and out.shape == x.shape and out.is_contiguous()
                and out.get_device() == self._index):
            raise ValueError(f"{what} is a contiguous tensor like q")
        return out.data_ptr()

    def _stream(self):
        if torch._C._cuda_getDevice() != self._index:
            raise ValueError(f"the cache is on GPU {self._index}, which is not the current one (torch.cuda.device)")
        return torch._C._cuda_getCurrentRawStream(self._index)  # torch.cuda.current_stream takes 2 us more

    # ---------------------------------------------------------------- the operators
    def append(self, k, v, table, idx, seq=None, pos=None, rope=None, pairs="halves", q=None, q_out=None):
        """Stores k, v [n, heads, dim] of n new tokens at logical places idx [n] (negative: not stored) of sequences seq
        [n] (default: token i is sequence i's).  The places of a call are distinct: where two tokens meet, the row is
        undefined afterwards.  rope: (cos, sin), fp32 [positions, rot / 2]: the first rot elements of the
        heads of k and of q [n, any, dim] are rotated at positions pos [n] (default idx), pairs "halves" (i, i + rot / 2)
        or "neighbours" (2i, 2i + 1).  Returns q_out, the rotated q (contiguous, default a new tensor, may be q; zeros for
        tokens that have no place), or None without q."""
        n = k.shape[0]
        ty = self._type(k.dtype, "k")
        if v.dtype is not k.dtype or (q is not None and q.dtype is not k.dtype):
            raise ValueError("k, v and q need one type")
        ka, va = self._heads(k, n, "k", self.heads), self._heads(v, n, "v", self.heads)
        qa, hq, qo = (None, 0, 0), 0, None
        if q is not None:
            qa, hq = self._heads(q, n, "q"), q.shape[1]
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            qo = self._like(q_out, q, "q_out")
        cos = sin = None
        positions = rot = 0
        if rope is not None:
            cos, sin = rope
            shape = cos.shape
            if not (cos.dtype is sin.dtype is torch.float32 and len(shape) == 2 and sin.shape == shape
                    and cos.is_contiguous() and sin.is_contiguous() and cos.get_device() == sin.get_device() == self._index):
                raise ValueError("rope is two contiguous fp32 [positions, rot / 2] on the cache's GPU")
            if cos.requires_grad or sin.requires_grad:
                for x in rope:
                    _no_gradient(x, "rope")
            positions, rot = shape[0], 2 * shape[1]
            if rot % 16 or not 0 < rot <= self.dim or positions < 1:
                raise ValueError(f"rotation of {rot} elements: a multiple of 16, at most {self.dim}")
            cos, sin = cos.data_ptr(), sin.data_ptr()
        if pairs not in _lib.PAIRS:
            raise ValueError(f"pairs {pairs!r}: one of {sorted(_lib.PAIRS)}")
        ta = self._table(table)
        if seq is None and n > ta[1]:
            raise ValueError("without seq there is a table row for each token")
        check(self._append(self._stream(), self._ref, ty, *ka, *va, *qa, hq, qo, *ta, self._ints(seq, n, "seq"),
                           self._ints(idx, n, "idx"), self._ints(pos, n, "pos"), n, cos, sin, positions, rot,
                           _lib.PAIRS[pairs]), "kv_append")
        self.launches += 1
        return q_out if q is not None else None

    def read(self, table, idx, seq=None, dtype=None):
        """The stored rows of tokens idx [n] of sequences seq [n] (default: token i is sequence i's) as (k, v), each
        [n, heads, dim] of `dtype` (fp16, bf16 or fp32; default the cache's, fp32 for int8 codes); zeros for a hole."""
        n = idx.shape[0]
        dtype = dtype or (torch.float32 if self.dtype is torch.int8 else self.dtype)
        if dtype not in _READ:
            raise ValueError(f"read as {dtype}: fp16, bf16 or fp32")
        ta = self._table(table)
        if seq is None and n > ta[1]:
            raise ValueError("without seq there is a table row for each token")
        k = torch.empty((n, self.heads, self.dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        check(self._read(self._stream(), self._ref, _CODE[dtype], k.data_ptr(), v.data_ptr(),
                         *ta, self._ints(seq, n, "seq"), self._ints(idx, n, "idx"), n), "kv_read")
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
        if hq < 1 or hq % self.heads:
            raise ValueError(f"{hq} query heads over {self.heads} key heads")
        ta = self._table(table)
        if ta[1] != n:
            raise ValueError(f"the page table has {ta[1]} rows for {n} sequences")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if lse is None:
            lse = torch.empty((n, hq), device=q.device)
        elif not (lse.dtype is torch.float32 and lse.shape == (n, hq) and lse.is_contiguous()
                  and lse.get_device() == self._index):
            raise ValueError("lse is a contiguous fp32 [sequences, query heads]")
        oa, la = self._like(out, q, "out"), self._ints(lens, n, "lens")
        if n == 0:
            return out, lse
        stream = self._stream()
        work, arrived = self._workspace(stream, 2 * n * hq + 2)
        check(self._attend(stream, self._ref, ty, *qa, hq, *ta, la, self.scale if scale is None else scale, oa,
                           lse.data_ptr(), work.data_ptr(), arrived.data_ptr()), "kv_attend")
        self.launches += 1
        return out, lse

    def _workspace(self, stream, n):
        """Tensors of the partial results and of n arrival counters (zeroed once, left zeroed by every call): one pair for
        each stream, whose calls come one after another, shared by all caches and held until `release_workspaces`.  A
        captured call's pair lives in its graph's memory, and the graph zeroes its counters: it may be replayed beside
        calls on any stream."""
        capturing = torch.cuda.is_current_stream_capturing()
        held = None if capturing else _WORK.get((self._index, stream))
        if held is None or held[0].numel() < self._work_bytes or held[1].numel() < n:
            work, arrived = (0, 0) if held is None else (held[0].numel(), held[1].numel())
            held = (torch.empty(max(self._work_bytes, work), dtype=torch.uint8, device=self.device),
                    torch.zeros(max(n, arrived), dtype=torch.int32, device=self.device))
            if not capturing:
                _WORK[self._index, stream] = held
        return held

    def check_status(self):
        """Raises if a call since the last check, on any stream, met an index outside its table (waits for the GPU)."""
        torch.cuda.synchronize(self.device)
        if int(self.status.item()) != 0:
            self.status.zero_()
            torch.cuda.synchronize(self.device)  # so that a call on any stream from here on is seen
            raise _lib.FvsError("paged cache: an index was outside its table (page, sequence, token or position); "
                                "that access was skipped")


def release_workspaces():
    """Gives the workspaces of attend back to torch's allocator (8 to 29 MB for each stream that attended; a stream's next
    call makes its own again).  Calls in flight keep what they have: the memory is used again on its own stream only."""
    _WORK.clear()


def passage_table(ids, pages_of, own=None):
    """Page table rows for found passages: ids [B, k] as `search` returns them (-1: none), pages_of int32 [N, m] the
    pages of each passage in order (-1 after its last), own int32 [B, w] the pages of each sequence's own tokens ->
    int32 [B, k * m + w].  The own tokens begin at logical token k * m * page.  An id that pages_of has no row for is a
    passage that is not there, like -1: its pages are holes."""
    _need(ids.dim() == 2 and not ids.is_floating_point(), "ids are whole numbers [sequences, passages of each]")
    _need(pages_of.dtype == torch.int32 and pages_of.dim() == 2, "pages_of is int32 [passages, pages of each]")
    B, k = ids.shape
    _need(own is None or (own.dtype == torch.int32 and own.dim() == 2 and own.shape[0] == B),
          f"own is int32 [{B}, pages of each]")
    N, m = pages_of.shape
    if N == 0:
        rows = pages_of.new_full((B, k * m), -1)
    else:
        there = (ids >= 0) & (ids < N)
        rows = pages_of[ids.clamp(0, N - 1).long()].masked_fill(~there[..., None], -1).reshape(B, k * m)
    return rows if own is None else torch.cat([rows, own], 1)
