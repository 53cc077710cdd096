"""Trees of drafted tokens on libfanar_b200: what a small model drafts behind a sequence, and how much of it the target
model takes.

A tree of a sequence is `parents`: int32 [nodes], node i stands behind node parents[i], or behind the sequence itself
where that is -1; parents come before their children.  One step over a `PagedKV` cache, with one token of each sequence
pending (drawn, not in the cache yet): append it and the nodes behind it at the places behind the sequence (rotated at the
positions that their depth gives) and `PagedKV.attend_tree` in every layer, with the pending token as node 0 of a tree [-1] +
[p + 1 for p in parents]; `verify`, whose target has a row behind the pending token and one behind each node; and in every layer
`PagedKV.compact` of 0 and the path's nodes + 1.  The drawn token is pending then.  The reference has no counterpart: it ends
with the found rows' ids.

Calls run on the current torch stream, neither synchronise nor read device memory on the host, and can be captured into a
CUDA graph.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check

MAX_NODES = _lib.TREE_NODES
_CODE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32T}


def _probabilities(x, index, what, like=None):
    """address, sequence stride and row stride of [sequences, rows, vocabulary]"""
    shape = x.shape
    if not (len(shape) == 3 and x.dtype in _CODE and x.get_device() == index and (like is None or (
            shape == like.shape and x.dtype is like.dtype))):
        raise ValueError(f"{what} is [sequences, nodes + 1, vocabulary] fp32, fp16 or bf16 on one GPU" if like is None else
                         f"{what} is a tensor of the target's shape and type on its GPU")
    s0, s1, s2 = x.stride()
    if s2 != 1 and shape[2] != 1:
        raise ValueError(f"{what} needs contiguous rows")
    return x.data_ptr(), s0, s1


def _ints(x, shape, index, what):
    if not (x.dtype is torch.int32 and x.shape == shape and x.is_contiguous() and x.get_device() == index):
        raise ValueError(f"{what} is a contiguous int32 {list(shape)} on the target's GPU")
    return x.data_ptr()


def tree_stride(parents, seqs, nodes, index):
    """address of a tree's parents and the distance between the sequences' (0: one tree for all)"""
    shape = parents.shape
    if not (parents.dtype is torch.int32 and shape in ((nodes,), (seqs, nodes)) and parents.is_contiguous()
            and parents.get_device() == index):
        raise ValueError(f"parents is a contiguous int32 [{nodes}] or [{seqs}, {nodes}] on the same GPU")
    return parents.data_ptr(), nodes if len(shape) == 2 else 0


def verify(target, parents, tokens, u, draft=None, counts=None):
    """Which drafted tokens the target model takes, and its next token, from given random numbers.

    target  : [sequences, nodes + 1, vocabulary] fp32, fp16 or bf16, the target's probabilities: row 0 behind the sequence,
              row i + 1 behind node i
    parents : int32 [nodes] or [sequences, nodes]; tokens: int32 [sequences, nodes], what each node was drafted as
    u       : fp32 [sequences, nodes + 1] in [0, 1): one number for each node, the last for the next token
    draft   : like target, the probabilities that a node's children were drawn from (rows behind nodes without children
              are not looked at); None: drafted with certainty
    counts  : int32 [sequences], the nodes that a sequence has (default: all)

    Children are tried in order of their index: taken if u m q(x) < r(x), with r the target's probabilities and m = 1 at
    first; where one is refused r becomes max(r - m q, 0) and m its sum.  Behind the last node taken the next token is the
    first whose running sum of r passes u sum(r).  The tokens are distributed as the target's own.  Decisions are made in
    64 bits.  Returns (path int32 [sequences, nodes]: the nodes taken in order, then -1; kept int32 [sequences]: how many;
    token int32 [sequences]: the next token, -1 for a row without any probability)."""
    if not target.is_cuda:
        raise ValueError("target has to be on a GPU (the library has no CPU path)")
    index = target.get_device()
    ta = _probabilities(target, index, "target")
    seqs, nodes, vocab = target.shape[0], target.shape[1] - 1, target.shape[2]
    if not (0 <= nodes <= MAX_NODES and vocab >= 1):
        raise ValueError(f"{nodes} nodes over a vocabulary of {vocab}: 0 to {MAX_NODES} nodes, at least one token")
    da = (None, 0, 0) if draft is None else _probabilities(draft, index, "draft", target)
    for x in (target, draft, u):
        if x is not None and x.requires_grad and torch.is_grad_enabled():
            raise ValueError("verification has no gradient (torch.no_grad())")
    pa, stride = tree_stride(parents, seqs, nodes, index)
    ka = _ints(tokens, (seqs, nodes), index, "tokens")
    ca = None if counts is None else _ints(counts, (seqs,), index, "counts")
    if not (u.dtype is torch.float32 and u.shape == (seqs, nodes + 1) and u.is_contiguous() and u.get_device() == index):
        raise ValueError(f"u is a contiguous fp32 [{seqs}, {nodes + 1}] on the target's GPU")
    if torch._C._cuda_getDevice() != index:
        raise ValueError(f"the target is on GPU {index}, which is not the current one (torch.cuda.device)")
    path = torch.empty((seqs, nodes), dtype=torch.int32, device=target.device)
    kept, token = (torch.empty(seqs, dtype=torch.int32, device=target.device) for _ in range(2))
    check(_lib.lib().fvs_verify(torch._C._cuda_getCurrentRawStream(index), _CODE[target.dtype], *ta, *da, pa, stride, ka, ca,
                                u.data_ptr(), seqs, nodes, vocab, path.data_ptr(), kept.data_ptr(), token.data_ptr()),
          "verify")
    return path, kept, token
