"""Beam search: selection over beams and vocabulary, and reordering of what belongs to a beam (``csrc/beam.cu``).

The engine's head samples one sequence (``head.py``); these entry points rank the continuations of several beams of several
requests.  The rows that ``beam_select`` returns go to ``ops.paged.fork_pages`` (pages of the cache) and to ``reorder_rows``
(recurrent states, conv histories, whatever has one row per beam).
"""

from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence, Tuple

import torch

from .lib import check_status, load as lib, longs, on_device, ptr, same_cuda_device
from .rope import TYPES

MAX_K = 64
MAX_BEAMS = 256
MAX_VOCAB = 1 << 24
_TENSORS = 16      # tensors of one launch of the reorder kernel


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, *, finished: Optional[torch.Tensor] = None, eos: int = -1,
                status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``k`` (at most 64) best continuations of every request: ``logits [requests, beams, vocabulary]`` (bf16, fp16 or fp32),
    ``scores`` fp32 ``[requests, beams]``, the beams' log-probabilities so far (-inf: a beam that does not exist).  Returns, best first,
    ``(scores fp32, rows int32, tokens int32)``, each ``[requests, k]``; ``rows`` counts beams over all requests (request * beams + beam).

    The total of a candidate is the beam's score plus the logit's log-softmax, in 64 bits; equal totals go to the lower beam, then
    to the larger logit, then to the lower token.  A beam marked in ``finished`` (bool ``[requests, beams]``) has one candidate, token
    ``eos`` at its own score.  Where fewer than ``k`` candidates are above -inf the rest are at -inf.  A beam with a NaN or +inf among its
    logits, or as its score, has no candidate and latches ``NON_FINITE`` in ``status``."""
    what = "beam_select"
    if logits.dim() != 3 or logits.dtype not in TYPES or (logits.shape[2] > 1 and logits.stride(2) != 1):
        raise ValueError(f"{what}: logits is [requests, beams, vocabulary] in bf16, fp16 or fp32 with a contiguous last dimension")
    batch, beams, vocab = logits.shape
    if not 1 <= beams <= MAX_BEAMS or not 1 <= vocab <= MAX_VOCAB or batch * beams > 65535:
        raise ValueError(f"{what}: at most {MAX_BEAMS} beams, 65535 in all, and a vocabulary of {MAX_VOCAB}")
    if not 1 <= k <= min(MAX_K, beams * vocab):
        raise ValueError(f"{what}: k is between 1 and {MAX_K} and no more than there are candidates")
    if scores.dtype != torch.float32 or scores.shape != (batch, beams):
        raise ValueError(f"{what}: scores is fp32 [requests, beams]")
    if finished is not None and (finished.dtype != torch.bool or finished.shape != (batch, beams) or not 0 <= eos < vocab):
        raise ValueError(f"{what}: finished is bool [requests, beams], with an end token of the vocabulary")
    check_status(what, status)
    device = same_cuda_device(what, logits, scores, finished, status)
    best = scores.new_empty((batch, k))
    rows, tokens = scores.new_empty((batch, k), dtype=torch.int32), scores.new_empty((batch, k), dtype=torch.int32)
    if batch:
        L = lib()
        scratch = scores.new_empty(batch * beams * L.nexrt_beam_slices(batch * beams, vocab, TYPES[logits.dtype]) * (k + 2), dtype=torch.int64)
        strides = longs(*logits.stride()[:2], *scores.stride(), *(finished.stride() if finished is not None else (0, 0)))
        on_device(device, lambda st: L.nexrt_beam_select(
            logits.data_ptr(), scores.data_ptr(), ptr(finished), strides, best.data_ptr(), rows.data_ptr(), tokens.data_ptr(), scratch.data_ptr(), ptr(status), batch, beams,
            vocab, k, eos, TYPES[logits.dtype], st), what)
    return best, rows, tokens


def _rows_of(what: str, t: torch.Tensor, n: int) -> Tuple[int, int, int]:
    """(address, bytes between rows, bytes of a row) of a tensor of ``n`` dense rows."""
    shape = t.shape
    if len(shape) == 0 or shape[0] != n or not (t.is_contiguous() or n == 0 or t[0].is_contiguous()):
        raise ValueError(f"{what}: every tensor has {n} rows, each of them dense")
    size = t.element_size()
    return t.data_ptr(), t.stride()[0] * size, t.numel() // n * size if n else 0


def reorder_rows(tensors: Sequence[torch.Tensor], rows: torch.Tensor, *, out: Optional[Sequence[torch.Tensor]] = None, status: Optional[torch.Tensor] = None) -> List[torch.Tensor]:
    """``out[t][i] = tensors[t][rows[i]]`` for all tensors (any type, rows dense) in one launch per sixteen of them; ``rows`` is int32,
    one- or two-dimensional (the columns of ``beam_select``'s that go on), and may name a row several times.  ``out`` must not share
    memory with ``tensors``: keep two sets and change places.  A row that does not exist is left as it was and latches ``BAD_PAGE``."""
    what = "reorder_rows"
    if rows.dtype != torch.int32 or rows.dim() not in (1, 2):
        raise ValueError(f"{what}: rows is int32 with one or two dimensions")
    n = rows.numel()
    if not tensors:
        return []
    n_in = tensors[0].shape[0] if tensors[0].dim() else 0
    if out is None:
        out = [t.new_empty((n, *t.shape[1:])) for t in tensors]
    if len(out) != len(tensors):
        raise ValueError(f"{what}: one out for every tensor")
    check_status(what, status)
    moves, spans = [], []
    for t, o in zip(tensors, out):
        src, src_row, size = _rows_of(what, t, n_in)
        dst, dst_row, out_size = _rows_of(what, o, n)
        if o.dtype != t.dtype or o.shape[1:] != t.shape[1:]:
            raise ValueError(f"{what}: out has the tensors' types and rows")
        if out_size:
            moves.append((src, dst, src_row, dst_row, out_size))
            spans += ((dst, dst + (n - 1) * dst_row + out_size, 1), (src, src + max(n_in - 1, 0) * src_row + size, 0))
    device = same_cuda_device(what, *tensors, *out, rows, status)
    ends = [0, 0]
    for first, end, side in sorted(spans):
        if first < ends[1 - side]:
            raise ValueError(f"{what}: out shares memory with the tensors")
        ends[side] = max(ends[side], end)
    cols = max(1, rows.shape[1]) if rows.dim() == 2 else 1
    r0, r1 = rows.stride() if rows.dim() == 2 else (rows.stride()[0], 0)
    for i in range(0, len(moves), _TENSORS):
        part = moves[i : i + _TENSORS]
        pointers = ctypes.c_void_p * len(part)
        ins, outs, meta = pointers(*[m[0] for m in part]), pointers(*[m[1] for m in part]), longs(*[x for m in part for x in m[2:]])
        on_device(device, lambda st: lib().nexrt_reorder_rows(ins, outs, meta, len(part), rows.data_ptr(), r0, r1, cols, n, n_in, ptr(status), st), what)
    return list(out)
