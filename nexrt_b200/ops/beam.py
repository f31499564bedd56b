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
    best = torch.empty(batch, k, dtype=torch.float32, device=device)
    rows = torch.empty(batch, k, dtype=torch.int32, device=device)
    tokens = torch.empty(batch, k, dtype=torch.int32, device=device)
    if batch:
        L = lib()
        scratch = torch.empty(batch * beams * L.nexrt_beam_slices(vocab) * (k + 2), dtype=torch.int64, device=device)
        strides = longs(logits.stride(0), logits.stride(1), *scores.stride(), *(finished.stride() if finished is not None else (0, 0)))
        on_device(device, lambda st: L.nexrt_beam_select(ptr(logits), ptr(scores), ptr(finished), strides, ptr(best), ptr(rows), ptr(tokens), ptr(scratch), ptr(status), batch,
                                                         beams, vocab, k, eos, TYPES[logits.dtype], st), what)
    return best, rows, tokens


def _row_dense(t: torch.Tensor) -> bool:
    return t.dim() > 0 and (t.shape[0] == 0 or t[0].is_contiguous())


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
    n_in = tensors[0].shape[0] if tensors[0].dim() else -1
    if any(t.dim() == 0 or t.shape[0] != n_in or not _row_dense(t) for t in tensors):
        raise ValueError(f"{what}: tensors have the same number of rows, each of them dense")
    if out is None:
        out = [torch.empty((n, *t.shape[1:]), dtype=t.dtype, device=t.device) for t in tensors]
    if len(out) != len(tensors) or any(o.dtype != t.dtype or o.shape != (n, *t.shape[1:]) or not _row_dense(o) for o, t in zip(out, tensors)):
        raise ValueError(f"{what}: out has {n} dense rows for every tensor")
    check_status(what, status)
    device = same_cuda_device(what, *tensors, *out, rows, status)
    held = {t.untyped_storage().data_ptr() for t in tensors if t.numel()}
    if any(o.numel() and o.untyped_storage().data_ptr() in held for o in out):
        raise ValueError(f"{what}: out shares memory with the tensors")
    cols, r0, r1 = (1, rows.stride(0), 0) if rows.dim() == 1 else (max(1, rows.shape[1]), rows.stride(0), rows.stride(1))
    live = [(t, o) for t, o in zip(tensors, out) if o.numel()]
    for i in range(0, len(live), _TENSORS):
        part = live[i : i + _TENSORS]
        ins, outs = ((ctypes.c_void_p * len(part))(*(p[j].data_ptr() for p in part)) for j in (0, 1))
        meta = longs(*(x for t, o in part for x in (t.stride(0) * t.element_size(), o.stride(0) * o.element_size(), t[0].numel() * t.element_size())))
        on_device(device, lambda st: lib().nexrt_reorder_rows(ins, outs, meta, len(part), ptr(rows), r0, r1, cols, n, n_in, ptr(status), st), what)
    return list(out)
