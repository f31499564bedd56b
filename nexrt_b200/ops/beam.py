"""Beam search: selection over beams and vocabulary, and reordering of what belongs to a beam (``csrc/beam.cu``).

The engine's head samples one sequence (``head.py``); these entry points rank the continuations of several beams of several
requests.  The rows that ``beam_select`` returns go to ``ops.paged.fork_pages`` (pages of the cache) and to ``reorder_rows``
(recurrent states, conv histories, whatever has one row per beam).  For inference: tensors that require a gradient are refused, unless
gradients are off.
"""

from __future__ import annotations

import struct
from typing import List, Optional, Sequence, Tuple

import torch

from .lib import address, check_status, inference_only, load as lib, on_device, same_cuda_device
from .rope import F32, I32, TYPES

MAX_K = 64
MAX_BEAMS = 256
MAX_VOCAB = 1 << 24
_TENSORS = 16                                   # of one launch of the reorder kernel
_BEAM = struct.Struct("Q8P6q8i")                # NexrtBeamArgs
_REORDER = struct.Struct("Q2P2q6i32P48q")       # NexrtReorderArgs
_BOOL = torch.bool


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, *, finished: Optional[torch.Tensor] = None, eos: int = -1,
                status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``k`` (at most 64) best continuations of every request: ``logits [requests, beams, vocabulary]`` (bf16, fp16 or fp32),
    ``scores`` fp32 ``[requests, beams]``, the beams' log-probabilities so far (-inf: a beam that does not exist).  Returns, best first,
    ``(scores fp32, rows int32, tokens int32)``, each ``[requests, k]``; ``rows`` counts beams over all requests (request * beams + beam).

    The total of a candidate is the beam's score plus the logit's log-softmax, added in 64 bits; equal totals go to the lower beam, then
    to the larger logit, then to the lower token.  A row's log of the sum of exp comes from 32-bit exponentials and is off by 1e-7 as a
    rule, at worst by a few 1e-6: candidates of different beams that are nearer than that may change places; beams with the same logits and the
    same score always tie.  A beam marked in ``finished`` (bool ``[requests, beams]``) has one candidate, token
    ``eos`` at its own score.  Where fewer than ``k`` candidates are above -inf the rest are at -inf.  A beam with a NaN or +inf among its
    logits, or as its score, has no candidate and latches ``NON_FINITE`` in ``status``."""
    what = "beam_select"
    shape, l_s, kind = logits.shape, logits.stride(), logits.dtype
    if len(shape) != 3 or kind not in TYPES or (shape[2] > 1 and l_s[2] != 1):
        raise ValueError(f"{what}: logits is [requests, beams, vocabulary] in bf16, fp16 or fp32 with a contiguous last dimension")
    batch, beams, vocab = shape
    if not 1 <= beams <= MAX_BEAMS or not 1 <= vocab <= MAX_VOCAB or batch * beams > 65535:
        raise ValueError(f"{what}: at most {MAX_BEAMS} beams, 65535 in all, and a vocabulary of {MAX_VOCAB}")
    if not 1 <= k <= min(MAX_K, beams * vocab):
        raise ValueError(f"{what}: k is between 1 and {MAX_K} and no more than there are candidates")
    if scores.dtype is not F32 or scores.shape != (batch, beams):
        raise ValueError(f"{what}: scores is fp32 [requests, beams]")
    s_s, f_s = scores.stride(), (0, 0)
    if finished is not None:
        if finished.dtype is not _BOOL or finished.shape != (batch, beams) or not 0 <= eos < vocab:
            raise ValueError(f"{what}: finished is bool [requests, beams], with an end token of the vocabulary")
        f_s = finished.stride()
    check_status(what, status)
    inference_only(what, logits, scores)
    device = same_cuda_device(what, {logits.get_device(), scores.get_device()}, finished, status)
    best, rows, tokens = scores.new_empty(batch, k), scores.new_empty(batch, k, dtype=I32), scores.new_empty(batch, k, dtype=I32)
    if batch:
        L = lib()
        slices = L.nexrt_beam_slices(batch * beams, beams, vocab, k, TYPES[kind])
        scratch = scores.new_empty(batch * beams * slices * (k + 2), dtype=torch.int64)
        on_device(device, L.nexrt_beam_select, _BEAM.pack(
            _BEAM.size, logits.data_ptr(), scores.data_ptr(), address(finished), best.data_ptr(), rows.data_ptr(), tokens.data_ptr(), scratch.data_ptr(), address(status),
            l_s[0], l_s[1], s_s[0], s_s[1], f_s[0], f_s[1], batch, beams, vocab, k, eos, TYPES[kind], slices, 0), what)
    return best, rows, tokens


def _row_stride(what: str, t: torch.Tensor) -> int:
    """Bytes between the rows of a tensor that is not contiguous, but whose rows are."""
    if not t[0].is_contiguous():
        raise ValueError(f"{what}: rows are dense")
    return t.stride()[0] * t.element_size()


def reorder_rows(tensors: Sequence[torch.Tensor], rows: torch.Tensor, *, out: Optional[Sequence[torch.Tensor]] = None, status: Optional[torch.Tensor] = None) -> List[torch.Tensor]:
    """``out[t][i] = tensors[t][rows[i]]`` for all tensors (any type, rows dense) in one launch per sixteen of them; ``rows`` is int32,
    one- or two-dimensional (the columns of ``beam_select``'s that go on), and may name a row several times.  ``out`` must not share
    memory with ``tensors``: keep two sets and change places.  A row that does not exist is left as it was, zeros where ``out`` is not given,
    and latches ``BAD_PAGE``."""
    what = "reorder_rows"
    r_shape, r_s = rows.shape, rows.stride()
    if rows.dtype is not I32 or len(r_shape) not in (1, 2):
        raise ValueError(f"{what}: rows is int32 with one or two dimensions")
    n = rows.numel()
    if not tensors:
        return []
    n_in = tensors[0].shape[0] if tensors[0].dim() else 0
    clear = out is None
    if clear:
        out = [t.new_empty((n, *t.shape[1:])) for t in tensors]
    if len(out) != len(tensors):
        raise ValueError(f"{what}: one out for every tensor")
    check_status(what, status)
    inference_only(what, *tensors, *out)
    moves, spans = [], []
    for t, o in zip(tensors, out):
        t_shape, o_shape = t.shape, o.shape
        if len(t_shape) == 0 or len(o_shape) == 0 or t_shape[0] != n_in or o_shape[0] != n or (t_shape != o_shape and t_shape[1:] != o_shape[1:]) or o.dtype is not t.dtype:
            raise ValueError(f"{what}: tensors have the same number of rows, and out the same rows of the same types")
        values = o.numel()
        if values:
            size = values // n * o.element_size()
            src, dst, src_row, dst_row = t.data_ptr(), o.data_ptr(), size, size
            if not o.is_contiguous():
                dst_row = _row_stride(what, o)
                if n > 1 and dst_row < size:
                    raise ValueError(f"{what}: rows of out lie over one another")
            if n_in and not t.is_contiguous():
                src_row = _row_stride(what, t)
            moves.append((src, dst, src_row, dst_row, size))
            spans.append((dst, dst + (n - 1) * dst_row + size, 1))
            spans.append((src, src + (n_in - 1) * src_row + size, 0))
    device = same_cuda_device(what, {rows.get_device()}, *tensors, *out, status)
    ends = [0, 0]
    spans.sort()
    for first, end, side in spans:
        if first < ends[1 - side]:
            raise ValueError(f"{what}: out shares memory with the tensors")
        if end > ends[side]:
            ends[side] = end
    cols, r0, r1 = (max(1, r_shape[1]), r_s[0], r_s[1]) if len(r_shape) == 2 else (1, r_s[0], 0)
    for i in range(0, len(moves), _TENSORS):
        part = moves[i : i + _TENSORS]
        none = [0] * (_TENSORS - len(part))
        columns = []
        for column in zip(*part):
            columns += [*column, *none]
        on_device(device, lib().nexrt_reorder_rows, _REORDER.pack(_REORDER.size, rows.data_ptr(), address(status), r0, r1, cols, n, n_in, len(part), clear, 0, *columns), what)
    return list(out)
