"""Rotary positions (``csrc/rope.cu``): rows of q and k heads normalised and rotated, k and v stored into the pages of their
sequences, in one launch.  The decode kernels of the engine rotate in their own prologue (half layout, unscaled, one sequence);
these entry points are for batches over a paged cache (``ops/paged.py``) and for models with another layout or scaling.

Pair ``i`` of a head at position ``p`` turns by ``p * inv_freq[i]``; ``scale`` multiplies cos and sin.  The angle is formed in
64 bits, so far positions lose nothing.  For inference: tensors that require a gradient are refused, unless gradients are off.
"""

from __future__ import annotations

import math
import struct
from typing import Optional, Tuple

import torch

from .lib import address, check_status, inference_only, load as lib, on_device, same_cuda_device

I32, F32 = torch.int32, torch.float32
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_DIM = 256
_POOL_TYPES = (torch.bfloat16, torch.float16)


def rope_frequencies(rotary: int, theta: float, scaling: Optional[str] = None, factor: float = 1.0, trained: int = 0, fast: float = 32.0,
                     slow: float = 1.0) -> Tuple[torch.Tensor, float]:
    """``(inv_freq [rotary / 2] fp32 on the CPU, scale)`` for a model trained on ``trained`` positions and used on ``factor`` times as many.

    ``scaling``: ``None``; ``"linear"`` - all positions divided by the factor; ``"base"`` - theta raised so that the slowest pair is
    divided by the factor; ``"ramp"`` - pairs that turn ``fast`` times or more over the trained positions are left, those that turn less
    than ``slow`` times are divided by the factor, with a linear ramp between, and cos and sin grow by 0.1 ln(factor) + 1."""
    if rotary < 2 or rotary % 2 or not theta > 1.0 or not math.isfinite(theta):
        raise ValueError("rope_frequencies: rotary is even and positive, theta finite and above 1")
    if scaling not in (None, "linear", "base", "ramp") or not factor >= 1.0 or not math.isfinite(factor):
        raise ValueError("rope_frequencies: scaling is None, 'linear', 'base' or 'ramp', with a factor of 1 or more")
    n = rotary // 2
    if scaling == "base":
        theta = theta * factor ** (rotary / (rotary - 2)) if rotary > 2 else theta
    inv = [theta ** (-2.0 * i / rotary) for i in range(n)]
    scale = 1.0
    if scaling == "linear":
        inv = [f / factor for f in inv]
    elif scaling == "ramp":
        if trained < 1 or not fast > slow > 0:
            raise ValueError("rope_frequencies: 'ramp' needs the trained positions and fast > slow > 0")
        at = lambda turns: rotary * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary - 1)
        keep = [1.0 - min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(n)]
        inv = [f / factor * (1.0 - m) + f * m for f, m in zip(inv, keep)]
        scale = 0.1 * math.log(factor) + 1.0
    return torch.tensor(inv, dtype=torch.float32), scale


_ARGS = struct.Struct("Q13P12q12i2f")      # NexrtRopeArgs


def _common(what, q, positions, inv_freq, norms):
    """(tokens, heads, dim, rotary, strides of q)."""
    shape, strides = q.shape, q.stride()
    if len(shape) != 3 or q.dtype not in TYPES or strides[2] != 1:
        raise ValueError(f"{what}: q is [tokens, heads, dim] in bf16, fp16 or fp32 with a contiguous last dimension")
    tokens, heads, dim = shape
    if dim < 8 or dim > MAX_DIM or dim % 8:
        raise ValueError(f"{what}: head dimensions are multiples of 8 up to {MAX_DIM}, not {dim}")
    if positions.dtype is not I32 or positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError(f"{what}: positions is int32 [tokens]")
    rotary = 2 * inv_freq.numel()
    if inv_freq.dtype is not F32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or rotary > dim:
        raise ValueError(f"{what}: inv_freq is fp32 [rotary / 2] with rotary at most the head dimension")
    for w in norms:
        if w is not None and (w.dtype is not F32 or w.shape != (dim,) or not w.is_contiguous()):
            raise ValueError(f"{what}: norm multipliers are fp32 [dim]")
    return tokens, heads, dim, rotary, strides


def _out(what, out, q, tokens, heads, dim, kind):
    """``out``, or a new one, and its strides."""
    if out is None:
        return q.new_empty(tokens, heads, dim) if q.dtype is kind else q.new_empty(tokens, heads, dim, dtype=kind), (heads * dim, dim)
    strides = out.stride()
    if out.shape != (tokens, heads, dim) or out.dtype is not kind or strides[2] != 1 or (strides[0] == 0 and tokens > 1) or (strides[1] == 0 and heads > 1):
        raise ValueError(f"{what}: out is [tokens, heads, dim] of {kind} with a contiguous last dimension, each head in a place of its own")
    return out, strides


def rope(q: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0, norm: Optional[torch.Tensor] = None,
         eps: float = 1e-6, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``q [tokens, heads, dim]`` at ``positions`` int32 ``[tokens]``, rotated (after an RMSNorm with the multiplier ``norm``, if given); ``out`` may be ``q``."""
    tokens, heads, dim, rotary, q_s = _common("rope", q, positions, inv_freq, (norm,))
    inference_only("rope", q, inv_freq, norm, out)
    out, o_s = _out("rope", out, q, tokens, heads, dim, q.dtype)
    device = same_cuda_device("rope", {q.get_device(), positions.get_device(), inv_freq.get_device(), out.get_device()}, norm)
    if tokens and heads:
        kind = TYPES[q.dtype]
        on_device(device, lib().nexrt_rope_append, _ARGS.pack(
            _ARGS.size, q.data_ptr(), 0, 0, positions.data_ptr(), 0, out.data_ptr(), 0, 0, 0, inv_freq.data_ptr(), address(norm), 0, 0,
            q_s[0], q_s[1], 0, 0, 0, 0, o_s[0], o_s[1], 0, 0, 0, 0,
            tokens, heads, 0, dim, rotary, interleaved, 0, 0, 1, 0, kind, kind, scale, eps), "rope")
    return out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                table: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0, q_norm: Optional[torch.Tensor] = None,
                k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """New tokens of a paged cache: q and k ``[tokens, heads, dim]`` are normalised (``q_norm``, ``k_norm``: fp32 ``[dim]``) and rotated
    to ``positions`` int32 ``[tokens]``; k and v go to the slot of that position in row ``rows[i]`` of ``table`` (``ops/paged.py``), the
    rotated q is returned in the pages' type.  q, k and v may be views of one projection's output, in the pages' type or in fp32.

    A negative ``rows[i]`` is padding: its q is rotated, nothing is stored.  A position whose page the table does not name is left out
    and latches ``BAD_PAGE`` in ``status``.  Two tokens of a call with the same slot leave it undefined."""
    what = "rope_append"
    tokens, hq, dim, rotary, q_s = _common(what, q, positions, inv_freq, (q_norm, k_norm))
    kind, pool_kind = q.dtype, k_pages.dtype
    k_shape, k_s, v_s = k.shape, k.stride(), v.stride()
    if len(k_shape) != 3 or k_shape != v.shape or k_shape[0] != tokens or k_shape[2] != dim or k.dtype is not kind or v.dtype is not kind or k_s[2] != 1 or v_s[2] != 1:
        raise ValueError(f"{what}: k and v are [tokens, kv heads, dim] like q, with contiguous last dimensions")
    if rows.dtype is not I32 or rows.shape != (tokens,) or not rows.is_contiguous():
        raise ValueError(f"{what}: rows is int32 [tokens]")
    pool, pool_s = k_pages.shape, k_pages.stride()
    if len(pool) != 4 or pool != v_pages.shape or pool_s != v_pages.stride() or v_pages.dtype is not pool_kind or pool_s[3] != 1:
        raise ValueError(f"{what}: k_pages and v_pages are [pages, kv heads, slots, dim] with the same strides and a contiguous last dimension")
    pages, hk, slots, pool_dim = pool
    if k_shape[1] != hk or pool_dim != dim or slots < 1:
        raise ValueError(f"{what}: the pages have other heads than k")
    if pool_kind not in _POOL_TYPES or (kind is not pool_kind and kind is not F32):
        raise ValueError(f"{what}: pages are bf16 or fp16, q, k and v the same or fp32")
    t_shape, t_s = table.shape, table.stride()
    if table.dtype is not I32 or len(t_shape) != 2 or t_s[1] != 1:
        raise ValueError(f"{what}: table is int32 [rows, pages of a row] with contiguous rows")
    check_status(what, status)
    inference_only(what, q, k, v, k_pages, v_pages, inv_freq, q_norm, k_norm, out)
    out, o_s = _out(what, out, q, tokens, hq, dim, pool_kind)
    device = same_cuda_device(what, {q.get_device(), k.get_device(), v.get_device(), positions.get_device(), rows.get_device(), k_pages.get_device(), v_pages.get_device(),
                                     table.get_device(), inv_freq.get_device(), out.get_device()}, q_norm, k_norm, status)
    if tokens:
        on_device(device, lib().nexrt_rope_append, _ARGS.pack(
            _ARGS.size, q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr(), rows.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            table.data_ptr(), inv_freq.data_ptr(), address(q_norm), address(k_norm), address(status),
            q_s[0], q_s[1], k_s[0], k_s[1], v_s[0], v_s[1], o_s[0], o_s[1], pool_s[0], pool_s[1], pool_s[2], t_s[0],
            tokens, hq, hk, dim, rotary, interleaved, t_shape[0], t_shape[1], slots, pages, TYPES[kind], TYPES[pool_kind], scale, eps), what)
    return out
