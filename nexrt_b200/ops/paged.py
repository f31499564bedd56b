"""A key-value cache in pages that several sequences share (``csrc/paged_attn.cuh``, ``csrc/pages.cu``).

The engine's own cache (``attn.py: FullAttn``) is one contiguous block for one sequence.  Here the keys and values of a batch lie
in a pool of pages: ``kv [layers, 2, pages, kv heads, slots, dim]`` (K and V of every layer), and ``table`` int32 ``[rows, width]``
names, row by row, the page of positions ``[slots * j, slots * (j + 1))``; behind a row's last page it holds -1.  ``lens`` int32
``[rows]`` are the rows' positions.  Rows may share pages (a common prompt, beams of one request); a page is free when no row
names it within its length.

Everything is planned on the device: no call waits for the host, all of them can be captured into a CUDA graph.  What a kernel
finds wrong (a page that does not exist, a full pool) is left out and latched in ``status`` (``runtime/control.py: Status``).  The calls
are for inference: they refuse tensors that require a gradient, unless gradients are off.
"""

from __future__ import annotations

import math
import struct
from typing import Optional, Tuple, Union

import torch

from ..runtime.control import Status
from .lib import KernelError, address, check_status, inference_only, load as lib, on_device, same_cuda_device, sm_count
from .rope import F32, I32, TYPES, rope_append

HEAD_DIMS = (64, 128, 192, 256)
MAX_ROWS = 4096
_CHUNK = 64                                     # keys of a unit of the attention's work, and what an item counts beside them
_ITEM_COST = 3
_ATTN = struct.Struct("Q10P9q10i2f")            # NexrtPagedAttnArgs
_PAGES = struct.Struct("Q13P2q10i")             # NexrtPagesArgs
_POOL_TYPES = (torch.bfloat16, torch.float16)


def _resident(dim: int) -> int:
    """CTAs of the attention kernel on an SM."""
    return 3 if dim == 64 else 2


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *, scale: Optional[float] = None,
                    softcap: float = 0.0, window: int = 0, slopes: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    status: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """One new token of every sequence over its pages: ``q [rows, heads, dim]`` against keys ``[max(0, len - window), len)`` of each row
    (``window`` 0: all), whose own key is the last of them.  ``k_pages`` / ``v_pages [pages, kv heads, slots, dim]`` are one layer's
    (``kv[layer, 0]``, ``kv[layer, 1]``), bf16 or fp16 like q; dims 64, 128, 192 or 256; heads a multiple of the kv heads.

    Scores are ``q.k * scale`` (default ``dim ** -0.5``), then ``softcap * tanh(s / softcap)`` if it is not zero, then
    ``s - slopes[head] * distance`` if ``slopes`` (fp32 ``[heads]``) is given.  A row without keys gives zeros and an lse of -inf, and so
    does one whose scores are all -inf.  Returns ``out [rows, heads, dim]``, with ``return_lse`` also fp32 ``[rows, heads]``: the natural
    logarithm of the sum of exp of the scores.  An infinite value that a row sees makes that dim of its result NaN or infinite.  Keys on a page that the table does not name count as masked and latch ``BAD_PAGE``.  A
    length beyond the table's columns is cut to them, here as in the calls below, and latches ``BAD_PAGE``: window and distances count
    from the last position that has a place.  ``out`` may be ``q``."""
    what = "paged_attention"
    kind, shape, q_s = q.dtype, q.shape, q.stride()
    if len(shape) != 3 or kind not in _POOL_TYPES or q_s[2] != 1:
        raise ValueError(f"{what}: q is [rows, heads, dim] in bf16 or fp16 with a contiguous last dimension")
    rows, heads, dim = shape
    pool, pool_s = k_pages.shape, k_pages.stride()
    if len(pool) != 4 or pool != v_pages.shape or pool_s != v_pages.stride() or pool_s[3] != 1 or k_pages.dtype is not kind or v_pages.dtype is not kind:
        raise ValueError(f"{what}: k_pages and v_pages are [pages, kv heads, slots, dim] of q's type, with the same strides and a contiguous last dimension")
    pages, kv_heads, slots, pool_dim = pool
    if dim not in HEAD_DIMS or pool_dim != dim:
        raise ValueError(f"{what}: head dimensions are {HEAD_DIMS}, those of q and of the pages the same")
    if kv_heads < 1 or slots < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{what}: {heads} heads on {kv_heads} kv heads")
    k_ptr, v_ptr = k_pages.data_ptr(), v_pages.data_ptr()
    if (pool_s[0] | pool_s[1] | pool_s[2]) % 8 or (k_ptr | v_ptr) % 16:
        raise ValueError(f"{what}: rows of the pages start on 16-byte boundaries")
    if pages * pool_s[0] + slots * pool_s[2] > 2**35 - 8:
        raise ValueError(f"{what}: one layer's keys or values take less than 64 GB")
    t_shape, t_s = table.shape, table.stride()
    if table.dtype is not I32 or len(t_shape) != 2 or t_shape[0] != rows or t_s[1] != 1:
        raise ValueError(f"{what}: table is int32 [rows, pages of a row] with contiguous rows")
    if lens.dtype is not I32 or lens.shape != (rows,) or not lens.is_contiguous():
        raise ValueError(f"{what}: lens is int32 [rows]")
    if not 0.0 <= softcap < math.inf or window < 0:
        raise ValueError(f"{what}: softcap and window are not negative")
    if slopes is not None and (slopes.dtype is not F32 or slopes.shape != (heads,) or not slopes.is_contiguous()):
        raise ValueError(f"{what}: slopes is fp32 [heads]")
    check_status(what, status)
    inference_only(what, q, k_pages, v_pages, slopes, out)
    if out is None:
        out, o_s = q.new_empty(rows, heads, dim), (heads * dim, dim)
    else:
        o_s = out.stride()
        if out.shape != shape or out.dtype is not kind or o_s[2] != 1 or (o_s[0] == 0 and rows > 1) or (o_s[1] == 0 and heads > 1):
            raise ValueError(f"{what}: out is like q, each head in a place of its own")
    lse = q.new_empty(rows, heads, dtype=F32) if return_lse else None
    device = same_cuda_device(what, {q.get_device(), k_pages.get_device(), v_pages.get_device(), table.get_device(), lens.get_device(), out.get_device()}, slopes, status)
    if rows:
        # as many CTAs as are resident, no more than there can be units of work
        width, window = t_shape[1], min(window, 2**31 - 1)
        keys = min(width * slots, window + _CHUNK) if window else width * slots
        ctas = min(_resident(dim) * sm_count(device), 1024, (keys // _CHUNK + 1 + _ITEM_COST) * rows * kv_heads * -(-heads // (16 * kv_heads)))
        scratch = q.new_empty(ctas * (32 * (dim + 2) + 4), dtype=F32)
        on_device(device, lib().nexrt_paged_attn, _ATTN.pack(
            _ATTN.size, q.data_ptr(), k_ptr, v_ptr, table.data_ptr(), lens.data_ptr(), address(slopes), out.data_ptr(), address(lse), scratch.data_ptr(), address(status),
            q_s[0], q_s[1], o_s[0], o_s[1], pool_s[0], pool_s[1], pool_s[2], t_s[0], heads,
            rows, heads, kv_heads, dim, width, slots, pages, window, TYPES[kind], ctas, dim**-0.5 if scale is None else scale, softcap), what)
    return (out, lse) if return_lse else out


def _pool(what: str, kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor):
    """Base of the pool; planes, pages, heads, slots, bytes of a slot, rows and width of the table; its row stride."""
    inference_only(what, kv)
    shape = kv.shape
    if len(shape) != 6 or shape[1] != 2 or not kv.is_contiguous():
        raise ValueError(f"{what}: kv is a contiguous [layers, 2, pages, kv heads, slots, dim]")
    base, slot = kv.data_ptr(), shape[5] * kv.element_size()
    if shape[3] < 1 or shape[4] < 1 or slot < 16 or slot % 16 or base % 16:
        raise ValueError(f"{what}: a slot of the pool takes a multiple of 16 bytes and starts on such a boundary")
    t_shape, t_s = table.shape, table.stride()
    if table.dtype is not I32 or len(t_shape) != 2 or t_s[1] != 1:
        raise ValueError(f"{what}: table is int32 [rows, pages of a row] with contiguous rows")
    if lens.dtype is not I32 or lens.shape != (t_shape[0],) or not lens.is_contiguous():
        raise ValueError(f"{what}: lens is int32 [rows]")
    return base, (2 * shape[0], shape[2], shape[3], shape[4], slot, t_shape[0], t_shape[1]), t_s[0]


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First byte and the one behind the last of an int32 list or table with contiguous rows."""
    first, shape = t.data_ptr(), t.shape
    if not t.numel():
        return 0, 0
    return first, first + 4 * (shape[0] if len(shape) == 1 else (shape[0] - 1) * t.stride()[0] + shape[1])


def _fresh(what: str, name: str, t: Optional[torch.Tensor], shape, like: torch.Tensor, *old: Optional[torch.Tensor]) -> torch.Tensor:
    if t is None:
        return like.new_empty(*shape)        # (ints cost half of what a tuple does)
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or (t.numel() and t.stride(-1) != 1) or (t.dim() == 1 and not t.is_contiguous()):
        raise ValueError(f"{what}: {name} is int32 {list(shape)} with contiguous rows")
    if t.dim() == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: rows of {name} lie over one another")
    begin, end = _span(t)
    for o in old:
        if o is not None and end:
            first, last = _span(o)
            if begin < last and first < end:
                raise ValueError(f"{what}: {name} shares memory with another argument: the rows are read while it is written")
    return t


def fork_pages(kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, grow: Union[int, torch.Tensor] = 0, *, table_out: Optional[torch.Tensor] = None,
               lens_out: Optional[torch.Tensor] = None, refs: Optional[torch.Tensor] = None, grown: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Row ``r`` of the new table goes on with row ``parents[r]`` of the old one (int32, at most 4096; -1: the row is empty) and gets
    room for ``grow`` more positions (an int for all rows, or int32 ``[rows]``): ``(table, lens + grow, refs)``, where ``refs`` int32
    ``[pages]`` says how many rows name a page.  Rows that nobody continues are freed with what they alone held.

    Full pages are shared.  A begun page that a growing row shares with others is copied, its written positions in all layers;
    where all its holders grow, the lowest row keeps it.  New pages are the lowest free ones, in the order of the rows.  A row for
    which there is no page, or no column in the table, keeps its length and latches ``NO_PAGES``; a page or parent that does not
    exist latches ``BAD_PAGE``, and so does a length beyond the table's columns, which is cut to them.  Where a row finds no page, the rows
    behind it that want one find none either.  The outputs must not share memory with the inputs.

    The last position of a row that did not grow may lie on a page that other rows read: nothing is to be stored there.  ``grown`` int32
    ``[rows]`` gets the row's number where the row grew and -1 elsewhere, which is what ``rope_append`` takes as ``rows``."""
    what = "fork_pages"
    base, sizes, row = _pool(what, kv, table, lens)
    n, width, pages = parents.numel(), sizes[6], sizes[1]
    if parents.dtype is not I32 or parents.dim() != 1 or not parents.is_contiguous() or n > MAX_ROWS:
        raise ValueError(f"{what}: parents is int32 [rows], at most {MAX_ROWS}")
    each = grow if isinstance(grow, torch.Tensor) else None
    if each is not None and (each.dtype is not I32 or each.shape != (n,) or not each.is_contiguous()):
        raise ValueError(f"{what}: grow is an int or int32 [rows]")
    if each is None and not 0 <= grow < 2**31:
        raise ValueError(f"{what}: grow is not negative")
    check_status(what, status)
    table_out = _fresh(what, "table_out", table_out, (n, width), table, table, lens, parents, each)
    lens_out = _fresh(what, "lens_out", lens_out, (n,), table, table, lens, parents, each, table_out)
    refs = _fresh(what, "refs", refs, (pages,), table, table, lens, parents, each, table_out, lens_out)
    if grown is not None:
        _fresh(what, "grown", grown, (n,), table, table, lens, parents, each, table_out, lens_out, refs)
    device = same_cuda_device(what, {kv.get_device(), table.get_device(), lens.get_device(), parents.get_device(), table_out.get_device(), lens_out.get_device(),
                                     refs.get_device()}, each, grown, status)
    scratch = table.new_empty(3 * pages + 3 * n + 1)
    on_device(device, lib().nexrt_page_fork, _PAGES.pack(
        _PAGES.size, base, table.data_ptr(), lens.data_ptr(), parents.data_ptr(), address(each), table_out.data_ptr(), lens_out.data_ptr(), refs.data_ptr(), 0, 0,
        scratch.data_ptr(), address(status), address(grown), row, table_out.stride()[0], *sizes, n, 0 if each is not None else grow, 0), what)
    return table_out, lens_out, refs


def compact_pages(kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *, table_out: Optional[torch.Tensor] = None, refs: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Moves the pages that rows name to the front of the pool, all layers: of ``live`` such pages those behind the first ``live``
    places go, in order, into the holes in front.  Returns ``(table, refs, remap, live)``: the renamed table, rows per page, new
    place of every page (-1: it was free) and ``live`` int32 ``[1]``.  What lies in the pool from ``live`` on is free."""
    what = "compact_pages"
    base, sizes, row = _pool(what, kv, table, lens)
    pages = sizes[1]
    check_status(what, status)
    table_out = _fresh(what, "table_out", table_out, tuple(table.shape), table, table, lens)
    refs = _fresh(what, "refs", refs, (pages,), table, lens, table, table_out)
    remap, live = table.new_empty(pages), table.new_empty(1)
    device = same_cuda_device(what, {kv.get_device(), table.get_device(), lens.get_device(), table_out.get_device(), refs.get_device()}, status)
    scratch = table.new_empty(5 * pages + 1)
    on_device(device, lib().nexrt_page_compact, _PAGES.pack(
        _PAGES.size, base, table.data_ptr(), lens.data_ptr(), 0, 0, table_out.data_ptr(), 0, refs.data_ptr(), remap.data_ptr(), live.data_ptr(), scratch.data_ptr(),
        address(status), 0, row, table_out.stride()[0], *sizes, 0, 0, 0), what)
    return table_out, refs, remap, live


def copy_pages(kv: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, *, status: Optional[torch.Tensor] = None) -> None:
    """Page ``src[i]`` to page ``dst[i]`` in all layers (int32, one list each).  A copy with a negative entry, or of a page to itself, is left out;
    one with an entry beyond the pool is too and latches ``BAD_PAGE``.  A copy to a page that is also a source is left out, of those to one
    page only the last counts (if it is left out, none); both latch ``PAGE_CONFLICT``.  Copies that are left out for an entry beyond the pool
    still count as naming their other page."""
    what = "copy_pages"
    for t in (src, dst):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.numel() != src.numel():
            raise ValueError(f"{what}: src and dst are int32 lists of the same length")
    base, sizes, _ = _pool(what, kv, src.view(-1, 1), src)
    check_status(what, status)
    device = same_cuda_device(what, {kv.get_device(), src.get_device(), dst.get_device()}, status)
    scratch = src.new_empty(3 * src.numel() + 2 * sizes[1])
    on_device(device, lib().nexrt_page_copy, _PAGES.pack(_PAGES.size, base, src.data_ptr(), dst.data_ptr(), 0, 0, 0, 0, 0, 0, 0, scratch.data_ptr(), address(status), 0, 1, 0, *sizes, 0, 0, 0), what)


class PagedCache:
    """Pool, table, lengths and status word of a batch, at fixed addresses (a captured step stays valid).

    One decode step: ``fork(parents, 1)`` - or ``fork(grow=1)`` to go on with every row -, then for every layer ``append`` with the
    positions ``lens - 1`` and the rows ``grown``, and ``attend``.  ``grown`` int32 ``[rows]`` is what the last fork left: the row's
    number where the row grew, -1 where it was freed, did not ask for room or found none, so that nothing is stored for it.  ``check()``
    waits for the device and raises what the kernels latched, once: the cache goes on with a clean status."""

    def __init__(self, layers: int, pages: int, kv_heads: int, slots: int, dim: int, rows: int, max_len: int, dtype: torch.dtype = torch.bfloat16,
                 device: Union[str, torch.device] = "cuda"):
        if min(layers, pages, kv_heads, slots, rows, max_len) < 1 or dim not in HEAD_DIMS or dtype not in (torch.bfloat16, torch.float16) or rows > MAX_ROWS:
            raise ValueError(f"PagedCache: sizes are positive, at most {MAX_ROWS} rows, head dimensions {HEAD_DIMS}, bf16 or fp16")
        i32 = dict(dtype=torch.int32, device=device)
        self.kv = torch.zeros(layers, 2, pages, kv_heads, slots, dim, dtype=dtype, device=device)
        self.table = torch.full((rows, -(-max_len // slots)), -1, **i32)
        self.lens = torch.zeros(rows, **i32)
        self.refs = torch.zeros(pages, **i32)
        self.status = torch.zeros(1, **i32)
        self.same = torch.arange(rows, **i32)
        self.grown = torch.full((rows,), -1, **i32)

    def fork(self, parents: Optional[torch.Tensor] = None, grow: Union[int, torch.Tensor] = 0) -> None:
        """``fork_pages`` on the cache's own table: every row of it goes on with one of its rows, or is freed (-1)."""
        parents = self.same if parents is None else parents
        if parents.shape != self.lens.shape:
            raise ValueError("PagedCache.fork: one parent for every row of the cache")
        table, lens, _ = fork_pages(self.kv, self.table, self.lens, parents, grow, refs=self.refs, grown=self.grown, status=self.status)
        self.table.copy_(table)
        self.lens.copy_(lens)

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor, inv_freq: torch.Tensor, **how) -> torch.Tensor:
        return rope_append(q, k, v, positions, rows, self.kv[layer, 0], self.kv[layer, 1], self.table, inv_freq, status=self.status, **how)

    def load_kv(self, layer: int, row: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Install ``k, v [kv heads][positions][dim]`` (already normalised and rotated, as ``DecodeEngine.export_state`` gives them) as the first
        positions of ``row``, which has room for them (``fork`` with ``grow``).  Rows that share its pages read them too."""
        if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or not 0 <= row < self.lens.numel():
            raise ValueError("PagedCache.load_kv: k and v are [kv heads, positions, dim] for a row of the cache")
        k, v = k.transpose(0, 1), v.transpose(0, 1)
        at = torch.arange(k.shape[0], dtype=I32, device=k.device)
        self.append(layer, k[:, :0], k, v, at, torch.full_like(at, row), torch.empty(0, dtype=F32, device=k.device))

    def attend(self, layer: int, q: torch.Tensor, **how) -> torch.Tensor:
        return paged_attention(q, self.kv[layer, 0], self.kv[layer, 1], self.table, self.lens, status=self.status, **how)

    def compact(self) -> torch.Tensor:
        """Pages in use move to the front; returns their number (int32 ``[1]`` on the device)."""
        table, _, _, live = compact_pages(self.kv, self.table, self.lens, refs=self.refs, status=self.status)
        self.table.copy_(table)
        return live

    def check(self) -> None:
        code = int(self.status.item())
        if code:
            self.status.zero_()
            names = {v: k for k, v in vars(Status).items() if isinstance(v, int)}
            raise KernelError(f"paged cache: {names.get(code, code)}")
