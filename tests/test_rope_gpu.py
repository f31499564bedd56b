"""Rotary positions against the formula in 64 bits: layouts, odd sizes, strides, far positions, padding and bad pages."""

import math

import pytest
import torch

from nexrt_b200.ops.rope import rope, rope_append, rope_frequencies
from nexrt_b200.runtime.control import Status

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def formula(x, pos, inv, interleaved=False, scale=1.0, norm=None, eps=1e-6):
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    n = 2 * inv.numel()
    ang = (pos.double()[:, None] * inv.double())[:, None]
    c, s = ang.cos() * scale, ang.sin() * scale
    y = x.clone()
    a, b = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def near(got, want, scale=1.0):
    # the result's own rounding (fp16: half a subnormal step, 2^-25, at least); before it about 16 roundings of 32 bits on values up to |a| + |b|: at most 2^-19 of the row's largest
    room = HALF_STEP[got.dtype] * want.abs() + 2.0**-25 + 2.0**-19 * want.abs().amax(-1, keepdim=True) * max(1.0, scale)
    assert torch.all((got.double() - want).abs() <= room * 1.0001), ((got.double() - want).abs() / room).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,rotary,interleaved", [(1, 1, 8, 8, False), (3, 5, 64, 64, True), (7, 3, 128, 20, False), (2, 9, 256, 64, False), (5, 2, 256, 256, True),
                                                                (4, 1, 72, 36, True), (1, 40, 200, 2, False), (130, 2, 96, 0, False), (1500, 2, 64, 30, False)])
def test_rope_alone(dtype, tokens, heads, dim, rotary, interleaved):
    g = torch.Generator(device=DEV).manual_seed(tokens + dim)
    x = torch.randn(tokens, heads, dim, device=DEV, generator=g).to(dtype)
    pos = torch.randint(-5, 300000, (tokens,), device=DEV, generator=g, dtype=torch.int32)
    inv = rope_frequencies(rotary, 1e4)[0].to(DEV) if rotary else torch.zeros(0, device=DEV)
    w = 1 + 0.1 * torch.randn(dim, device=DEV, generator=g)
    near(rope(x, pos, inv, interleaved=interleaved), formula(x, pos, inv, interleaved))
    near(rope(x, pos, inv, interleaved=interleaved, scale=1.3, norm=w), formula(x, pos, inv, interleaved, 1.3, w), 1.3)
    want = formula(x, pos, inv, interleaved)
    near(rope(x, pos, inv, interleaved=interleaved, out=x), want)                  # in place


def test_far_positions_keep_their_angle():
    """At position 2^31 - 1 a 32-bit product would be hundreds of radians off."""
    inv = torch.tensor([1.0, 0.7312345, 1e-3, 1e-7], device=DEV)
    pos = torch.tensor([2**31 - 1, 262143, 16777217, 0, -7], dtype=torch.int32, device=DEV)
    x = torch.ones(5, 1, 8, device=DEV)
    near(rope(x, pos, inv), formula(x, pos, inv))
    assert torch.equal(rope(x, pos, inv)[3], x[3])


def test_strided_and_unaligned_views():
    g = torch.Generator(device=DEV).manual_seed(5)
    flat = torch.randn(6 * 1001 + 7, device=DEV, generator=g).to(torch.bfloat16)
    x = flat[3 : 3 + 6 * 1001].view(6, 1001)[:, 1:769].unflatten(1, (6, 128))[:, ::2]      # odd start, odd row stride, every second head
    pos = torch.arange(6, dtype=torch.int32, device=DEV)
    inv = rope_frequencies(64, 1e4)[0].to(DEV)
    near(rope(x, pos, inv), formula(x, pos, inv))


@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
@pytest.mark.parametrize("hq,hk,dim,rotary,page,interleaved", [(4, 1, 256, 64, 64, False), (8, 8, 64, 64, 7, True), (3, 1, 128, 50, 1, False), (32, 2, 256, 64, 300, False)])
def test_append(src, dst, hq, hk, dim, rotary, page, interleaved):
    g = torch.Generator(device=DEV).manual_seed(hq * dim + page)
    rows, width, pages = 4, 9, 40
    table = torch.randperm(pages, device=DEV, generator=g)[: rows * width].view(rows, width).to(torch.int32)
    spots = torch.randperm(rows * width * page, device=DEV, generator=g)[:25]
    row, pos = (spots // (width * page)).to(torch.int32), (spots % (width * page)).to(torch.int32)
    row[3] = -1                                                                    # padding: rotated, not stored
    qkv = torch.randn(25, hq + 2 * hk, dim, device=DEV, generator=g).to(src)
    q, k, v = qkv[:, :hq], qkv[:, hq : hq + hk], qkv[:, hq + hk :]
    kv = torch.randn(2, pages, hk, page, dim, device=DEV, generator=g).to(dst)
    inv = rope_frequencies(rotary, 1e6)[0].to(DEV)
    qn, kn = 1 + 0.2 * torch.randn(dim, device=DEV, generator=g), 1 + 0.2 * torch.randn(dim, device=DEV, generator=g)
    before, status = kv.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    out = rope_append(q, k, v, pos, row, kv[0], kv[1], table, inv, interleaved=interleaved, q_norm=qn, k_norm=kn, status=status)
    assert int(status) == 0 and out.dtype == dst
    near(out, formula(q, pos, inv, interleaved, norm=qn))
    wk, wv = formula(k, pos, inv, interleaved, norm=kn), v.double()
    written = torch.zeros(2, pages, page, dtype=torch.bool, device=DEV)
    for i in range(25):
        if i != 3:
            p, s = int(table[row[i], pos[i] // page]), int(pos[i]) % page
            near(kv[0, p, :, s], wk[i])
            near(kv[1, p, :, s], wv[i])
            written[:, p, s] = True
    keep = ~written[:, :, None, :, None].expand_as(kv)
    assert torch.equal(kv[keep], before[keep])                                     # all else is as it was


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [16, 48, 80, 96, 112, 144, 192, 240])
def test_all_dims_turned_of_heads_that_fill_no_power_of_two(dtype, dim):
    test_rope_alone(dtype, 67, 5, dim, dim, False)
    test_rope_alone(dtype, 3, 2, dim, dim, True)
    if dtype != torch.float32:
        test_append(dtype, dtype, 6, 2, dim, dim, 5, False)
        test_append(torch.float32, dtype, 1, 3, dim, dim, 16, False)


def test_append_leaves_out_what_has_no_page():
    table = torch.tensor([[2, -1, 9, 1]], dtype=torch.int32, device=DEV)           # no page, a page that the pool does not have
    kv = torch.zeros(2, 3, 1, 4, 64, dtype=torch.bfloat16, device=DEV)
    x = torch.ones(6, 1, 64, dtype=torch.bfloat16, device=DEV)
    inv = torch.zeros(4, device=DEV)
    run = lambda pos, row: (rope_append(x[: len(pos)], x[: len(pos)], x[: len(pos)], torch.tensor(pos, dtype=torch.int32, device=DEV),  # noqa: E731
                                        torch.tensor(row, dtype=torch.int32, device=DEV), kv[0], kv[1], table, inv, status=status))
    for pos, row in (([5], [0]), ([8], [0]), ([16], [0]), ([-1], [0]), ([0], [1]), ([5, 1, 8, -3, 99, 14], [0, 0, 0, 0, 0, 0])):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        run(pos, row)
        assert int(status) == Status.BAD_PAGE
    assert float(kv[0].float().sum()) == 128.0 and float(kv[0, 2, 0, 1].float().sum()) == 64.0 and float(kv[0, 1, 0, 2].float().sum()) == 64.0
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    run([], [])
    run([0], [-5])
    assert int(status) == 0


def test_pool_strides_and_offsets_beyond_32_bits():
    """A window of a wider pool whose last page starts beyond 2^32 bytes."""
    pages, page = 70, 65536
    wide = torch.empty(pages, 1, page, 2, 256, dtype=torch.bfloat16, device=DEV)
    kp, vp = wide[:, :, :, 0], wide[:, :, :, 1]
    wide[69].zero_()
    table = torch.tensor([[0, 69]], dtype=torch.int32, device=DEV)
    x = torch.randn(1, 1, 256, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    pos, row, inv = torch.tensor([2 * page - 1], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), rope_frequencies(64, 1e7)[0].to(DEV)
    rope_append(x, x, x, pos, row, kp, vp, table, inv)
    near(kp[69, :, page - 1], formula(x, pos, inv)[0])
    assert torch.equal(vp[69, :, page - 1], x[0]) and float(wide[69, :, : page - 1].float().abs().sum()) == 0.0


@pytest.mark.parametrize("shape", [(0, 4), (3, 0), (0, 0)])
def test_append_with_a_table_without_entries(shape):
    """Padding is rotated as ever; a token that names a row has no page."""
    kv = torch.zeros(2, 3, 1, 4, 64, dtype=torch.bfloat16, device=DEV)
    x = torch.randn(2, 1, 64, device=DEV).to(torch.bfloat16)
    pos, inv = torch.tensor([0, 3], dtype=torch.int32, device=DEV), rope_frequencies(16, 1e4)[0].to(DEV)
    table = torch.zeros(*shape, dtype=torch.int32, device=DEV)
    for rows, code in (([-1, -1], 0), ([0, -1], Status.BAD_PAGE)):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = rope_append(x, x, x, pos, torch.tensor(rows, dtype=torch.int32, device=DEV), kv[0], kv[1], table, inv, status=status)
        near(out, formula(x, pos, inv))
        assert int(status) == code and not kv.any()
    none = torch.zeros(2, 0, 1, 4, 64, dtype=torch.bfloat16, device=DEV)          # and so has one of a pool without pages
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    near(rope_append(x, x, x, pos, pos * 0, none[0], none[1], torch.zeros(1, 2, dtype=torch.int32, device=DEV), inv, status=status), formula(x, pos, inv))
    assert int(status) == Status.BAD_PAGE
