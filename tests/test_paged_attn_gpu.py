"""Attention over a paged cache against the formula in 64 bits: lengths from nothing to long, pages of any size, head groups, strides, caps, biases and
windows, garbage in masked places, bad pages, captured graphs."""

import math

import pytest
import torch

from nexrt_b200.ops.paged import paged_attention
from nexrt_b200.runtime.capture import graph_capture
from nexrt_b200.runtime.control import Status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(lens, hq, hk, dim, page, dtype, seed=0, std=1.5, extra=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [max(0, -(-n // page)) for n in lens]
    pages, width = sum(need) + extra, max(max(need), 1) + 1
    order = torch.randperm(pages, device=DEV, generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = torch.tensor(order[at : at + c], dtype=torch.int32)
        at += c
    kv = torch.randn(2, pages, hk, page, dim, device=DEV, generator=g).to(dtype)
    q = (torch.randn(len(lens), hq, dim, device=DEV, generator=g) * std).to(dtype)
    return q, kv, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


def formula(q, kv, table, lens, scale=None, softcap=0.0, window=0, slopes=None):
    """(out, lse, room): room is how far 32-bit sums and products may be off: a score's error is at most (dim + 16) steps of 2^-23 of
    sum |q k| scale (the products' sum, the scaling, tanh and the bias in 32 bits), and a 16-bit pair holds P to 2^-16; it enters the
    result twice (numerator and sum)."""
    B, hq, dim = q.shape
    hk, page = kv.shape[2], kv.shape[3]
    per, scale = hq // hk, dim**-0.5 if scale is None else scale
    out = torch.zeros(B, hq, dim, dtype=torch.float64, device=DEV)
    lse = torch.full((B, hq), -math.inf, dtype=torch.float64, device=DEV)
    room, lroom = torch.zeros_like(out), torch.zeros_like(lse)
    for b, n in enumerate(lens.tolist()):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        pages = table[b, : -(-n // page)].long()
        for h in range(hk):
            K, V = (kv[i][pages, h].reshape(-1, dim)[lo:n].double() for i in (0, 1))
            x = q[b, h * per : (h + 1) * per].double()
            s = x @ K.T * scale
            size = (x.abs() @ K.abs().T * abs(scale)).amax(-1, keepdim=True)
            if softcap:
                s = torch.tanh(s / softcap) * softcap
            if slopes is not None:
                d = slopes[h * per : (h + 1) * per].double()[:, None] * torch.arange(n - 1 - lo, -1, -1, device=DEV)
                s, size = s - d, size + d.amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            at = slice(h * per, (h + 1) * per)
            out[b, at], lse[b, at] = p @ V, torch.logsumexp(s, -1)
            err = (dim + 16) * 2.0**-23 * size + 2.0**-16
            room[b, at], lroom[b, at] = 2 * err * (p @ V.abs()), err[:, 0] + 2.0**-22 * lse[b, at].abs()
    return out, lse, room, lroom


def check(got, lse, want):
    out, wl, room, lroom = want
    half = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[got.dtype]
    room = half * out.abs() + room * (1 + half) + 2.0**-25
    assert torch.all((got.double() - out).abs() <= room), ((got.double() - out).abs() / room).max()
    fine = torch.isfinite(wl)
    assert torch.equal(lse[~fine].double(), wl[~fine]) and torch.all((lse[fine].double() - wl[fine]).abs() <= lroom[fine])


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 1000, 0, 5000]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,dim,page", [(4, 1, 256, 64), (32, 2, 256, 16), (9, 3, 128, 1), (8, 8, 64, 7), (20, 1, 192, 100), (64, 1, 64, 16), (17, 1, 128, 300), (2, 2, 256, 33)])
def test_lengths_groups_and_pages(dtype, hq, hk, dim, page):
    case = build(LENS, hq, hk, dim, page, dtype, seed=hq + page)
    q, kv, table, lens = case
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True, status=status)
    check(out, lse, formula(q, kv, table, lens))
    assert int(status) == 0
    again, _ = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True)
    assert torch.equal(out, again) and torch.equal(out, paged_attention(q, kv[0], kv[1], table, lens))   # the joins have an order
    assert not out[0].any() and not out[11].any()


@pytest.mark.parametrize("softcap,window,bias,scale", [(0.0, 1, False, None), (0.0, 63, False, None), (0.0, 64, True, 0.05), (20.0, 0, False, None), (30.0, 1000, True, None), (0.0, 0, True, None), (5.0, 129, False, 1.0)])
@pytest.mark.parametrize("hq,hk,dim,page", [(8, 2, 128, 24), (12, 1, 64, 16), (16, 1, 256, 64)])
def test_caps_windows_and_biases(softcap, window, bias, scale, hq, hk, dim, page):
    q, kv, table, lens = build(LENS, hq, hk, dim, page, torch.bfloat16, seed=7)
    slopes = 0.5 ** torch.arange(hq, device=DEV).float() if bias else None
    how = dict(softcap=softcap, window=window, slopes=slopes, scale=scale)
    out, lse = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True, **how)
    check(out, lse, formula(q, kv, table, lens, scale, softcap, window, slopes))


@pytest.mark.parametrize("seqs,keys", [(1, 1), (1, 100000), (3, 40000), (300, 50), (700, 3)])
def test_one_long_and_many_short(seqs, keys):
    q, kv, table, lens = build([max(0, keys - i % 5) for i in range(seqs)], 8, 2, 128, 32, torch.bfloat16, seed=seqs)
    out, lse = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True)
    check(out, lse, formula(q, kv, table, lens))


def test_masked_places_may_hold_anything():
    """Slots behind a row's end, in front of its window and on pages of nobody hold NaN and infinities."""
    lens = [5, 70, 200, 0, 1000]
    q, kv, table, lens = build(lens, 8, 1, 128, 48, torch.float16, seed=3)
    seen = torch.zeros(kv.shape[1], 48, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens.tolist()):
        for j in range(max(0, n - 60), n):
            seen[table[b, j // 48], j % 48] = True
    dirty = kv.clone()
    junk = torch.tensor([math.nan, math.inf, -math.inf, 65504.0], device=DEV, dtype=torch.float16).repeat(kv.numel() // 4 + 1)[: kv.numel()].view(kv.shape)
    dirty = torch.where(seen[None, :, None, :, None], kv, junk)
    table[:, -1] = 10**6                                                       # behind every row's last page
    a = paged_attention(q, kv[0], kv[1], table, lens, window=60)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    b = paged_attention(q, dirty[0], dirty[1], table, lens, window=60, status=status)
    assert torch.equal(a, b) and int(status) == 0


@pytest.mark.parametrize("keys", [40, 3000])
def test_infinities_and_nan_in_sight(keys):
    q, kv, table, lens = build([keys] * 4, 4, 1, 64, 16, torch.bfloat16, seed=1)
    q = q.abs() + 0.1
    kv[0][table[0, : -(-keys // 16)].long()] = -math.inf                       # every score -inf: nothing is seen
    kv[0][table[1, 0].long(), 0, 3] = -math.inf                                # one of them: the key drops out
    q[2] = math.nan
    kv[0][table[3, 1].long(), 0, 5, 7] = math.nan
    out, lse = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True)
    assert not out[0].any() and torch.all(lse[0] == -math.inf)
    clean = kv.clone()
    clean[0][table[1, 0].long(), 0, 3] = -30000.0
    want = formula(q[1:2], clean, table[1:2], lens[1:2])
    check(out[1:2], lse[1:2], want[:2] + formula(q[1:2], kv.nan_to_num(neginf=0.0), table[1:2], lens[1:2])[2:])
    assert torch.isnan(out[2:]).all() and torch.isnan(lse[2:]).all()


@pytest.mark.parametrize("entry", [-1, -2**31, 10**9, "pages"])
def test_a_bad_page_is_masked_and_reported(entry):
    q, kv, table, lens = build([300, 90], 4, 1, 128, 32, torch.bfloat16, seed=2)
    table[0, 4] = kv.shape[1] if entry == "pages" else entry
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True, status=status)
    assert int(status) == Status.BAD_PAGE
    # as if the 32 keys were not there
    short = torch.cat([table[:1, :4], table[:1, 5:]], 1)
    check(out[:1], lse[:1], formula(q[:1], kv, short, torch.tensor([268], dtype=torch.int32, device=DEV)))
    check(out[1:], lse[1:], formula(q[1:], kv, table[1:], lens[1:]))


def test_a_length_without_room_is_cut_and_reported():
    q, kv, table, lens = build([64, 40], 4, 1, 64, 16, torch.bfloat16, seed=2)
    table = table[:, :4].contiguous()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    long = torch.tensor([2**31 - 1, -5], dtype=torch.int32, device=DEV)
    out = paged_attention(q, kv[0], kv[1], table, long, status=status)
    assert int(status) == Status.BAD_PAGE and torch.equal(out[0], paged_attention(q, kv[0], kv[1], table, lens)[0]) and not out[1].any()


def test_views_and_given_outputs():
    q, kv, table, lens = build([100, 7, 513], 6, 2, 128, 16, torch.float16, seed=4)
    want = paged_attention(q, kv[0], kv[1], table, lens)
    wide_q = torch.randn(3, 20, 3 * 128 + 1, device=DEV).to(torch.float16)
    wide_q[:, 1:13:2, 3 : 3 + 128] = q
    pool = torch.randn(kv.shape[1], 2, 2, 16, 136, device=DEV).to(torch.float16)      # K and V side by side, padded rows
    kp, vp = pool[:, 0, :, :, :128], pool[:, 1, :, :, :128]
    kp.copy_(kv[0])
    vp.copy_(kv[1])
    wide_t = torch.full((3, 50), -1, dtype=torch.int32, device=DEV)
    wide_t[:, 10 : 10 + table.shape[1]] = table
    out = torch.full((3, 9, 130), 7.0, device=DEV, dtype=torch.float16)
    view = out[:, 1:7, 1:129]
    got = paged_attention(wide_q[:, 1:13:2, 3 : 3 + 128], kp, vp, wide_t[:, 10 : 10 + table.shape[1]], lens, out=view)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
    assert torch.all(out[:, 0] == 7) and torch.all(out[:, 7:] == 7) and torch.all(out[..., 0] == 7) and torch.all(out[..., 129] == 7)
    empty = paged_attention(q[:0], kv[0], kv[1], table[:0], lens[:0], return_lse=True)
    assert empty[0].shape == (0, 6, 128) and empty[1].shape == (0, 6)
    assert not paged_attention(q, kv[0], kv[1], table[:, :0], torch.zeros_like(lens)).any()


def test_offsets_beyond_32_bits():
    pages, page = 40, 65536
    kv = torch.empty(2, pages, 1, page, 256, dtype=torch.bfloat16, device=DEV)        # 1.3 GB a plane: pages from 32 on start beyond 2^31 values
    kv[:, 38:].normal_()
    table = torch.tensor([[38, 39]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([70000], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, 256, device=DEV).to(torch.bfloat16)
    out, lse = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True)
    check(out, lse, formula(q, kv, table, lens))


def test_captured_graphs_follow_their_inputs():
    """Two graphs of the same call replayed in turn while lengths, table and q change in place; and one on another stream than its tensors' own."""
    q, kv, table, lens = build([3000, 64, 500], 8, 2, 128, 32, torch.bfloat16, seed=6)
    st = torch.cuda.Stream()
    outs, graphs = [torch.empty_like(q) for _ in range(2)], []
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        paged_attention(q, kv[0], kv[1], table, lens)
    for o in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with graph_capture(graphs[-1], st):
            paged_attention(q, kv[0], kv[1], table, lens, out=o, window=0 if o is outs[0] else 100)
    for lengths in ([3000, 64, 500], [1, 0, 400], [2999, 65, 16]):
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        table[1, 2] = int(table[1, 1])
        q.mul_(0.9)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], paged_attention(q, kv[0], kv[1], table, lens)) and torch.equal(outs[1], paged_attention(q, kv[0], kv[1], table, lens, window=100))
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        side = paged_attention(q, kv[0], kv[1], table, lens)
    st.synchronize()
    assert torch.equal(side, paged_attention(q, kv[0], kv[1], table, lens))


def test_two_streams_at_once():
    """Calls that overlap have scratch of their own."""
    cases = [build([9000, 3, 700], 16, 2, 256, 32, torch.bfloat16, seed=i) for i in range(2)]
    want = [paged_attention(q, kv[0], kv[1], table, lens) for q, kv, table, lens in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                q, kv, table, lens = cases[i]
                got[i].append(paged_attention(q, kv[0], kv[1], table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [5.0, 10.0, 17.0, 25.0, 30.0])
@pytest.mark.parametrize("hq,dim,page", [(4, 64, 16), (12, 128, 40), (1, 256, 64), (16, 192, 16)])
def test_a_key_that_outweighs_all_others(dtype, gap, hq, dim, page):
    """One key of a row, the first, one in the middle, the last, with a value of zero (an attention sink): the result is what the others weigh, however
    little that is.  Values are large, so that the result is a number that fp16 holds."""
    lens = [3000, 2999, 70, 800]
    q, kv, table, n = build(lens, hq, 1, dim, page, dtype, seed=5)
    q.zero_()
    q[..., 0] = 4 * dim**0.5                                                   # scores are 4 K[0]: about N(0, 1)
    kv[0, ..., 0] *= 0.25
    kv[1] = (kv[1].abs().clamp(max=2.0) + 0.5) * 2.0**13
    for b, j in ((0, 0), (1, 1500), (2, 69), (3, 17)):
        kv[0, table[b, j // page].long(), 0, j % page, 0] = gap / 4
        kv[1, table[b, j // page].long(), 0, j % page] = 0.0
    out, lse = paged_attention(q, kv[0], kv[1], table, n, return_lse=True)
    check(out, lse, formula(q, kv, table, n))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rise", [1, -1])
def test_scores_that_rise_and_fall_through_their_range(dtype, rise):
    """Scores from 0 to 200 from key to key, upwards and downwards, and back and forth between 0 and 40 from tile to tile: what a weight is formed against moves all the time."""
    q, kv, table, n = build([2000, 1111], 3, 1, 128, 16, dtype, seed=9)
    q.zero_()
    q[..., 0] = 4 * 128**0.5
    ramp = torch.arange(2000, device=DEV) / 40.0
    for b, x in ((0, ramp if rise > 0 else ramp.flip(0)), (1, 10.0 * (torch.arange(2000, device=DEV) // 16 % 2))):
        for j in range(int(n[b])):
            kv[0, table[b, j // 16].long(), 0, j % 16, 0] = x[j]
    out, lse = paged_attention(q, kv[0], kv[1], table, n, return_lse=True)
    check(out, lse, formula(q, kv, table, n))


@pytest.mark.parametrize("keys", [40, 3000])
def test_infinities_and_nan_in_fp16(keys):
    q, kv, table, lens = build([keys] * 5, 4, 1, 64, 16, torch.float16, seed=1)
    q = q.abs() + 0.1
    kv[0][table[0, : -(-keys // 16)].long()] = -math.inf                       # every score -inf: nothing is seen
    kv[0][table[1, 0].long(), 0, 3] = -math.inf                                # one of them: the key drops out
    q[2] = math.nan
    kv[0][table[3, 1].long(), 0, 5, 7] = math.nan
    kv[0][table[4, 1].long(), 0, 5] = math.inf                                 # inf - inf
    out, lse = paged_attention(q, kv[0], kv[1], table, lens, return_lse=True)
    assert not out[0].any() and torch.all(lse[0] == -math.inf)
    clean = kv.clone()
    clean[0][table[1, 0].long(), 0, 3] = -30000.0
    want = formula(q[1:2], clean, table[1:2], lens[1:2])
    check(out[1:2], lse[1:2], want[:2] + formula(q[1:2], kv.nan_to_num(neginf=0.0, posinf=0.0), table[1:2], lens[1:2])[2:])
    assert torch.isnan(out[2:]).all() and torch.isnan(lse[2:]).all()


def test_a_length_that_is_cut_moves_the_window_and_the_distances():
    """A row longer than its table is the row that ends with the table's last column."""
    q, kv, table, lens = build([640, 40], 4, 2, 128, 16, torch.bfloat16, seed=2)
    table = table[:, :40].contiguous()
    slopes = torch.tensor([0.5, 0.1, 0.0, 1.0], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for n in (641, 700, 2**31 - 1):
        status.zero_()
        long = torch.tensor([n, 40], dtype=torch.int32, device=DEV)
        got = paged_attention(q, kv[0], kv[1], table, long, window=100, slopes=slopes, return_lse=True, status=status)
        want = paged_attention(q, kv[0], kv[1], table, lens, window=100, slopes=slopes, return_lse=True)
        assert int(status) == Status.BAD_PAGE and all(torch.equal(a, b) for a, b in zip(got, want))
    check(*want, formula(q, kv, table, lens, window=100, slopes=slopes))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 256])
def test_infinite_values_stay_in_their_dim(dtype, dim):
    q, kv, table, lens = build([40, 700, 700], 8, 2, dim, 16, dtype, seed=8)
    want = formula(q, kv, table, lens)
    bad = kv.clone()
    bad[1][table[0, 1].long(), 0, 3, 5] = math.inf
    bad[1][table[1, 30].long(), 1, 0, 6] = -math.inf
    bad[1][table[1, 31].long(), 1, 9, 7] = math.nan
    out, lse = paged_attention(q, bad[0], bad[1], table, lens, return_lse=True)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, :4, 5] = hit[1, 4:, 6] = hit[1, 4:, 7] = True
    assert not torch.isfinite(out[hit]).any() and torch.isfinite(out[~hit]).all()
    check(torch.where(hit, want[0].to(dtype), out), lse, want)


def test_the_result_may_take_the_place_of_q():
    """Items cut over many CTAs, whole ones and rows without keys."""
    for keys in ([50000], [3000, 0, 3, 70, 1000], [40] * 300):
        q, kv, table, lens = build(keys, 20, 2, 128, 16, torch.bfloat16, seed=5)
        want = paged_attention(q, kv[0], kv[1], table, lens)
        assert paged_attention(q, kv[0], kv[1], table, lens, out=q) is q and torch.equal(q, want)
