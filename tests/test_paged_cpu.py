"""Host side of the paged cache and beam search operators: refusals, the index arithmetic that the kernels share with the host, the split of
a batch's keys over CTAs, scaled rotary frequencies.  No GPU."""

import ctypes
import math
import random

import pytest
import torch

from nexrt_b200.ops import lib as L
from nexrt_b200.ops.beam import beam_select, reorder_rows
from nexrt_b200.ops.paged import PagedCache, compact_pages, copy_pages, fork_pages, paged_attention
from nexrt_b200.ops.rope import rope, rope_append, rope_frequencies

I32 = torch.int32


def _i32(*shape):
    return torch.zeros(*shape, dtype=I32)


def _attn(**change):
    kv = torch.zeros(2, 5, 2, 16, 64, dtype=torch.bfloat16)
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k_pages=kv[0], v_pages=kv[1], table=_i32(3, 4), lens=_i32(3))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(),                                                                      # tensors on the CPU
    dict(q=torch.zeros(3, 4, 64)),
    dict(q=torch.zeros(3, 5, 64, dtype=torch.bfloat16)),                         # 5 heads on 2
    dict(q=torch.zeros(3, 4, 80, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)),
    dict(q=torch.zeros(4, 64, dtype=torch.bfloat16)),
    dict(v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16)),
    dict(v_pages=torch.zeros(5, 2, 16, 128, dtype=torch.bfloat16)[..., :64]),    # strides differ
    dict(table=_i32(2, 4)),
    dict(table=torch.zeros(3, 4, dtype=torch.int64)),
    dict(table=_i32(4, 3).T),
    dict(lens=_i32(4)),
    dict(lens=torch.zeros(3)),
    dict(softcap=-1.0),
    dict(softcap=math.inf),
    dict(softcap=math.nan),
    dict(window=-1),
    dict(slopes=torch.zeros(4, dtype=torch.float16)),
    dict(slopes=torch.zeros(2)),
    dict(out=torch.zeros(3, 4, 64)),
    dict(status=torch.zeros(1)),
])
def test_attention_refuses(change):
    a = _attn(**change)
    with pytest.raises(ValueError):
        paged_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), a.pop("table"), a.pop("lens"), **a)


@pytest.mark.parametrize("change", [
    dict(),
    dict(q=torch.zeros(3, 4, 260)),
    dict(q=torch.zeros(3, 4, 60)),
    dict(k=torch.zeros(3, 2, 64, dtype=torch.bfloat16)),
    dict(v=torch.zeros(3, 3, 64)),
    dict(k=torch.zeros(2, 2, 64)),
    dict(positions=torch.zeros(3, dtype=torch.int64)),
    dict(rows=_i32(2)),
    dict(rows=_i32(6)[::2]),
    dict(inv_freq=torch.zeros(33)),
    dict(inv_freq=torch.zeros(8, dtype=torch.float64)),
    dict(q_norm=torch.zeros(32)),
    dict(k_norm=torch.zeros(64, dtype=torch.bfloat16)),
    dict(k_pages=torch.zeros(5, 3, 16, 64, dtype=torch.bfloat16), v_pages=torch.zeros(5, 3, 16, 64, dtype=torch.bfloat16)),
    dict(k_pages=torch.zeros(5, 2, 16, 64), v_pages=torch.zeros(5, 2, 16, 64)),
    dict(table=_i32(3)),
    dict(out=torch.zeros(3, 5, 64, dtype=torch.bfloat16)),
])
def test_rope_refuses(change):
    kv = torch.zeros(2, 5, 2, 16, 64, dtype=torch.bfloat16)
    a = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), positions=_i32(3), rows=_i32(3), k_pages=kv[0], v_pages=kv[1], table=_i32(3, 4),
             inv_freq=torch.zeros(16))
    a.update(change)
    args = [a.pop(n) for n in ("q", "k", "v", "positions", "rows", "k_pages", "v_pages", "table", "inv_freq")]
    with pytest.raises(ValueError):
        rope_append(*args, **a)


def test_rope_alone_refuses():
    q, pos, inv = torch.zeros(3, 4, 64), _i32(3), torch.zeros(16)
    for args, kw in (((q, pos, inv), {}), ((q.to(torch.float64), pos, inv), {}), ((q, pos.long(), inv), {}), ((q, pos, inv), dict(out=torch.zeros(3, 4, 64, dtype=torch.bfloat16))),
                     ((q, pos, inv), dict(norm=torch.zeros(16)))):
        with pytest.raises(ValueError):
            rope(*args, **kw)


def test_pages_refuse():
    kv, table, lens = torch.zeros(1, 2, 4, 1, 16, 64, dtype=torch.bfloat16), _i32(3, 4), _i32(3)
    par = _i32(3)
    bad = [
        lambda: fork_pages(kv, table, lens, par),                                    # on the CPU
        lambda: fork_pages(kv[0], table, lens, par),
        lambda: fork_pages(kv.transpose(3, 4), table, lens, par),
        lambda: fork_pages(torch.zeros(1, 2, 4, 1, 16, 7, dtype=torch.bfloat16), table, lens, par),
        lambda: fork_pages(kv, table.long(), lens, par),
        lambda: fork_pages(kv, table, _i32(4), par),
        lambda: fork_pages(kv, table, lens, par.long()),
        lambda: fork_pages(kv, table, lens, _i32(4097)),
        lambda: fork_pages(kv, table, lens, par, grow=-1),
        lambda: fork_pages(kv, table, lens, par, grow=_i32(2)),
        lambda: fork_pages(kv, table, lens, par, table_out=table),                   # rows are read while they are written
        lambda: fork_pages(kv, table, lens, par, lens_out=lens),
        lambda: fork_pages(kv, table, lens, par, refs=_i32(3)),
        lambda: compact_pages(kv, table, lens),
        lambda: compact_pages(kv, table, lens, table_out=table),
        lambda: compact_pages(kv, table, lens, refs=torch.zeros(4)),
        lambda: copy_pages(kv, par, _i32(2)),
        lambda: copy_pages(kv, par, par.long()),
        lambda: copy_pages(kv, par, par),
        lambda: PagedCache(1, 4, 1, 16, 80, 2, 64, device="cpu"),
        lambda: PagedCache(1, 0, 1, 16, 64, 2, 64, device="cpu"),
        lambda: PagedCache(1, 4, 1, 16, 64, 2, 64, device="cpu").fork(_i32(3)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise SystemExit(f"call {i} was taken")


def test_beam_refuses():
    x, s = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    bad = [
        lambda: beam_select(x, s, 3),                                                # on the CPU
        lambda: beam_select(x.double(), s, 3),
        lambda: beam_select(x[0], s, 3),
        lambda: beam_select(x.transpose(1, 2), s, 3),
        lambda: beam_select(x, s.double(), 3),
        lambda: beam_select(x, s[:, :2], 3),
        lambda: beam_select(x, s, 0),
        lambda: beam_select(x, s, 65),
        lambda: beam_select(x, s, 31),                                               # 30 candidates
        lambda: beam_select(x, s, 3, finished=torch.zeros(2, 3, dtype=torch.bool)),  # without an end token
        lambda: beam_select(x, s, 3, finished=torch.zeros(2, 3, dtype=torch.bool), eos=10),
        lambda: beam_select(x, s, 3, finished=torch.zeros(2, 3), eos=1),
        lambda: beam_select(torch.zeros(1, 257, 4), torch.zeros(1, 257), 3),
        lambda: reorder_rows([x], _i32(2)),
        lambda: reorder_rows([x, torch.zeros(3, 2)], _i32(2)),
        lambda: reorder_rows([x.transpose(1, 2)], _i32(2)),
        lambda: reorder_rows([x], torch.zeros(2, dtype=torch.int64)),
        lambda: reorder_rows([x], _i32(2), out=[torch.zeros(3, 3, 10)]),
        lambda: reorder_rows([x], _i32(2), out=[]),
        lambda: reorder_rows([x], _i32(1, 1, 2)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise SystemExit(f"call {i} was taken")


def test_no_rows_no_launch():
    assert reorder_rows([], _i32(2)) == []


def test_split_constants_match():
    """What the caller sizes its launch by is what the kernel splits by."""
    from nexrt_b200.ops import paged

    assert L.load().nexrt_paged_item_cost() == paged._ITEM_COST
    assert all(L.load().nexrt_paged_resident(d) == paged._resident(d) for d in paged.HEAD_DIMS)


def test_slot_of_a_position():
    """The device's page lookup, run on the host: entries that name no page of the pool, and places outside the table, give -1."""
    lib = L.load()
    table = torch.tensor([[3, 0, -1, 99], [5, 6, -7, 4]], dtype=I32)
    slot = lambda row, pos, width=3, rows=2: lib.nexrt_paged_slot(table.data_ptr(), table.stride(0), rows, width, 10, 6, row, pos)  # noqa: E731
    assert [slot(0, p) for p in (0, 9, 10, 19)] == [30, 39, 0, 9]
    assert slot(1, 3) == 53
    assert [slot(0, 20), slot(0, -1), slot(0, 30), slot(2, 0), slot(-1, 0), slot(1, 10), slot(1, 29)] == [-1] * 7    # -1, behind the row, no row, page 6 of 6, page -7
    assert slot(0, 30, width=4) == -1                                                                                # page 99
    assert lib.nexrt_paged_slot(torch.tensor([[2**30]], dtype=I32).data_ptr(), 1, 1, 1, 64, 2**30 + 1, 0, 5) == 2**36 + 5   # beyond 32 bits


@pytest.mark.parametrize("seed", range(60))
def test_split_covers_every_key_once(seed):
    """The walk of every CTA, run on the host: each chunk of each item exactly once and with the owners that the joining kernel reckons with
    (else the count comes back as -1), equal work (an item counts three chunks more than it has), and at most two cut items a CTA
    (the one it goes on with and the one it begins), which is what the parts' scratch has room for."""
    r = random.Random(seed)
    lib = L.load()
    lens = [r.choice([0, 0, 1, 63, 64, 65, -3, int(math.exp(r.uniform(0, 11)))]) for _ in range(r.randint(1, 40))]
    items, window, grid = r.randint(1, 9), r.choice([0, 0, 1, 64, 100, 5000]), r.choice([1, 3, 148, 296])
    room = r.choice([max(1, max(lens)), 100000, 50])
    out = torch.zeros(60000, 5, dtype=torch.int64)
    n = lib.nexrt_paged_split((ctypes.c_int * len(lens))(*lens), len(lens), items, room, window, grid, out.data_ptr(), 60000)
    assert n <= 60000
    want = {}
    for b, x in enumerate(lens):
        hi = max(0, min(x, room))
        lo = max(0, hi - window) if window else 0
        if hi > lo:
            for i in range(items):
                want[b, i] = (hi - 1) // 64 - lo // 64 + 1
    got, load, cut = {}, {}, {}
    for cta, b, i, first, count in out[:n].tolist():
        assert count > 0 and got.get((b, i), 0) == first          # in the order of the keys, without a gap
        got[b, i] = first + count
        load[cta] = load.get(cta, 0) + count + (3 if first == 0 else 0)
        if count < want[b, i]:
            cut.setdefault(cta, []).append(first > 0)
    assert got == want
    if load:
        total = sum(w + 3 for w in want.values())
        share = total / min(grid, total)
        assert max(load.values()) <= share + 4 and all(len(set(c)) == len(c) for c in cut.values()) and len(load) <= grid


def test_frequencies():
    inv, scale = rope_frequencies(64, 1e7)
    assert scale == 1.0 and torch.equal(inv, torch.tensor([1e7 ** (-i / 32) for i in range(32)], dtype=torch.float32))
    lin, _ = rope_frequencies(64, 1e7, "linear", 4.0)
    assert torch.allclose(lin * 4, inv, rtol=1e-6)
    base, _ = rope_frequencies(64, 1e7, "base", 4.0)
    assert base[0] == inv[0] and abs(base[-1] * 4 / inv[-1] - 1) < 1e-5
    ramp, scale = rope_frequencies(128, 1e4, "ramp", 8.0, trained=4096)
    plain, _ = rope_frequencies(128, 1e4)
    turns = plain.double() * 4096 / (2 * math.pi)
    ratio = plain.double() / ramp.double()
    assert scale == pytest.approx(1 + 0.1 * math.log(8)) and torch.all(ratio[turns > 40] < 1.001) and torch.all((ratio[turns < 0.8] - 8).abs() < 1e-3)
    assert torch.all(ratio[1:] >= ratio[:-1] - 1e-6)
    for bad in (lambda: rope_frequencies(63, 1e4), lambda: rope_frequencies(64, 1.0), lambda: rope_frequencies(64, 1e4, "other"), lambda: rope_frequencies(64, 1e4, "ramp", 2.0),
                lambda: rope_frequencies(64, 1e4, "linear", 0.5), lambda: rope_frequencies(0, 1e4)):
        with pytest.raises(ValueError):
            bad()


def test_gradients_are_not_lost_without_a_word():
    """Nothing here has a backward pass: a tensor that requires a gradient is refused, and taken as any other where gradients are off (here: until
    its device is looked at)."""
    kv, table, lens, one = torch.zeros(1, 2, 4, 2, 16, 64), _i32(3, 4), _i32(3), torch.zeros(3, 2, 64)
    bf = kv.to(torch.bfloat16)
    need = lambda t: t.clone().requires_grad_()  # noqa: E731
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    append = dict(q=one, k=one, v=one, positions=lens, rows=lens, k_pages=bf[0, 0], v_pages=bf[0, 1], table=table, inv_freq=torch.zeros(8), q_norm=torch.ones(64), k_norm=torch.ones(64))
    attend = dict(q=q, k_pages=bf[0, 0], v_pages=bf[0, 1], table=table, lens=lens, slopes=torch.ones(4))
    turn = dict(q=one, positions=lens, inv_freq=torch.zeros(8), norm=torch.ones(64))
    pick = dict(logits=torch.zeros(2, 3, 10), scores=torch.zeros(2, 3), k=3)
    calls = [(rope_append, append, n) for n in ("q", "k", "v", "k_pages", "v_pages", "inv_freq", "q_norm", "k_norm")]
    calls += [(paged_attention, attend, n) for n in ("q", "k_pages", "v_pages", "slopes")] + [(rope, turn, n) for n in ("q", "inv_freq", "norm")]
    calls += [(beam_select, pick, n) for n in ("logits", "scores")]
    calls += [(fork_pages, dict(kv=bf, table=table, lens=lens, parents=lens), "kv"), (compact_pages, dict(kv=bf, table=table, lens=lens), "kv"), (copy_pages, dict(kv=bf, src=lens, dst=lens), "kv")]
    for call, args, name in calls:
        args = dict(args, **{name: need(args[name])})
        with pytest.raises(ValueError, match="backward"):
            call(**args)
        with torch.no_grad(), pytest.raises(ValueError, match="CPU"):
            call(**args)
    with pytest.raises(ValueError, match="backward"):
        reorder_rows([need(one)], _i32(2))
    with pytest.raises(ValueError, match="backward"):
        reorder_rows([one], _i32(2), out=[need(torch.zeros(2, 2, 64))])


def test_outputs_whose_rows_lie_over_one_another_are_refused():
    kv, table, lens = torch.zeros(1, 2, 4, 1, 16, 64, dtype=torch.bfloat16), _i32(3, 4), _i32(3)
    q, kp = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)
    one = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    flat = _i32(20)
    append = lambda out: rope_append(q, one, one, lens, lens, kp, kp, table, torch.zeros(8), out=out)  # noqa: E731
    for call in (lambda: fork_pages(kv, table, lens, lens, table_out=flat[:4].expand(3, 4)),
                 lambda: fork_pages(kv, table, lens, lens, table_out=flat.as_strided((3, 4), (3, 1))),
                 lambda: compact_pages(kv, table, lens, table_out=flat[:4].expand(3, 4)),
                 lambda: paged_attention(q, kp, kp, table, lens, out=q[:1].clone().expand(3, 4, 64)),
                 lambda: paged_attention(q, kp, kp, table, lens, out=q[:, :1].clone().expand(3, 4, 64)),
                 lambda: rope(q, lens, torch.zeros(8), out=q[:1].clone().expand(3, 4, 64)),
                 lambda: append(q[:, :1].clone().expand(3, 4, 64)),
                 lambda: reorder_rows([torch.zeros(4, 6)], lens, out=[torch.zeros(1, 6).expand(3, 6)])):
        with pytest.raises(ValueError, match="over one another|place of its own"):
            call()
    with pytest.raises(ValueError, match="CPU"):                                  # one row may have any stride
        fork_pages(kv, table, lens, lens[:1], table_out=flat.as_strided((1, 4), (0, 1)))
