"""Beam selection against float64 and Python's sort - ties, masked and odd vocabularies, finished, missing and broken beams -, the reordering of rows, and a
beam search with an attention layer of the framework's over a paged cache against its oracle."""

import copy
import math

import pytest
import torch

from nexrt_b200.models.reference import RefLayerState, RefModel, rms_norm
from nexrt_b200.ops.beam import beam_select, reorder_rows
from nexrt_b200.ops.paged import PagedCache
from nexrt_b200.ops.rope import rope_frequencies
from nexrt_b200.runtime.capture import graph_capture
from nexrt_b200.runtime.control import Status
from nexrt_b200.testing import shrunk_checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def by_sorting(logits, scores, k, finished=None, eos=-1):
    """[(total, row, token)] best first, of every request."""
    x, out = logits.double().cpu(), []
    B, W, V = x.shape
    for b in range(B):
        found = []
        for w in range(W):
            s = float(scores[b, w].double())
            done = finished is not None and bool(finished[b, w])
            dead = not math.isfinite(s) or not bool(torch.all(x[b, w] < math.inf))
            if done or dead:
                own = [(-s, w, 0.0, eos)] if done and s < math.inf else []
                found += own + [(math.inf, w, 0.0, t) for t in range(min(V, k + 1)) if not (own and t == eos)]
                continue
            lse = torch.logsumexp(x[b, w], -1)
            p = s + (x[b, w] - lse) if lse > -math.inf else x[b, w]
            order = torch.sort(x[b, w], descending=True, stable=True).indices[:k].tolist()
            found += [(-float(p[t]), w, -float(x[b, w, t]), t) for t in order]
        found.sort()
        out.append([(-f[0], b * W + f[1], f[3]) for f in found[:k]])
    return out


def check(logits, scores, k, finished=None, eos=-1, code=0):
    status = ints([0])
    s, r, t = beam_select(logits, scores, k, finished=finished, eos=eos, status=status)
    want = by_sorting(logits, scores, k, finished, eos)
    assert r.tolist() == [[f[1] for f in row] for row in want]
    assert t.tolist() == [[f[2] for f in row] for row in want]
    w = torch.tensor([[f[0] for f in row] for row in want], dtype=torch.float64)
    fine = torch.isfinite(w)
    # the sum of exp is good to 2^-20 (each term's argument below 2^-18 off where it matters: |x - max| < 20), then one rounding to 32 bits
    assert torch.equal(s.cpu()[~fine].double(), w[~fine]) and torch.all((s.cpu().double() - w)[fine].abs() <= 2.0**-20 + 2.0**-23 * w[fine].abs())
    assert int(status) == code
    return s, r, t


def inputs(B, W, V, dtype=torch.float32, seed=0, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + V)
    return (torch.randn(B, W, V, device=DEV, generator=g) * std).to(dtype), -torch.rand(B, W, device=DEV, generator=g) * 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,W,V,k", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 20), (1, 4, 8192, 8), (3, 2, 8193, 4), (2, 5, 50257, 10), (1, 8, 248320, 16), (5, 16, 1001, 32), (1, 256, 300, 64), (40, 2, 4096, 3)])
def test_select(dtype, B, W, V, k):
    check(*inputs(B, W, V, dtype), k)


@pytest.mark.parametrize("V,k", [(9000, 16), (70000, 64), (64, 64), (8000, 1)])
def test_ties_go_to_the_lowest(V, k):
    """Constant rows, a few distinct values, and two beams that are equal to the last bit."""
    x, s = inputs(2, 3, V, std=1.0)
    s[:, 1] = s[:, 0]
    check(torch.zeros_like(x), s, k)
    check(x.round(), s, k)
    x[:, 1] = x[:, 0]
    check(x, s, k)
    x[..., ::3] = 0.0
    x[..., 1::3] = -0.0
    check(x, s, k)


def test_masked_vocabularies():
    x, s = inputs(3, 4, 20000)
    x[0] = -math.inf
    x[0, 2, 17] = 1.0                                  # one token in all
    x[1, :, 100:] = -math.inf
    x[1, 3] = -math.inf
    x[2, 0, :19999] = torch.finfo(torch.float32).min   # masked by the lowest number instead: far below, but numbers
    check(x, s, 8)
    s[1] = -math.inf
    s[2, 1:] = -math.inf                               # the first step of a search: one beam
    check(x, s, 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,k", [(50257, 8), (248320, 16), (33000, 64)])
def test_values_in_masses(dtype, V, k):
    """Almost everything masked, by -inf and by the lowest number, the little that is allowed at either end, in the middle, or less than k; a
    block of equal values; logits in ascending order, where every step has more above the bound than there is room for."""
    x, s = inputs(2, 4, V, dtype)
    for mask in (-math.inf, torch.finfo(dtype).min):
        for first, n in ((0, 40), (V - 700, 700), (V // 2, 3), (V // 3, 9000)):
            y = torch.full_like(x, mask)
            y[..., first : first + n] = x[..., first : first + n]
            check(y, s, k)
    y = x.clone()
    y[..., 100 : V // 2] = 3.0
    check(y, s, k)
    check(torch.sort(x, -1).values, s, k)
    check(torch.sort(x, -1, descending=True).values, s, k)


def test_many_beams_of_one_score():
    """Candidates of eight beams whose lists lie side by side in the join; and of 256, where the high ones all lie with half of its threads and
    more of them reach its bound than there is room for - different ones, and equal ones, of which the order of beams and tokens decides."""
    x, s = inputs(1, 8, 248320)
    check(x, torch.zeros_like(s), 64)
    x, s = inputs(1, 256, 300, std=0.01)
    w = torch.arange(256, device=DEV)
    high = (64 * (w % 8) - 199 * (w // 8)) % 512 <= 188
    assert int(high.sum()) * 64 > 4096
    s = torch.where(high, 0.0, -1000.0)[None]
    check(x, s, 64)
    check(torch.zeros_like(x), s, 64)


def test_finished_and_broken_beams():
    x, s = inputs(4, 4, 3000)
    fin = torch.zeros(4, 4, dtype=torch.bool, device=DEV)
    fin[0, 1] = fin[1] = fin[2, 0] = True
    s[0, 1], s[2, 0] = -0.001, -1e6
    x[0, 1] = math.nan                                 # a finished beam's logits are not looked at
    check(x, s, 6, fin, 2)
    check(x, s, 6, fin, 0)
    check(x, s, 6, fin, 2999)
    s[2, 0] = -math.inf
    check(x, s, 6, fin, 5)
    x[3, 2, 77] = math.nan
    check(x, s, 6, fin, 5, Status.NON_FINITE)
    x[3, 2, 77] = math.inf
    check(x, s, 6, fin, 5, Status.NON_FINITE)
    x[3, 2, 77] = 0.0
    s[3, 0] = math.nan
    check(x, s, 6, fin, 5, Status.NON_FINITE)
    x[3] = math.nan
    check(x, s, 6, fin, 5, Status.NON_FINITE)


def test_strides_and_repeated_rows():
    x, s = inputs(3, 4, 1003, torch.bfloat16)
    wide = torch.zeros(3, 9, 1010, device=DEV, dtype=torch.bfloat16)
    wide[:, 1:9:2, 3:1006] = x
    a = beam_select(x, s, 8)
    b = beam_select(wide[:, 1:9:2, 3:1006], s.t().contiguous().t(), 8)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    check(x[:, :1].expand(-1, 4, -1), s, 8)            # the first step: all beams look at one row
    e = beam_select(x[:0], s[:0], 8)
    assert e[0].shape == (0, 8)


def test_sums_of_a_large_vocabulary():
    """A million equal logits beside a few large ones."""
    x = torch.full((1, 2, 1 << 20), 3.0, device=DEV)
    x[0, 1, 5] = 3.5
    check(x, torch.zeros(1, 2, device=DEV), 4)


@pytest.mark.parametrize("dtype,shape", [(torch.float32, (3, 5)), (torch.bfloat16, (7,)), (torch.int8, (3, 1, 11)), (torch.float16, (4, 128, 128)), (torch.float32, (20000, 3)), (torch.int64, ())])
def test_reorder(dtype, shape):
    x = torch.randint(-100, 100, (9, *shape), device=DEV).to(dtype)
    rows = ints([3, 3, 0, 8, 1, 3])
    assert torch.equal(reorder_rows([x], rows)[0], x[rows.long()])
    two = ints([[1, 2, 3], [8, 0, 0]])
    assert torch.equal(reorder_rows([x], two[:, :2])[0], x[two[:, :2].reshape(-1).long()])


def test_reorder_many_strided_and_bad():
    xs = [torch.randn(6, 10 + i, device=DEV) for i in range(37)]
    rows = ints([5, 0, 0, 2])
    assert all(torch.equal(o, x[rows.long()]) for o, x in zip(reorder_rows(xs, rows), xs))
    wide = torch.randn(6, 4, 33, device=DEV)
    out = torch.zeros(4, 3, 33, device=DEV)
    reorder_rows([wide[:, 1]], rows, out=[out[:, 1]])
    assert torch.equal(out[:, 1], wide[rows.long(), 1]) and not out[:, 0].any() and not out[:, 2].any()
    x, out, status = torch.ones(3, 100, device=DEV), torch.full((4, 100), 7.0, device=DEV), ints([0])
    reorder_rows([x], ints([0, 3, -1, 2]), out=[out], status=status)
    assert int(status) == Status.BAD_PAGE and out[:, 0].tolist() == [1.0, 7.0, 7.0, 1.0]
    with pytest.raises(ValueError):
        reorder_rows([x], ints([0, 1, 2]), out=[x])
    assert reorder_rows([x], ints([]))[0].shape == (0, 100)


def test_captured_selection():
    x, s = inputs(2, 4, 5000)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        beam_select(x, s, 8)
    graphs, outs = [], []
    for k in (8, 3):
        graphs.append(torch.cuda.CUDAGraph())
        with graph_capture(graphs[-1], st):
            outs.append(beam_select(x, s, k))
    for i in range(3):
        x.copy_(torch.randn_like(x).round() if i else torch.randn_like(x))
        graphs[0].replay()
        graphs[1].replay()
        for o, k in zip(outs, (8, 3)):
            assert all(torch.equal(a, b) for a, b in zip(o, beam_select(x, s, k)))


def test_beam_search_over_a_paged_cache():
    """A language model of one attention layer of the shrunk checkpoint: embedding, attention with its norms, rotation and gate, head.
    Every beam's logits against the oracle run on the beam's own tokens, and the selection against the oracle's totals."""
    cfg, ckpt = shrunk_checkpoint(0)
    ref = RefModel(cfg, ckpt)
    w = ref.layers[1]
    hd, nq, nk, W, page = cfg.head_dim, cfg.n_q_heads, cfg.n_kv_heads, 3, 4
    dev = {n: w[n].to(DEV) for n in ("in_ln", "q", "k", "v", "o", "qn", "kn")}
    embed, final_ln, head = ref.embed.to(DEV), ref.final_ln.to(DEV), ref.lm_head.to(DEV)
    inv = rope_frequencies(cfg.rotary_dim, cfg.rope_theta)[0].to(DEV)
    cache = PagedCache(1, 24, nk, page, hd, W, 64)
    state = torch.zeros(W, 6, device=DEV)                          # a beam's last six tokens: what a recurrent state is here

    def gpu_step(tokens):
        x = embed[tokens]
        xn = rms_norm(x, dev["in_ln"], cfg.rms_eps)
        q, gate = (xn @ dev["q"].T).view(W, nq, 2, hd).unbind(2)
        q = cache.append(0, q, (xn @ dev["k"].T).view(W, nk, hd), (xn @ dev["v"].T).view(W, nk, hd), cache.lens - 1, cache.same, inv, q_norm=dev["qn"], k_norm=dev["kn"], eps=cfg.rms_eps)
        y = cache.attend(0, q).float() * torch.sigmoid(gate)
        return rms_norm(x + y.flatten(1) @ dev["o"].T, final_ln, cfg.rms_eps) @ head.T

    def oracle_step(st, token, pos):
        x = ref.embed[token]
        return rms_norm(x + ref._attn(w, st, x, pos), ref.final_ln, cfg.rms_eps) @ ref.lm_head.T

    beams = [(0.0, [7], RefLayerState())] + [(-math.inf, [7], RefLayerState()) for _ in range(W - 1)]
    scores = torch.tensor([[0.0] + [-math.inf] * (W - 1)], device=DEV)
    tokens, parents = torch.full((W,), 7, device=DEV), None
    for pos in range(11):
        cache.fork(parents, 1)
        logits = gpu_step(tokens)
        for i, (_, seq, st) in enumerate(beams):
            want = oracle_step(st, seq[-1], pos)
            got = logits[i].cpu()
            assert float((got - want).norm() / want.norm()) < 6e-3   # K, V, q and the output rounded to bf16: half a step, 2^-8 = 4e-3, each, in quadrature behind a residual
        scores, rows, picked = beam_select(logits[None], scores, W)
        totals = torch.stack([s + torch.log_softmax(logits[i].double().cpu(), -1) for i, (s, _, _) in enumerate(beams)])
        best = totals.flatten().topk(W).values
        for j, (r, t) in enumerate(zip(rows[0].tolist(), picked[0].tolist())):
            assert abs(float(totals[r, t]) - float(scores[0, j])) < 1e-5 * (pos + 1) and abs(float(totals[r, t]) - float(best[j])) < 1e-5 * (pos + 1)
        state = torch.roll(reorder_rows([state], rows[0])[0], -1, 1)
        state[:, -1] = picked[0].float()
        beams = [(float(scores[0, j]), beams[r][1] + [t], copy.deepcopy(beams[r][2])) for j, (r, t) in enumerate(zip(rows[0].tolist(), picked[0].tolist()))]
        assert state.tolist() == [([0.0] * 6 + [float(t) for t in b[1][1:]])[-6:] for b in beams]
        parents, tokens = rows[0].contiguous(), picked[0].long()
        if pos == 5:
            cache.compact()
    cache.check()
    assert len({tuple(b[1]) for b in beams}) == W


def test_a_captured_beam_step_goes_on_like_an_eager_one():
    """Fork, append, attend, select and reorder as one graph, replayed, against the same step called eagerly on a second cache; a row of the batch is padding."""
    W, hq, hk, dim, V, page = 4, 6, 2, 128, 700, 8
    g = torch.Generator(device=DEV).manual_seed(3)
    embed, wq, wo = (torch.randn(*n, device=DEV, generator=g) * 0.1 for n in ((V, 64), (64, (hq + 2 * hk) * dim), (hq * dim, V)))
    inv = rope_frequencies(dim, 1e4)[0].to(DEV)

    class Run:
        def __init__(self):
            self.cache = PagedCache(1, 60, hk, page, dim, W + 1, 96)
            self.parents, self.tokens = ints([0, 0, 0, 0, -1]), torch.full((W,), 5, device=DEV)
            self.scores = torch.tensor([[0.0, -math.inf, -math.inf, -math.inf]], device=DEV)
            self.state, self.other = torch.zeros(W, 33, device=DEV), torch.zeros(W, 33, device=DEV)

        def step(self):
            c = self.cache
            c.fork(self.parents, 1)
            x = torch.zeros(W + 1, 64, device=DEV)
            x[:W] = embed[self.tokens]
            h = (x @ wq).view(W + 1, -1, dim)
            rows = torch.where(c.lens > 0, c.same, -1)                         # the last row is empty: nothing is stored for it
            q = c.append(0, h[:, :hq], h[:, hq : hq + hk], h[:, hq + hk :], c.lens - 1, rows, inv)
            y = c.attend(0, q, softcap=20.0).float()
            assert y.shape == (W + 1, hq, dim)
            s, r, t = beam_select((y[:W].flatten(1) @ wo)[None], self.scores, W)
            reorder_rows([self.state], r, out=[self.other])
            self.state.copy_(self.other)
            self.state[:, 0] += t[0].float()
            self.scores.copy_(s)
            self.tokens.copy_(t[0])
            self.parents[:W].copy_(r[0])

    a, b = Run(), Run()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a.step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph, st):
        a.step()
    b.step()
    for _ in range(20):
        graph.replay()
        b.step()
        for x, y in ((a.cache.table, b.cache.table), (a.cache.lens, b.cache.lens), (a.cache.refs, b.cache.refs), (a.scores, b.scores), (a.tokens, b.tokens), (a.state, b.state)):
            assert torch.equal(x, y)
    a.cache.check()
    b.cache.check()
    assert a.cache.lens.tolist() == [21] * W + [0] and torch.equal(a.cache.kv, b.cache.kv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [501, 1001, 4098, 50257, 131075])
def test_equal_beams_of_any_alignment_tie(dtype, V):
    """Rows of an odd vocabulary start anywhere between two 16-byte boundaries.  Beams that hold the same numbers have the same totals to the last bit
    all the same, so the lower beam goes first; and a row's totals do not go by its address."""
    one = inputs(1, 1, V, dtype, seed=1)[0]
    x, s = one.expand(2, 9, V).contiguous(), torch.full((2, 9), -1.5, device=DEV)
    scores, rows, tokens = beam_select(x, s, 20)
    logits, at = torch.sort(one[0, 0].float(), descending=True, stable=True)
    want = sorted((-v, w, t) for v, t in zip(logits[:40].tolist(), at[:40].tolist()) for w in range(9))[:20]
    for b in range(2):
        assert list(zip(rows[b].tolist(), tokens[b].tolist())) == [(w + 9 * b, t) for _, w, t in want]
        assert len(set(scores[b].tolist())) == len({v for v, _, _ in want})
    totals = []
    for off in range(8):
        wide = torch.zeros(V + 8, device=DEV, dtype=dtype)
        wide[off : off + V] = one[0, 0]
        totals.append(beam_select(wide[off : off + V].view(1, 1, V), s[:1, :1], 20)[0])
    assert all(torch.equal(t, totals[0]) for t in totals)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("off", range(1, 8))
@pytest.mark.parametrize("V", [1, 6, 8, 13, 4093, 4096, 8192, 16384 + 5, 33000])
def test_rows_at_every_start(dtype, off, V):
    """Vocabularies that end in, at and behind a step, between neighbours that must not be read as logits."""
    x, s = inputs(1, 1, V, dtype, seed=off)
    wide = torch.full((V + 16,), 1000.0, device=DEV, dtype=dtype)
    wide[off : off + V] = x[0, 0]
    check(wide[off : off + V].view(1, 1, V), s, min(V, 12))


@pytest.mark.parametrize("n_in", [3, 0])
def test_rows_that_do_not_exist_are_zeros_of_a_new_tensor(n_in):
    torch.full((1 << 20,), 7.0, device=DEV)                                     # what the allocator gives out next is not zeros
    xs = [torch.ones(n_in, *s, device=DEV).to(t) for s, t in (((100,), torch.float32), ((7,), torch.int8), ((3, 5), torch.float16), ((40000,), torch.bfloat16), ((), torch.int64))]
    status = ints([0])
    got = reorder_rows(xs, ints([0, 3, -1, 2]), status=status)
    want = [float(0 <= r < n_in) for r in (0, 3, -1, 2)]
    assert all(torch.equal(g.double().flatten(1) if g.dim() > 1 else g.double()[:, None], torch.tensor(want, device=DEV, dtype=torch.float64)[:, None].expand(4, max(1, g[0].numel()))) for g in got)
    assert int(status) == Status.BAD_PAGE
