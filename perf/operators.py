"""Operators of a paged key-value cache and of beam search over it, in their plain form and as the framework's calls.

Kinds of case, and what each stands for in real use:

* ``rope``     rotary positions: the new tokens' q and k heads are normalised and rotated, and k and v stored into the pages
               of their sequences (``ops.rope.rope_append``).  ``decode`` gives every row one token at a position of its own,
               otherwise the rows are chunks of prompts that start anywhere in a long context.
* ``attn``     attention of one new token of every sequence over its pages (``ops.paged.paged_attention``): ragged lengths,
               empty rows, capped scores, a bias that falls with the distance, a window.
* ``fork``     one beam-search step of the cache (``ops.paged.fork_pages``): every row continues one of the old rows, shared
               pages are counted, a shared page that is about to be written is copied, new pages are taken.
* ``compact``  live pages move to the front of the pool (``ops.paged.compact_pages``), so that its end can be given back.
* ``beam``     selection over beams and vocabulary (``ops.beam.beam_select``) and reordering of the recurrent states of the
               rows that go on (``ops.beam.reorder_rows``).

The geometries are the served model's (32 query heads, 2 key-value heads of 256, rotary 64, vocabulary 248320, gated-delta-net
states of 64 heads of 128 x 128; divided by eight in the deployment) and generic ones of the same families.
"""

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # eight beams of the deployment's shard, one token each, far into a long context: the smallest call
        {"name": "rope_8rows_tp8", "kind": "rope", "tokens": 8, "rows": 8, "decode": True, "q_heads": 4, "kv_heads": 1, "dim": 256, "rotary": 64,
         "interleaved": False, "scaled": False, "norm": True, "dtype": "bf16", "page": 64, "context": 262144},
        # a chunk of three prompts, unsharded heads
        {"name": "rope_prompt_4099", "kind": "rope", "tokens": 4099, "rows": 3, "decode": False, "q_heads": 32, "kv_heads": 2, "dim": 256, "rotary": 64,
         "interleaved": False, "scaled": False, "norm": True, "dtype": "bf16", "page": 64, "context": 262144},
        # interleaved pairs over the whole head, frequencies stretched for four times the trained context
        {"name": "rope_interleaved_1111", "kind": "rope", "tokens": 1111, "rows": 7, "decode": False, "q_heads": 16, "kv_heads": 4, "dim": 128, "rotary": 128,
         "interleaved": True, "scaled": True, "norm": False, "dtype": "fp16", "page": 16, "context": 131072},
        # one short chat on the deployment's shard: latency
        {"name": "attn_1seq_1100_tp8", "kind": "attn", "seqs": 1, "q_heads": 4, "kv_heads": 1, "dim": 256, "page": 64, "keys": 1100, "ragged": False,
         "dtype": "bf16", "softcap": 0.0, "window": 0, "bias": False},
        # one book-length document, unsharded heads
        {"name": "attn_1seq_200k", "kind": "attn", "seqs": 1, "q_heads": 32, "kv_heads": 2, "dim": 256, "page": 64, "keys": 200000, "ragged": False,
         "dtype": "bf16", "softcap": 0.0, "window": 0, "bias": False},
        # a serving batch of very different lengths, an empty row among them
        {"name": "attn_48seqs_ragged", "kind": "attn", "seqs": 48, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "keys": 16384, "ragged": True,
         "dtype": "fp16", "softcap": 0.0, "window": 0, "bias": False},
        # capped scores with a distance bias in a window, pages that end inside a tile
        {"name": "attn_16seqs_capped", "kind": "attn", "seqs": 16, "q_heads": 24, "kv_heads": 8, "dim": 64, "page": 40, "keys": 9000, "ragged": True,
         "dtype": "bf16", "softcap": 30.0, "window": 4097, "bias": True},
        # one beam-search step of one request on the deployment's shard: all full-attention layers
        {"name": "fork_8beams_tp8", "kind": "fork", "groups": 1, "beams": 8, "keys": 8191, "page": 64, "layers": 15, "kv_heads": 1, "dim": 256, "dtype": "bf16"},
        # the same for sixteen requests at once, a few layers of a smaller model
        {"name": "fork_16x8beams", "kind": "fork", "groups": 16, "beams": 8, "keys": 20000, "page": 32, "layers": 4, "kv_heads": 4, "dim": 64, "dtype": "fp16"},
        # a pool that long-running requests have left full of holes
        {"name": "compact_1500pages_tp8", "kind": "compact", "pages": 1500, "live": 0.6, "rows": 24, "page": 64, "layers": 15, "kv_heads": 1, "dim": 256,
         "dtype": "bf16"},
        # four beams over the served vocabulary, states of two gated-delta-net layers of a shard
        {"name": "beam_4", "kind": "beam", "batch": 1, "beams": 4, "k": 8, "vocab": 248320, "dtype": "fp32", "finished": 0, "state_heads": 8, "states": 2},
        # sixteen requests of eight beams, logits in bf16 (full of ties), some beams finished
        {"name": "beam_16x8", "kind": "beam", "batch": 16, "beams": 8, "k": 16, "vocab": 248320, "dtype": "bf16", "finished": 11, "state_heads": 8, "states": 1},
    ]


def _span(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "attn", "attn", "attn", "fork", "compact", "beam", "beam"])
    dim = rng.choice([64, 128, 128, 256, 256])
    kv_heads = rng.choice([1, 1, 2, 4, 8]) if dim < 256 else rng.choice([1, 1, 2])
    page = rng.choice([16, 16, 32, 64, 64, 128, 24, 100])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "rope":
        decode = rng.random() < 0.5
        tokens = _span(rng, 1, 300) if decode else _span(rng, 20, 4099)
        rotary = rng.choice([dim, dim, dim // 2, dim // 4, dim // 2 + 4])
        return {"kind": kind, "tokens": tokens, "rows": tokens if decode else rng.randint(1, 7), "decode": decode, "q_heads": kv_heads * rng.choice([1, 4, 7, 8]),
                "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": rng.random() < 0.4, "scaled": rng.random() < 0.4, "norm": rng.random() < 0.5,
                "dtype": dtype, "page": page, "context": rng.choice([4096, 32768, 131072, 262144])}
    if kind == "attn":
        seqs = _span(rng, 1, 64)
        keys = _span(rng, 1, min(200000, 400000 * 256 // (seqs * kv_heads * dim)))
        return {"kind": kind, "seqs": seqs, "q_heads": kv_heads * rng.choice([1, 3, 4, 8, 16]), "kv_heads": kv_heads, "dim": dim, "page": page, "keys": keys,
                "ragged": rng.random() < 0.7, "dtype": dtype, "softcap": rng.choice([0.0, 0.0, 20.0, 50.0]), "window": rng.choice([0, 0, 0, 1, 128, 1000, 4096]),
                "bias": rng.random() < 0.3}
    if kind == "fork":
        groups, beams = _span(rng, 1, 16), rng.choice([1, 2, 3, 4, 5, 8])
        layers = rng.randint(1, 8)
        keys = _span(rng, 1, min(20000, 10 ** 9 // (groups * layers * kv_heads * dim * 4)))
        return {"kind": kind, "groups": groups, "beams": beams, "keys": keys, "page": page, "layers": layers, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if kind == "compact":
        layers = rng.randint(1, 15)
        most = min(1500, 1200 * 10 ** 6 // (layers * kv_heads * page * dim * 4))
        pages = _span(rng, 30, max(31, most))
        return {"kind": kind, "pages": pages, "live": round(rng.uniform(0.05, 0.95), 3), "rows": rng.randint(1, 64), "page": page, "layers": layers,
                "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    batch, beams = _span(rng, 1, 16), rng.choice([1, 2, 3, 4, 5, 8])
    vocab = _span(rng, 500, 248320)
    return {"kind": kind, "batch": batch, "beams": beams, "k": rng.choice([beams, 2 * beams]), "vocab": vocab, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
            "finished": rng.randint(0, batch * (beams - 1)), "state_heads": rng.choice([1, 4, 8]), "states": rng.randint(1, 2)}


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * seed + 17)
    return g


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _fixed(case):
    """What is random about a case's shape (lengths, who forks whom) and not about its data: the same for every seed."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _frequencies(case):
    """Inverse frequencies of the rotated pairs, in 32 bits, and the factor on cos and sin.  Scaled: pairs that turn less than
    once over the trained context are slowed down four times, those that turn 32 times or more are left, with a ramp between."""
    n, theta = case["rotary"], 1.0e7
    inv = [theta ** (-2.0 * i / n) for i in range(n // 2)]
    if not case["scaled"]:
        return torch.tensor(inv, dtype=torch.float32, device=DEV), 1.0
    factor, trained = 4.0, case["context"] // 4
    at = lambda turns: n * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), n - 1)
    keep = [1.0 - min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(n // 2)]
    inv = [f / factor * (1.0 - m) + f * m for f, m in zip(inv, keep)]
    return torch.tensor(inv, dtype=torch.float32, device=DEV), 0.1 * math.log(factor) + 1.0


def _lengths(case):
    """Keys of every sequence of an ``attn`` case."""
    n, r = case["seqs"], _fixed(case)
    if not case["ragged"]:
        return [case["keys"]] * n
    most = max(1, case["keys"])
    lens = [min(most, int(round(math.exp(r.uniform(0.0, math.log(most + 0.49)))))) for _ in range(n)]
    lens[0] = most
    if n > 4:
        lens[1], lens[2] = 0, 1
    return lens


def _spread(case):
    """(start, count) of the chunk of every row of a ``rope`` case."""
    r, n = _fixed(case), case["rows"]
    if case["decode"]:
        return [(r.randrange(case["context"]), 1) for _ in range(n)]
    cuts = sorted(r.sample(range(1, case["tokens"]), n - 1)) if n > 1 else []
    counts = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    return [(r.randrange(max(1, case["context"] - c)), c) for c in counts]


def _parents(case):
    """Old row that each new row of a ``fork`` case goes on with, and the old rows' lengths: the beams of a group have one prompt."""
    r, w = _fixed(case), case["beams"]
    parents, lens = [], []
    for g in range(case["groups"]):
        keys = case["keys"] if g == 0 else _span(r, 1, case["keys"])
        lens += [keys] * w
        parents += [g * w + p for p in sorted(min(r.randrange(w), r.randrange(w)) for _ in range(w))]
    return parents, lens


def _prepare_rope(case, g):
    dt, ps, D = TYPES[case["dtype"]], case["page"], case["dim"]
    T, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
    spread = _spread(case)
    need = [(s + c - 1) // ps - s // ps + 1 for s, c in spread]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    # pages of earlier positions are of no use to this call: the table does not name them
    table = torch.full((case["rows"], -(-case["context"] // ps)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, (s, c) in enumerate(spread):
        table[i, s // ps : s // ps + need[i]] = order[at : at + need[i]]
        at += need[i]
    # one projection's output, its heads as views
    qkv = _randn(g, T, hq + 2 * hk, D, dtype=dt)
    inv, scale = _frequencies(case)
    kv = _randn(g, 2, pages, hk, ps, D, dtype=dt)
    return {"q": qkv[:, :hq], "k": qkv[:, hq : hq + hk], "v": qkv[:, hq + hk :], "kv": kv, "table": table, "inv": inv, "scale": scale,
            "positions": _ints([s + j for s, c in spread for j in range(c)]), "rows": _ints([i for i, (s, c) in enumerate(spread) for _ in range(c)]),
            "q_norm": 1.0 + _randn(g, D, std=0.1) if case["norm"] else None, "k_norm": 1.0 + _randn(g, D, std=0.1) if case["norm"] else None}


def _prepare_attn(case, g):
    dt, ps, D, n = TYPES[case["dtype"]], case["page"], case["dim"], case["seqs"]
    lens = _lengths(case)
    mix = torch.randperm(n, generator=g, device=DEV).tolist()
    lens = [lens[i] for i in mix]
    need = [-(-x // ps) for x in lens]
    pages, width = sum(need) + 2, max(need) + 1
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32)
    at, host = 0, order.cpu()
    for i, c in enumerate(need):
        table[i, :c] = host[at : at + c]
        at += c
    kv = torch.empty(2, pages, case["kv_heads"], ps, D, dtype=dt, device=DEV)
    kv.normal_(generator=g)
    # slots behind a sequence's end hold what an earlier owner left there
    slopes = (0.5 ** (1 + torch.arange(case["q_heads"], device=DEV) % 8)).float() if case["bias"] else None
    return {"q": _randn(g, n, case["q_heads"], D, dtype=dt, std=2.0), "kv": kv, "table": table.to(DEV), "lens": _ints(lens), "slopes": slopes}


def _pool(case, g, pages):
    kv = torch.empty(case["layers"], 2, pages, case["kv_heads"], case["page"], case["dim"], dtype=TYPES[case["dtype"]], device=DEV)
    return kv.normal_(generator=g)


def _prepare_fork(case, g):
    ps, w = case["page"], case["beams"]
    parents, lens = _parents(case)
    # beams share their prompt's full pages; a page that is begun belongs to one beam each
    whole = [lens[i * w] // ps for i in range(case["groups"])]
    open_ = [1 if lens[i * w] % ps else 0 for i in range(case["groups"])]
    used = sum(whole) + w * sum(open_)
    pages = used + 2 * len(parents) + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.full((len(parents), -(-case["keys"] // ps) + 2), -1, dtype=torch.int32)
    at = 0
    for i in range(case["groups"]):
        table[i * w : (i + 1) * w, : whole[i]] = order[at : at + whole[i]]
        at += whole[i]
        if open_[i]:
            table[i * w : (i + 1) * w, whole[i]] = order[at : at + w]
            at += w
    mix = torch.stack([torch.randperm(w, generator=g, device=DEV) for _ in range(case["groups"])]).cpu()
    parents = [i * w + int(mix[i][p - i * w]) for i in range(case["groups"]) for p in parents[i * w : (i + 1) * w]]
    return {"kv": _pool(case, g, pages), "table": table.to(DEV), "lens": _ints(lens), "parents": _ints(parents)}


def _prepare_compact(case, g):
    n, rows, ps = case["pages"], case["rows"], case["page"]
    live = max(1, int(n * case["live"]))
    order = torch.randperm(n, generator=g, device=DEV)[:live].to(torch.int32).cpu()
    r = _fixed(case)
    cuts = sorted(r.randint(0, live) for _ in range(rows - 1))
    counts = [b - a for a, b in zip([0] + cuts, cuts + [live])]
    table = torch.full((rows, max(counts) + 1), -1, dtype=torch.int32)
    lens, at = [], 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at : at + c]
        lens.append(max(0, c * ps - r.randrange(ps)))
        at += c
    # every third row is a fork of the row before it and shares all its pages
    for i in range(2, rows, 3):
        table[i], lens[i] = table[i - 1].clone(), lens[i - 1]
    return {"kv": _pool(case, g, n), "table": table.to(DEV), "lens": _ints(lens)}


def _prepare_beam(case, g):
    B, W, V = case["batch"], case["beams"], case["vocab"]
    logits = _randn(g, B, W, V, std=2.5).to(TYPES[case["dtype"]])
    scores = -torch.rand(B, W, generator=g, device=DEV) * 6.0 - 2.0
    finished = torch.zeros(B * W, dtype=torch.bool, device=DEV)
    # the first beam of a request goes on
    at = (torch.randperm(B * (W - 1), generator=g, device=DEV)[: case["finished"]] if W > 1 else torch.zeros(0, dtype=torch.int64, device=DEV))
    finished[at // max(1, W - 1) * W + at % max(1, W - 1) + 1] = True
    states = []
    for _ in range(case["states"]):
        states += [_randn(g, B * W, case["state_heads"], 128, 128), _randn(g, B * W, case["state_heads"] * 256, 3)]
    return {"logits": logits, "scores": scores, "finished": finished.view(B, W), "k": case["k"], "eos": V - 2, "beams": W, "states": states,
            "moved": [torch.empty_like(s) for s in states]}


def prepare(case, seed):
    g = _gen(seed)
    state = globals()["_prepare_" + case["kind"]](case, g)
    state["case"] = case
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------------
def _plain_rope(s):
    c = s["case"]
    n, half = c["rotary"], c["rotary"] // 2
    turn = s["positions"].double()[:, None] * s["inv"].double()
    cos, sin = (torch.cos(turn) * s["scale"]).float()[:, None], (torch.sin(turn) * s["scale"]).float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if c["interleaved"]:
            a, b = x[..., 0:n:2], x[..., 1:n:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:n]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([y, x[..., n:]], -1)

    kv, ps = s["kv"], c["page"]
    at = s["positions"].long()
    page, slot = s["table"][s["rows"].long(), at // ps].long(), at % ps
    kv[0].transpose(1, 2)[page, slot] = turned(s["k"], s["k_norm"]).to(kv.dtype)
    kv[1].transpose(1, 2)[page, slot] = s["v"].to(kv.dtype)
    return turned(s["q"], s["q_norm"]).to(kv.dtype)


def _plain_attn(s):
    c = s["case"]
    B, hk, D, ps = c["seqs"], c["kv_heads"], c["dim"], c["page"]
    table = s["table"].long().clamp(min=0)
    K = s["kv"][0][table].permute(0, 2, 1, 3, 4).reshape(B, hk, -1, D).float()
    V = s["kv"][1][table].permute(0, 2, 1, 3, 4).reshape(B, hk, -1, D).float()
    q = s["q"].float().view(B, hk, -1, D)
    x = torch.matmul(q, K.transpose(2, 3)) * D ** -0.5
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    lens = s["lens"].long()[:, None]
    at = torch.arange(K.shape[2], device=DEV)[None]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, hk, -1, 1) * (lens - 1 - at).float()[:, None, None]
    seen = at < lens
    if c["window"]:
        seen = seen & (at >= lens - c["window"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    V = V.masked_fill(~seen[:, None, :, None], 0.0)
    y = torch.matmul(p, V) / torch.where(total == 0.0, 1.0, total)
    lse = torch.where(total == 0.0, -math.inf, top + torch.log(total))
    return y.view(B, -1, D).to(s["q"].dtype), lse.view(B, -1)


def _plain_fork(s):
    ps, kv, parents = s["case"]["page"], s["kv"], s["parents"].long()
    n, pages, width = parents.numel(), kv.shape[2], s["table"].shape[1]
    lens = s["lens"][parents].long()
    used, row = -(-lens // ps), torch.arange(n, device=DEV)
    at = torch.arange(width, device=DEV)[None]
    table = torch.where(at < used[:, None], s["table"][parents].long(), -1)
    count = torch.zeros(pages + 1, dtype=torch.int64, device=DEV)
    count.index_add_(0, torch.where(table < 0, pages, table).view(-1), torch.ones(1, dtype=torch.int64, device=DEV).expand(table.numel()))
    # a begun page that other rows hold is copied, by all but the first where all its holders go on writing
    fill = lens % ps
    last = table.gather(1, (used - 1).clamp(min=0)[:, None])[:, 0]
    open_ = fill > 0
    same = (last[:, None] == last[None]) & open_[:, None] & open_[None]
    held = count[last.clamp(min=0)]
    first = ~(same & (row[None] < row[:, None])).any(1)
    copies = open_ & (held > 1) & ~((same.sum(1) == held) & first)
    grown = lens + 1
    fresh = (copies | (fill == 0)).long()
    free = torch.sort(torch.where(count[:pages] == 0, torch.arange(pages, device=DEV), pages)).values
    taken = free[(torch.cumsum(fresh, 0) - fresh).clamp(max=pages - 1)]
    place = torch.where(fill > 0, used - 1, used)
    table.scatter_(1, place[:, None], torch.where(fresh > 0, taken, table.gather(1, place[:, None])[:, 0])[:, None])
    count.index_add_(0, torch.where(fresh > 0, taken, pages), torch.ones_like(taken))
    count.index_add_(0, torch.where(copies, last, pages), -torch.ones_like(taken))
    src, dst = last.clamp(min=0), torch.where(copies, taken, last.clamp(min=0))
    slot = torch.arange(ps, device=DEV)[:, None] < fill[:, None, None, None]
    kv[:, :, dst] = torch.where(slot & copies[:, None, None, None], kv[:, :, src], kv[:, :, dst])
    return table.to(torch.int32), grown.to(torch.int32), count[:pages].to(torch.int32)


def _plain_compact(s):
    ps, kv, pages = s["case"]["page"], s["kv"], s["kv"].shape[2]
    at = torch.arange(s["table"].shape[1], device=DEV)[None]
    table = torch.where(at < -(-s["lens"].long() // ps)[:, None], s["table"].long(), -1)
    count = torch.zeros(pages + 1, dtype=torch.int64, device=DEV)
    count.index_add_(0, torch.where(table < 0, pages, table).view(-1), torch.ones(1, dtype=torch.int64, device=DEV).expand(table.numel()))
    live = count[:pages] > 0
    n = live.sum()
    page = torch.arange(pages, device=DEV)
    hole, late = ~live & (page < n), live & (page >= n)
    holes = torch.sort(torch.where(hole, page, pages)).values
    rank = torch.cumsum(late.long(), 0) - 1
    to = torch.where(late, holes[rank.clamp(min=0)].clamp(max=pages - 1), page)
    source = torch.zeros(pages, dtype=torch.int64, device=DEV).index_add_(0, to, torch.where(live, page, 0))
    stays = ~(hole & (source > 0))
    kv.copy_(kv[:, :, torch.where(stays, page, source)])
    to = torch.where(live, to, -1)
    table = torch.where(table < 0, -1, to[table.clamp(min=0)])
    count = torch.where(page < n, torch.where(stays, count[:pages], count[source]), 0)
    return table.to(torch.int32), count.to(torch.int32), to.to(torch.int32), n.to(torch.int32).view(1)


def _plain_beam(s):
    x, scores, finished, k = s["logits"], s["scores"].double(), s["finished"], s["k"]
    B, W, V = x.shape
    m = min(k, V)
    lse = torch.logsumexp(x.double(), -1, keepdim=True)
    # within a row the larger logit goes first, then the lower token: one whole number holds both
    bits = (x.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) - torch.arange(V, device=DEV)
    token = order.topk(m, dim=-1).indices
    total = scores[..., None] + (x.double().gather(-1, token) - lse)
    only = torch.arange(m, device=DEV)
    done = finished[..., None]
    total = torch.where(done, torch.where(only == 0, scores[..., None], -math.inf), total)
    token = torch.where(done & (only == 0), s["eos"], token)
    best = torch.sort(total.view(B, -1), dim=-1, descending=True, stable=True)
    at = best.indices[:, :k]
    rows = at // m + W * torch.arange(B, device=DEV)[:, None]
    keep = rows[:, : s["beams"]].reshape(-1)
    moved = [torch.index_select(t, 0, keep) for t in s["states"]]
    return best.values[:, :k].float(), rows.to(torch.int32), token.view(B, -1).gather(1, at).to(torch.int32), moved


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    s, kind = state, state["case"]["kind"]
    if kind == "rope":
        if own:
            from nexrt_b200.ops.rope import rope_append

            q = rope_append(s["q"], s["k"], s["v"], s["positions"], s["rows"], s["kv"][0], s["kv"][1], s["table"], s["inv"], interleaved=s["case"]["interleaved"],
                            scale=s["scale"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        else:
            q = _plain_rope(s)
        return {"q": q, "k_pages": s["kv"][0], "v_pages": s["kv"][1]}
    if kind == "attn":
        if own:
            from nexrt_b200.ops.paged import paged_attention

            out, lse = paged_attention(s["q"], s["kv"][0], s["kv"][1], s["table"], s["lens"], softcap=s["case"]["softcap"], window=s["case"]["window"],
                                       slopes=s["slopes"], return_lse=True)
        else:
            out, lse = _plain_attn(s)
        return {"out": out, "lse": lse}
    if kind == "fork":
        if own:
            from nexrt_b200.ops.paged import fork_pages

            table, lens, refs = fork_pages(s["kv"], s["table"], s["lens"], s["parents"], grow=1)
        else:
            table, lens, refs = _plain_fork(s)
        return {"kv": s["kv"], "table": table, "lens": lens, "refs": refs}
    if kind == "compact":
        if own:
            from nexrt_b200.ops.paged import compact_pages

            table, refs, remap, live = compact_pages(s["kv"], s["table"], s["lens"])
        else:
            table, refs, remap, live = _plain_compact(s)
        return {"kv": s["kv"], "table": table, "refs": refs, "remap": remap, "live": live}
    if own:
        from nexrt_b200.ops.beam import beam_select, reorder_rows

        scores, rows, tokens = beam_select(s["logits"], s["scores"], s["k"], finished=s["finished"], eos=s["eos"])
        moved = reorder_rows(s["states"], rows[:, : s["beams"]], out=s["moved"])
    else:
        scores, rows, tokens, moved = _plain_beam(s)
    return {"scores": scores, "rows": rows, "tokens": tokens, "states": moved}


def work(case):
    kind = case["kind"]
    if kind == "rope":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        values = case["tokens"] * heads * case["dim"]
        return {"bytes": 2 * values * 2 + case["tokens"] * 12 + 2 * case["rotary"] + (8 * case["dim"] if case["norm"] else 0), "flops": 10.0 * values}
    if kind == "attn":
        seen = [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]
        size = case["kv_heads"] * case["dim"] * 2
        entries = sum(-(-n // case["page"]) for n in seen)
        q = case["seqs"] * case["q_heads"]
        return {"bytes": 2 * sum(seen) * size + 4 * entries + q * (case["dim"] * 4 + 4) + 4 * case["seqs"], "flops": 4.0 * sum(seen) * case["q_heads"] * case["dim"]}
    if kind == "fork":
        parents, lens = _parents(case)
        ps = case["page"]
        row = case["layers"] * 2 * case["kv_heads"] * case["dim"] * 2
        used = sum(-(-lens[p] // ps) for p in parents)
        fill = sum(lens[p] % ps for p in parents)
        held = sum(lens[p] % ps for p in set(parents))
        # a begun page of n rows that go on is read once and copied n - 1 times
        many = sum(lens[p] % ps for p in set(parents) if parents.count(p) > 1)
        width = -(-case["keys"] // ps) + 2
        return {"bytes": row * ((fill - held) + many) + 4 * (used + len(parents) * (width + 3)), "flops": used}
    if kind == "compact":
        live = max(1, int(case["pages"] * case["live"]))
        size = case["layers"] * 2 * case["kv_heads"] * case["page"] * case["dim"] * 2
        # of `live` pages spread evenly, those behind the first `live` places move
        moved = live * (case["pages"] - live) / case["pages"]
        return {"bytes": 2 * moved * size + 8 * live + 8 * case["pages"], "flops": case["pages"]}
    rows = case["batch"] * case["beams"]
    state = case["states"] * case["state_heads"] * (128 * 128 + 256 * 3) * 4
    size = 4 if case["dtype"] == "fp32" else 2
    # about two thirds of the beams of a request go on
    return {"bytes": (rows - case["finished"]) * case["vocab"] * size + rows * state * 5 // 3, "flops": 4.0 * rows * case["vocab"]}


# ---- the same in 64 bits, row by row ------------------------------------------------------------------------------------
def _exact_rope(c, s):
    kv = s["kv"].double()
    pos = s["positions"].double()
    ang = pos.view(-1, 1) * s["inv"].double().view(1, -1)
    z = torch.polar(torch.full_like(ang, s["scale"]), ang).unsqueeze(1)

    def go(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
        n = c["rotary"]
        if c["interleaved"]:
            pairs = torch.view_as_complex(x[..., :n].contiguous().unflatten(-1, (-1, 2))) * z
            return torch.cat([torch.view_as_real(pairs).flatten(-2), x[..., n:]], -1)
        pairs = torch.complex(x[..., : n // 2].contiguous(), x[..., n // 2 : n].contiguous()) * z
        return torch.cat([pairs.real, pairs.imag, x[..., n:]], -1)

    k, v = go(s["k"], s["k_norm"]), s["v"].double()
    table, rows, ps = s["table"].tolist(), s["rows"].tolist(), c["page"]
    flat = torch.tensor([table[r][p // ps] * ps + p % ps for r, p in zip(rows, s["positions"].tolist())], device=DEV)
    for plane, x in ((0, k), (1, v)):
        for h in range(c["kv_heads"]):
            line = kv[plane, :, h].reshape(-1, c["dim"])
            line[flat] = x[:, h]
            kv[plane, :, h] = line.view(-1, ps, c["dim"])
    return {"q": go(s["q"], s["q_norm"]), "k_pages": kv[0], "v_pages": kv[1]}


def _exact_attn(c, s):
    out = torch.zeros(c["seqs"], c["q_heads"], c["dim"], dtype=torch.float64, device=DEV)
    lse = torch.full((c["seqs"], c["q_heads"]), -math.inf, dtype=torch.float64, device=DEV)
    lens, ps, per = s["lens"].tolist(), c["page"], c["q_heads"] // c["kv_heads"]
    for b, n in enumerate(lens):
        lo = max(0, n - c["window"]) if c["window"] else 0
        if n <= lo:
            continue
        pages = s["table"][b, : -(-n // ps)].long()
        dist = torch.arange(n - 1 - lo, -1, -1, dtype=torch.float64, device=DEV)
        for h in range(c["kv_heads"]):
            K = s["kv"][0][pages, h].reshape(-1, c["dim"])[lo:n].double()
            V = s["kv"][1][pages, h].reshape(-1, c["dim"])[lo:n].double()
            x = s["q"][b, h * per : (h + 1) * per].double() @ K.T / math.sqrt(c["dim"])
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            if s["slopes"] is not None:
                x = x - s["slopes"][h * per : (h + 1) * per].double()[:, None] * dist
            lse[b, h * per : (h + 1) * per] = torch.logsumexp(x, -1)
            out[b, h * per : (h + 1) * per] = torch.softmax(x, -1) @ V
    return {"out": out, "lse": lse}


def _held(table, lens, ps):
    count = {}
    for row, n in zip(table, lens):
        for p in row[: -(-n // ps)]:
            count[p] = count.get(p, 0) + 1
    return count


def _exact_fork(c, s):
    ps, kv = c["page"], s["kv"].double()
    old, parents, lens = s["table"].tolist(), s["parents"].tolist(), s["lens"].tolist()
    lens = [lens[p] for p in parents]
    table = [old[p][: -(-n // ps)] for p, n in zip(parents, lens)]
    count = _held(table, lens, ps)
    begun = {}
    for r, n in enumerate(lens):
        if n % ps:
            begun.setdefault(table[r][-1], []).append(r)
    free = iter([p for p in range(kv.shape[2]) if p not in count])
    new = dict(count)
    for r, n in enumerate(lens):
        if n % ps == 0:
            table[r].append(next(free))
            new[table[r][-1]] = 1
            continue
        p = table[r][-1]
        if count[p] == 1 or (len(begun[p]) == count[p] and begun[p][0] == r):
            continue
        to = next(free)
        kv[:, :, to, :, : n % ps] = s["kv"][:, :, p, :, : n % ps].double()
        table[r][-1], new[to], new[p] = to, 1, new[p] - 1
    width = len(old[0])
    return {"kv": kv, "table": _ints([t + [-1] * (width - len(t)) for t in table]), "lens": _ints([n + 1 for n in lens]),
            "refs": _ints([new.get(p, 0) for p in range(kv.shape[2])])}


def _exact_compact(c, s):
    old, lens, ps = s["table"].tolist(), s["lens"].tolist(), c["page"]
    count = _held(old, lens, ps)
    n, pages = len(count), s["kv"].shape[2]
    holes = iter([p for p in range(n) if p not in count])
    to = {p: p if p < n else next(holes) for p in sorted(count)}
    kv = s["kv"].double()
    for p, q in to.items():
        if p != q:
            kv[:, :, q] = s["kv"][:, :, p].double()
    refs = [0] * pages
    for p, q in to.items():
        refs[q] = count[p]
    table = [[to[p] if j < -(-m // ps) else -1 for j, p in enumerate(row)] for row, m in zip(old, lens)]
    return {"kv": kv, "table": _ints(table), "refs": _ints(refs), "remap": _ints([to.get(p, -1) for p in range(pages)]), "live": _ints([n])}


def _exact_beam(c, s):
    scores, rows, tokens = [], [], []
    B, W, V = s["logits"].shape
    done, past = s["finished"].tolist(), s["scores"].double().tolist()
    for b in range(B):
        found = []
        for w in range(W):
            if done[b][w]:
                found.append((-past[b][w], w, s["eos"]))
                continue
            p = torch.log_softmax(s["logits"][b, w].double(), -1) + past[b][w]
            edge = p.topk(min(s["k"], V)).values[-1]
            at = (p >= edge).nonzero().view(-1)
            found += [(-v, w, t) for v, t in zip(p[at].tolist(), at.tolist())]
        found = sorted(found)[: s["k"]]
        scores.append([-f[0] for f in found])
        rows.append([b * W + f[1] for f in found])
        tokens.append([f[2] for f in found])
    keep = [r for row in rows for r in row[:W]]
    return {"scores": torch.tensor(scores, dtype=torch.float64, device=DEV), "rows": _ints(rows), "tokens": _ints(tokens),
            "states": [t[torch.tensor(keep, device=DEV)].double() for t in s["states"]]}


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))
