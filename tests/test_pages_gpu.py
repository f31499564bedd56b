"""Pages of a shared cache: forking, freeing, growing, copying and compacting against a statement in plain Python, full pools and tables, bad entries,
and a random walk of a cache whose contents are followed token by token."""

import random

import pytest
import torch

from nexrt_b200.ops.lib import KernelError
from nexrt_b200.ops.paged import PagedCache, compact_pages, copy_pages, fork_pages
from nexrt_b200.runtime.capture import graph_capture
from nexrt_b200.runtime.control import Status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def held(table, lens, page):
    count = {}
    for row, n in zip(table, lens):
        for p in row[: -(-n // page)]:
            count[p] = count.get(p, 0) + 1
    return count


def fork_in_python(kv, table, lens, parents, grow, page):
    """(kv, table, lens, refs, short): ``short`` - a row did not get its pages."""
    pages, width = kv.shape[2], len(table[0]) if table else 0
    new = [table[p][: -(-lens[p] // page)] if p >= 0 else [] for p in parents]
    n = [lens[p] if p >= 0 else 0 for p in parents]
    count = held(new, n, page)
    short, want, open_ = False, [0] * len(n), [None] * len(n)
    g = [x if p >= 0 else 0 for x, p in zip(grow, parents)]
    for r in range(len(n)):
        if g[r] > 0 and n[r] + g[r] > width * page:
            g[r], short = 0, True
        if g[r] > 0:
            want[r] = -(-(n[r] + g[r]) // page) - len(new[r])
            open_[r] = new[r][-1] if n[r] % page else None
    copies = [o is not None and count[o] > 1 and not (open_.count(o) == count[o] and open_.index(o) == r) for r, o in enumerate(open_)]
    free = [p for p in range(pages) if p not in count]
    refs, out, at = dict(count), kv.clone(), 0
    for r in range(len(n)):
        k = want[r] + copies[r]
        mine, at = free[at : at + k], at + k
        if len(mine) < k:
            g[r], short = 0, True
            continue
        if copies[r]:
            p = mine.pop(0)
            out[:, :, p, :, : n[r] % page] = kv[:, :, open_[r], :, : n[r] % page]
            new[r][-1], refs[p] = p, 1
            refs[open_[r]] -= 1
        for p in mine:
            new[r].append(p)
            refs[p] = 1
    return out, [t + [-1] * (width - len(t)) for t in new], [a + b for a, b in zip(n, g)], [refs.get(p, 0) for p in range(pages)], short


def random_rows(r, rows, width, pages, page):
    """A table with shared prefixes, as forks leave it, and rows of any length."""
    table, lens = [], []
    free = list(range(pages))
    r.shuffle(free)
    for i in range(rows):
        if table and r.random() < 0.5:
            j = r.randrange(i)
            n = r.randint(0, lens[j])
            t = table[j][: -(-n // page)]
        else:
            n = min(r.choice([0, 1, page - 1, page, page + 1, r.randint(0, width * page)]), width * page, len(free) * page)
            t = [free.pop() for _ in range(-(-n // page))]
        table.append(t)
        lens.append(n)
    return [t + [-1] * (width - len(t)) for t in table], lens


@pytest.mark.parametrize("seed", range(24))
def test_fork_is_its_statement(seed):
    r = random.Random(seed)
    page, rows, width, heads, dim = r.choice([1, 2, 16, 5]), r.randint(1, 40), r.randint(1, 12), r.choice([1, 3]), r.choice([64, 128])
    pages = r.choice([rows * width * 2 + 5, max(4, rows * width // 3)])
    table, lens = random_rows(r, rows, width, pages, page)
    n = r.choice([rows, 1, rows * 3])
    parents = [r.choice([-1, r.randrange(rows), r.randrange(rows)]) for _ in range(n)]
    grow = r.choice([[1] * n, [0] * n, [r.randint(0, 2 * page + 1) for _ in range(n)]])
    dtype = r.choice([torch.bfloat16, torch.float32, torch.int8])
    kv = torch.randint(-100, 100, (r.randint(1, 3), 2, pages, heads, page, dim), device=DEV).to(dtype)
    want = fork_in_python(kv, table, lens, parents, grow, page)
    status = ints([0])
    t, l, refs = fork_pages(kv, ints(table), ints(lens), ints(parents), grow[0] if len(set(grow)) == 1 else ints(grow), status=status)
    assert t.tolist() == want[1] and l.tolist() == want[2] and refs.tolist() == want[3]
    assert torch.equal(kv, want[0]) and int(status) == (Status.NO_PAGES if want[4] else 0)


def test_fork_of_many_rows_and_a_wide_table():
    r = random.Random(1)
    page, rows, width = 2, 2500, 600
    pages = 30000
    table, lens = random_rows(r, 40, width, pages, page)
    parents = [r.randrange(40) for _ in range(rows)]
    kv = torch.randint(-100, 100, (1, 2, pages, 1, page, 16), device=DEV).to(torch.int8)
    want = fork_in_python(kv, table, lens, parents, [1] * rows, page)
    t, l, refs = fork_pages(kv, ints(table), ints(lens), ints(parents), 1)
    assert t.tolist() == want[1] and l.tolist() == want[2] and refs.tolist() == want[3] and torch.equal(kv, want[0])


@pytest.mark.parametrize("rows,width", [(9, 7), (33, 3), (256, 3), (257, 3), (700, 5), (700, 9)])
def test_begun_pages_that_many_rows_hold(rows, width):
    """Groups of rows on one begun page, all of which write on, or some; tables that the planning kernel counts itself, by rows and by entries, and
    one that it does not."""
    r = random.Random(rows + width)
    page, table, lens, at = 4, [], [], 0
    while len(table) < rows:
        n = r.choice([0, 3, page, page + 1, 2 * page + 3])
        used, many = -(-n // page), min(r.choice([1, 2, 40]), rows - len(table))
        table += [list(range(at, at + used)) + [-1] * (width - used)] * many
        lens += [n] * many
        at += used
    pages = at + 2 * rows
    kv = torch.randint(-100, 100, (1, 2, pages, 1, page, 16), device=DEV).to(torch.int8)
    for grow in ([1] * rows, [r.choice([0, 1, 1, 2]) for _ in range(rows)]):
        a = kv.clone()
        want = fork_in_python(a, table, lens, list(range(rows)), grow, page)
        status = ints([0])
        t, l, refs = fork_pages(a, ints(table), ints(lens), ints(range(rows)), ints(grow), status=status)
        assert t.tolist() == want[1] and l.tolist() == want[2] and refs.tolist() == want[3] and torch.equal(a, want[0])
        assert int(status) == (Status.NO_PAGES if want[4] else 0)


def test_outputs_beside_the_inputs_in_one_allocation():
    """Disjoint parts of one buffer are outputs like any others."""
    kv = torch.zeros(1, 2, 8, 1, 4, 64, dtype=torch.bfloat16, device=DEV)
    work = torch.full((40,), -7, dtype=torch.int32, device=DEV)
    table, lens, out, lens_out, refs = work[:4].view(2, 2), work[4:6], work[6:10].view(2, 2), work[10:12], work[12:20]
    table.copy_(ints([[3, 5], [-1, -1]]))
    lens.copy_(ints([6, 0]))
    fork_pages(kv, table, lens, ints([0, 0]), 0, table_out=out, lens_out=lens_out, refs=refs)
    assert work[:22].tolist() == [3, 5, -1, -1, 6, 0, 3, 5, 3, 5, 6, 6, 0, 0, 0, 2, 0, 2, 0, 0, -7, -7]
    compact_pages(kv, out, lens_out, table_out=table, refs=refs)
    assert table.tolist() == [[0, 1], [0, 1]]
    for bad in (dict(table_out=work[2:6].view(2, 2)), dict(lens_out=work[5:7]), dict(refs=work[5:13]), dict(lens_out=work[20:22], refs=work[21:29])):
        with pytest.raises(ValueError, match="shares memory"):
            fork_pages(kv, table, lens, ints([0, 0]), 0, **bad)


def test_fork_reports_and_survives_bad_input():
    kv = torch.zeros(1, 2, 6, 1, 4, 64, dtype=torch.bfloat16, device=DEV)

    def run(table, lens, parents, grow=0):
        status = ints([0])
        t, l, refs = fork_pages(kv, ints(table), ints(lens), ints(parents), grow, status=status)
        return t.tolist(), l.tolist(), refs.tolist(), int(status)

    assert run([[0, 1]], [8], [5, 0]) == ([[-1, -1], [0, 1]], [0, 8], [1, 1, 0, 0, 0, 0], Status.BAD_PAGE)          # a parent that does not exist
    assert run([[0, 6]], [8], [0]) == ([[0, -1]], [8], [1, 0, 0, 0, 0, 0], Status.BAD_PAGE)                          # a page that does not exist
    assert run([[0, -9]], [7], [0], 1) == ([[0, -1]], [7], [1, 0, 0, 0, 0, 0], Status.BAD_PAGE)                      # ... and is written next: the row stays
    assert run([[0, 1]], [9], [0]) == ([[0, 1]], [8], [1, 1, 0, 0, 0, 0], Status.BAD_PAGE)                           # longer than the table
    assert run([[0, 1]], [8], [0], 1) == ([[0, 1]], [8], [1, 1, 0, 0, 0, 0], Status.NO_PAGES)                        # no column left
    assert run([[0, 1]], [2**31 - 1], [0], 2**31 - 1)[1] == [8]
    assert run([[0]], [-3], [0], 0) == ([[-1]], [0], [0] * 6, 0)
    assert run([[0]], [4], []) == ([], [], [0] * 6, 0)
    full = run([[0, 1, 2, 3, 4, 5]], [24], [0, -1])
    assert full == ([[0, 1, 2, 3, 4, 5], [-1] * 6], [24, 0], [1] * 6, 0)
    assert run([[0, 1, 2, 3, 4, 5], [-1] * 6], [24, 0], [0, 1], ints([0, 1]))[1:] == ([24, 0], [1] * 6, Status.NO_PAGES)   # the pool is full


def test_a_length_that_32_bits_do_not_hold_is_refused():
    """A table with room for more positions than an int32 counts."""
    kv = torch.zeros(1, 2, 3, 1, 65536, 16, dtype=torch.int8, device=DEV)
    table, status = torch.zeros(1, 40000, dtype=torch.int32, device=DEV), ints([0])
    t, l, refs = fork_pages(kv, table, ints([2**31 - 65536]), ints([0]), 65535, status=status)
    assert l.tolist() == [2**31 - 1] and int(status) == 0 and refs.tolist() == [32767, 1, 0]
    t, l, refs = fork_pages(kv, table, ints([2**31 - 65536]), ints([0]), 65536, status=status)
    assert l.tolist() == [2**31 - 65536] and int(status) == Status.NO_PAGES and refs.tolist() == [32767, 0, 0]


@pytest.mark.parametrize("seed", range(16))
def test_compact_is_its_statement(seed):
    r = random.Random(100 + seed)
    page, rows, width = r.choice([1, 4, 16]), r.randint(1, 30), r.randint(1, 40)
    pages = r.choice([rows * width + 3, rows * width * 5 + 9000 * (seed % 2)])
    table, lens = random_rows(r, rows, width, pages, page)
    kv = torch.randint(-100, 100, (r.randint(1, 2), 2, pages, r.choice([1, 2]), page, 64), device=DEV).to(torch.int8)
    count = held(table, lens, page)
    live = len(count)
    holes = iter([p for p in range(live) if p not in count])
    to = {p: p if p < live else next(holes) for p in sorted(count)}
    want = kv.clone()
    for p, q in to.items():
        want[:, :, q] = kv[:, :, p]
    dirty = [[p if j < -(-n // page) else r.choice([-1, 0, 10**6]) for j, p in enumerate(row)] for row, n in zip(table, lens)]   # behind the last page: anything
    status = ints([0])
    t, refs, remap, n = compact_pages(kv, ints(dirty), ints(lens), status=status)
    assert t.tolist() == [[to[p] if p >= 0 else -1 for p in row] for row in table] and int(n) == live and int(status) == 0
    assert remap.tolist() == [to.get(p, -1) for p in range(pages)]
    back = {q: p for p, q in to.items()}
    assert refs.tolist() == [count[back[p]] if p in back else 0 for p in range(pages)]
    assert torch.equal(kv, want)


def test_copy_pages():
    kv = torch.randint(-100, 100, (3, 2, 50, 2, 7, 64), device=DEV).to(torch.bfloat16)

    def run(src, dst):
        a, status = kv.clone(), ints([0])
        copy_pages(a, ints(src), ints(dst), status=status)
        return a, int(status)

    a, code = run([3, 4, 3, -1, 9, 11], [40, 41, 42, 0, -1, 11])
    want = kv.clone()
    want[:, :, [40, 41, 42]] = kv[:, :, [3, 4, 3]]
    assert code == 0 and torch.equal(a, want)
    a, code = run([3, 50, 4], [40, 41, 1000])
    want = kv.clone()
    want[:, :, 40] = kv[:, :, 3]
    assert code == Status.BAD_PAGE and torch.equal(a, want)
    a, code = run([3, 4, 40, 5], [40, 41, 42, 41])                # 40 is a source too; 41 is given twice
    want = kv.clone()
    want[:, :, 42], want[:, :, 41] = kv[:, :, 40], kv[:, :, 5]
    assert code == Status.PAGE_CONFLICT and torch.equal(a, want)
    assert torch.equal(run([], [])[0], kv)


@pytest.mark.parametrize("n", [31, 1000, 1025, 6000])
def test_long_lists_of_copies(n):
    """Sources and targets at random, some of them both, given twice, left out or beyond the pool."""
    r = random.Random(n)
    pages = 3 * n
    src = [r.choice([r.randrange(n), r.randrange(n), r.randrange(pages), -1, pages + r.randrange(3)]) if r.random() < 0.3 else r.randrange(n) for _ in range(n)]
    dst = [r.choice([r.randrange(n), -2, pages]) if r.random() < 0.1 else n + r.randrange(2 * n) for _ in range(n)]
    src[5] = dst[5] = 7
    kv = torch.randint(-100, 100, (1, 2, pages, 1, 1, 16), device=DEV).to(torch.int8)
    want, told = kv.clone(), set()
    pairs = [(s, d) for s, d in zip(src, dst) if s >= 0 and d >= 0 and s != d]
    sources, last = {s for s, _ in pairs}, {d: i for i, (_, d) in enumerate(pairs)}
    for i, (s, d) in enumerate(pairs):
        if s >= pages or d >= pages:
            told.add(Status.BAD_PAGE)
        elif d in sources or last[d] != i:
            told.add(Status.PAGE_CONFLICT)
        else:
            want[:, :, d] = kv[:, :, s]
    status = ints([0])
    copy_pages(kv, ints(src), ints(dst), status=status)
    assert torch.equal(kv, want) and int(status) in (told or {0})


def test_offsets_beyond_32_bits():
    """Planes of 2.6 GB, so that pages at the end start beyond 2^32 bytes."""
    kv = torch.empty(1, 2, 80, 1, 32768, 512, dtype=torch.bfloat16, device=DEV)
    kv[:, :, 79].normal_()
    copy_pages(kv, ints([79]), ints([78]))
    assert torch.equal(kv[:, :, 78], kv[:, :, 79])
    t, refs, remap, live = compact_pages(kv, ints([[79]]), ints([32768]))
    assert t.tolist() == [[0]] and torch.equal(kv[:, :, 0], kv[:, :, 79])


@pytest.mark.parametrize("seed", range(4))
def test_a_cache_followed_token_by_token(seed):
    """Rows fork, grow, are freed and compacted at random; each token's K and V are its number, and every row has to read back its own tokens."""
    r = random.Random(seed)
    page, rows, width = r.choice([1, 3, 8]), 9, 12
    cache = PagedCache(2, 60 if page == 1 else 40, 1, page, 64, rows, width * page)
    tokens, counter = [[] for _ in range(rows)], 0
    inv = torch.zeros(0, device=DEV)
    for step in range(60):
        parents = [r.choice([i, i, i, r.randrange(rows), -1]) for i in range(rows)]
        grow = [r.choice([0, 1, 1, 3]) for _ in range(rows)]
        cache.fork(ints(parents), ints(grow))
        lens, old = cache.lens.tolist(), tokens
        tokens = []
        for i, p in enumerate(parents):
            before = list(old[p]) if p >= 0 else []
            assert lens[i] in (len(before), len(before) + (grow[i] if p >= 0 else 0))
            new = lens[i] - len(before)
            tokens.append(before + list(range(counter, counter + new)))
            counter += new
        at = [(i, j) for i in range(rows) for j in range(len(tokens[i])) if tokens[i][j] >= counter - sum(grow) and j >= len(old[parents[i]] if parents[i] >= 0 else [])]
        if at:
            for layer in range(2):
                x = torch.tensor([float(tokens[i][j] % 199 + layer) for i, j in at], device=DEV)[:, None, None].expand(-1, 1, 64).to(torch.bfloat16).contiguous()
                cache.append(layer, x, x, -x, ints([j for _, j in at]), ints([i for i, _ in at]), inv)
        if r.random() < 0.2:
            live = int(cache.compact())
            assert live == int((cache.refs > 0).sum()) and not cache.refs[live:].any()
        table, refs = cache.table.tolist(), cache.refs.tolist()
        assert refs == [held(table, lens, page).get(p, 0) for p in range(len(refs))]
        for i in range(rows):
            for layer in range(2):
                for j, t in enumerate(tokens[i]):
                    slot = cache.kv[layer, :, table[i][j // page], 0, j % page, 0].tolist() if step % 10 == 9 else None
                    assert slot is None or slot == [t % 199 + layer, -(t % 199 + layer)], (step, i, j)
    if int(cache.status) not in (0, Status.NO_PAGES):
        cache.check()


def test_check_raises_what_was_latched():
    cache = PagedCache(1, 2, 1, 4, 64, 2, 40)
    cache.fork(grow=4)
    cache.check()
    cache.fork(grow=1)
    assert cache.lens.tolist() == [4, 4]
    with pytest.raises(KernelError, match="NO_PAGES"):
        cache.check()


def test_a_captured_step_goes_on_from_replay_to_replay():
    cache, twin = (PagedCache(1, 30, 1, 4, 64, 3, 64) for _ in range(2))
    parents = ints([0, 1, 2])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        cache.fork(parents, 1)
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph, st):
        cache.fork(parents, 1)
    twin.fork(parents, 1)
    for p in ([0, 0, 1], [2, 1, 0], [0, -1, 0], [0, 1, 2], [0, 0, 0]):
        parents.copy_(ints(p))
        graph.replay()
        twin.fork(parents, 1)
        assert torch.equal(cache.table, twin.table) and torch.equal(cache.lens, twin.lens) and torch.equal(cache.refs, twin.refs)
    cache.check()


def test_an_engine_prefill_becomes_rows_of_a_cache():
    """The engine prefills one prompt; its keys and values go into a paged row, three beams fork it, and each attends like the engine's own cache."""
    from nexrt_b200.models.reference import synthetic_prompt
    from nexrt_b200.ops.paged import paged_attention
    from nexrt_b200.testing import make_engine, shrunk_checkpoint

    cfg, ckpt = shrunk_checkpoint(0)
    eng = make_engine(cfg, ckpt)
    prompt = synthetic_prompt(cfg.vocab, 37, seed=3)
    eng.prefill(prompt)
    state = eng.export_state()
    full = [x for x in state["layers"].values() if x["kind"] == "full"]
    L, nk, hd = state["L"], cfg.n_kv_heads, cfg.head_dim
    cache = PagedCache(len(full), 30, nk, 8, hd, 3, 64)
    cache.fork(grow=ints([L, 0, 0]))
    for i, x in enumerate(full):
        cache.load_kv(i, 0, x["k_cache"], x["v_cache"])
    cache.fork(ints([0, 0, 0]))
    cache.check()
    assert cache.lens.tolist() == [L] * 3 and int((cache.refs > 0).sum()) == -(-L // 8)
    q = torch.randn(3, cfg.n_q_heads, hd, device=DEV).to(torch.bfloat16)
    for i, x in enumerate(full):
        assert torch.equal(cache.kv[i, 0][cache.table[1, : -(-L // 8)].long()].transpose(0, 1).reshape(nk, -1, hd)[:, :L], x["k_cache"])
        whole = torch.stack([x["k_cache"], x["v_cache"]])[:, None].contiguous()       # the engine's cache as one page of L slots
        want = paged_attention(q, whole[0], whole[1], torch.zeros(3, 1, dtype=torch.int32, device=DEV), cache.lens)
        got = cache.attend(i, q)
        # both are within half a step (2^-8) and the sums' own error of the same numbers; the two splits of the keys differ
        assert torch.all((got.float() - want.float()).abs() <= 2.0**-7 * want.float().abs() + 2.0**-10)
    with pytest.raises(ValueError):
        cache.load_kv(0, 3, full[0]["k_cache"], full[0]["v_cache"])


def test_load_kv_under_another_default_type():
    cache = PagedCache(1, 4, 1, 4, 64, 1, 8)
    k = torch.randn(1, 6, 64, device=DEV).to(torch.bfloat16)
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        cache.fork(grow=6)
        cache.load_kv(0, 0, k, -k)
    finally:
        torch.set_default_dtype(before)
    cache.check()
    got = cache.kv[0][:, cache.table[0].long()].reshape(2, 8, 64)[:, :6]
    assert torch.equal(got[0], k[0]) and torch.equal(got[1], -k[0])


@pytest.mark.parametrize("seed", range(6))
def test_rows_that_grew(seed):
    """``grown`` names the rows that got their positions: not those that are freed, bad, did not ask, or found no page or column."""
    r = random.Random(50 + seed)
    page, rows, width = r.choice([1, 4, 7]), r.choice([5, 31, 200]), r.randint(1, 6)
    pages = max(4, rows * width // 3)
    table, lens = random_rows(r, rows, width, pages, page)
    parents = [r.choice([-1, rows + 3, r.randrange(rows), r.randrange(rows), r.randrange(rows)]) for _ in range(rows)]
    grow = [r.choice([-2, 0, 1, 1, page + 1]) for _ in range(rows)]
    kv = torch.zeros(1, 2, pages, 1, page, 64, dtype=torch.bfloat16, device=DEV)
    grown = torch.full((rows + 2,), 77, dtype=torch.int32, device=DEV)
    t, l, _ = fork_pages(kv, ints(table), ints(lens), ints(parents), ints(grow), grown=grown[1 : rows + 1])
    before = [lens[p] if 0 <= p < rows else 0 for p in parents]
    assert grown.tolist() == [77] + [i if n > b else -1 for i, (n, b) in enumerate(zip(l.tolist(), before))] + [77]
    fork_pages(kv, ints(table), ints(lens), ints([]), 0, grown=ints([]))
    with pytest.raises(ValueError, match="shares memory"):
        fork_pages(kv, ints(table), l, ints(parents), 0, grown=l)


@pytest.mark.parametrize("n", [6, 4])
def test_a_row_without_a_page_leaves_the_others_alone(n):
    """Two rows go on with one prompt that ends inside a page (6 positions of 4 a page), or fills its page; there is a page for one of them.  What the
    step stores for the other would lie on a position of the prompt that both read.  A third row is freed, which is no fault."""
    cache = PagedCache(2, 2, 1, 4, 64, 3, 40)
    inv = torch.zeros(0, device=DEV)
    line = lambda v: torch.tensor([float(x) for x in v], device=DEV)[:, None, None].expand(-1, 1, 64).to(torch.bfloat16)  # noqa: E731
    cache.fork(grow=ints([n, 0, 0]))
    for layer in range(2):
        cache.append(layer, line(range(n)), line(range(n)), line(range(n)), ints(range(n)), ints([0] * n), inv)
    cache.fork(ints([0, 0, -1]), 0)
    assert cache.grown.tolist() == [-1, -1, -1]
    cache.check()
    cache.fork(ints([0, 1, -1]), 1)
    assert cache.lens.tolist() == [n + 1, n, 0] and cache.grown.tolist() == [0, -1, -1]
    assert int(cache.status) == Status.NO_PAGES
    cache.status.zero_()
    for layer in range(2):
        cache.append(layer, line([50, 60, 70]), line([50, 60, 70]), line([50, 60, 70]), cache.lens - 1, cache.grown, inv)
    cache.check()                                                              # the freed row and the one that waits latch nothing
    for layer in range(2):
        for row, want in ((0, [*range(n), 50]), (1, [*range(n)])):
            got = cache.kv[layer][:, cache.table[row, : -(-len(want) // 4)].long(), 0, :, 0].reshape(2, -1)[:, : len(want)]
            assert got.tolist() == [want, want]


def test_a_cache_goes_on_after_a_raised_status():
    """The status keeps the first code: one that stayed would hide what comes later."""
    cache = PagedCache(1, 2, 1, 4, 64, 2, 40)
    cache.fork(grow=4)
    cache.fork(grow=1)
    with pytest.raises(KernelError, match="NO_PAGES"):
        cache.check()
    cache.check()
    cache.fork(ints([0, -1]), 1)
    cache.check()
    assert cache.lens.tolist() == [5, 0]
    cache.fork(ints([7, 0]))
    with pytest.raises(KernelError, match="BAD_PAGE"):
        cache.check()


def test_the_documented_step():
    """The README's order: room for a prompt, its keys and values, a fork, then append and attend in every layer; a freed row among them."""
    from nexrt_b200.ops.rope import rope_frequencies

    L, layers, W = 11, 3, 8
    cache = PagedCache(layers=layers, pages=64, kv_heads=2, slots=4, dim=64, rows=W, max_len=64)
    inv, scale = rope_frequencies(32, 1e7)
    cache.fork(grow=ints([L] + [0] * (W - 1)))
    state = torch.randn(layers, 2, 2, L, 64, device=DEV).to(torch.bfloat16)
    for layer in range(layers):
        cache.load_kv(layer, 0, state[layer, 0], state[layer, 1])
    for parents in ([0] * 7 + [-1], [3, 3, 2, 0, 5, 5, -1, 0]):
        cache.fork(ints(parents), grow=1)
        for layer in range(layers):
            q, k, v = (torch.randn(W, n, 64, device=DEV) for n in (4, 2, 2))
            q = cache.append(layer, q, k, v, cache.lens - 1, cache.grown, inv.cuda(), scale=scale)
            y = cache.attend(layer, q, softcap=0.0, window=0, slopes=None)
            assert y.shape == (W, 4, 64) and torch.isfinite(y).all()
    cache.check()
    assert cache.lens.tolist() == [L + 2] * 6 + [0, L + 2]
    for layer in range(layers):
        for row in (0, 5, 7):
            got = cache.kv[layer][:, cache.table[row, :4].long()].transpose(1, 2).reshape(2, 2, 16, 64)[:, :, :L]
            assert torch.equal(got, state[layer])


@pytest.mark.parametrize("seed", range(6))
def test_every_row_after_every_step(seed):
    """The walk of a cache by its documented step (positions ``lens - 1``, rows ``grown``) in a pool that runs full: after each step all rows read back
    their own tokens in all layers, and each status is the one that the step earns."""
    r = random.Random(200 + seed)
    page, rows, width, layers = r.choice([1, 3, 8]), 7, 6, 2
    cache = PagedCache(layers, r.choice([20, 30]), 2, page, 64, rows, width * page)
    inv, tokens, counter, full = torch.zeros(0, device=DEV), [[] for _ in range(rows)], 0, 0
    for step in range(80):
        parents = [r.choice([i, i, i, r.randrange(rows), -1]) for i in range(rows)]
        grow = [r.choice([0, 1, 1, 1]) for _ in range(rows)]
        cache.fork(ints(parents), ints(grow))
        lens, grown = cache.lens.tolist(), cache.grown.tolist()
        old, tokens = tokens, []
        for i, p in enumerate(parents):
            before = list(old[p]) if p >= 0 else []
            assert grown[i] == (i if lens[i] > len(before) else -1) and lens[i] - len(before) in (0, grow[i])
            tokens.append(before + ([counter + i] if grown[i] >= 0 else []))
        short = any(p >= 0 and g > 0 and n < 0 for p, g, n in zip(parents, grow, grown))
        assert int(cache.status) == (Status.NO_PAGES if short else 0), step
        cache.status.zero_()
        full += short
        number = torch.arange(counter, counter + rows, device=DEV) % 199
        for layer in range(layers):
            x = (number + layer).float()[:, None, None].expand(-1, 2, 64).to(torch.bfloat16).contiguous()
            x[:, 1] += 1
            cache.append(layer, x, x, -x, cache.lens - 1, cache.grown, inv)
        counter += rows
        if r.random() < 0.2:
            live = int(cache.compact())
            assert live == int((cache.refs > 0).sum()) and not cache.refs[live:].any()
        assert int(cache.status) == 0, step
        table, refs = cache.table.tolist(), cache.refs.tolist()
        assert refs == [held(table, lens, page).get(p, 0) for p in range(len(refs))]
        pool = cache.kv[..., 0].float().cpu()                                  # [layers, 2, pages, heads, slots]
        for i in range(rows):
            for j, t in enumerate(tokens[i]):
                for layer in range(layers):
                    want = [float(t % 199 + layer + h) for h in range(2)]
                    assert pool[layer, :, table[i][j // page], :, j % page].tolist() == [want, [-w for w in want]], (step, i, j)
    assert full > 5 or page > 1                                                # (of one position a page the pool runs out all the time)
