"""Beam search over a paged cache: the selection against its definition in 64 bits, the reordering of slots against a
model of the tables on the host, and a whole search on caches of both kinds against one that keeps every beam's history.

A selected score is off by the rounding to fp32 (2^-24 of it) and by its beam's log z. Each of z's terms is off by 2^-23
(|x - m| log2 e + 2) (the argument's roundings and the exponential's), its sum by 2^-24 for each of the adds on a
term's way (vocab / 256 / 4 in a thread, a few to join), all relative; log z is off by the sum. With |x - m| at most 40 where
a term counts (e^-40 of 10^6 terms is 10^-11) this is at most (60 + vocab / 1024 + 20) 2^-23: 2.5e-5 for 131071."""
import math
import random

import pytest
import torch

import kv4_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def H():
    assert torch.cuda.is_available()
    import hesa_cuda
    hesa_cuda.lib()
    hesa_cuda.clear_device_status()
    return hesa_cuda


def select(logits, scores, width, ended=None):
    """(scores in 64 bits, parents, tokens) by sorting every candidate on the host."""
    x = logits.double().cpu()
    n, vocab = x.shape
    out = []
    for r0 in range(0, n, width):
        cand = []
        for b in range(width):
            s = float(scores[r0 + b])
            bad = math.isnan(s) or s == math.inf
            if ended is not None and int(ended[r0 + b]):
                cand.append((-math.inf if bad else s, b, 0, -1, math.nan if bad else s))
                continue
            row = x[r0 + b]
            if s != -math.inf and (bool(torch.isnan(row).any()) or bool((row == math.inf).any())):
                bad = True
            if bad or s == -math.inf:
                cand += [(-math.inf, b, i, i, math.nan if bad else s) for i in range(min(width, vocab))]
                continue
            m = float(row.max())
            lp = torch.full_like(row, -math.inf) if m == -math.inf else s + (row - m) - torch.log(torch.exp(row - m).sum())
            order = torch.sort(row, descending=True, stable=True).indices[:width]
            cand += [(float(lp[t]), b, i, int(t), float(lp[t])) for i, t in enumerate(order)]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        out += cand[:width]
    return torch.tensor([c[4] for c in out], dtype=torch.float64), [c[1] for c in out], [c[3] for c in out]


def check(H, logits, scores, width, ended=None, **kw):
    want, par, tok = select(logits, scores.cpu(), width, None if ended is None else ended.cpu())
    got, gp, gt = H.beam_select(logits, scores, width, ended=ended, **kw)
    assert gp.tolist() == par and gt.tolist() == tok
    got = got.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
    tol = (80 + logits.shape[1] / 1024) * 2.0 ** -23 + 2.0 ** -24 * want[fin].abs()
    assert bool(((got - want)[fin].abs() <= tol).all())
    return got


@pytest.mark.parametrize("n_seq,width,vocab", [(1, 1, 1), (1, 4, 32000), (3, 5, 7), (2, 8, 3), (1, 32, 131071), (5, 32, 40), (40, 6, 1003), (1, 2, 262144),
                                               (2, 3, 1023), (130, 8, 517), (1, 32, 1), (300, 2, 2050)])
@pytest.mark.parametrize("ends", [False, True])
def test_select(H, n_seq, width, vocab, ends):
    g = torch.Generator(device="cuda").manual_seed(vocab + width)
    x = torch.randn(n_seq * width, vocab, generator=g, device="cuda") * 3
    scores = -torch.rand(n_seq * width, generator=g, device="cuda") * 5
    ended = (torch.rand(n_seq * width, generator=g, device="cuda") < 0.3).int() if ends else None
    check(H, x, scores, width, ended)
    assert H.device_status() == 0


def test_ruled_out_dead_and_unsound_beams(H):
    g = torch.Generator(device="cuda").manual_seed(7)
    for vocab in (3, 70, 5000):
        x = torch.randn(8 * 4, vocab, generator=g, device="cuda") * 2
        scores = -torch.rand(32, generator=g, device="cuda")
        ended = torch.zeros(32, dtype=torch.int32, device="cuda")
        scores[1:4] = -math.inf                # a search that begins
        x[4, 1:] = -math.inf                   # one token left
        x[5] = -math.inf                       # none
        scores[6] = -math.inf
        x[8, vocab // 2] = math.nan
        x[9, 0] = math.inf
        scores[10], scores[11] = math.nan, math.inf
        ended[12:16] = 1                       # all have ended
        ended[16], scores[16] = 1, math.nan
        ended[17], scores[17] = -7, -math.inf
        x[16] = math.nan                       # not looked at
        scores[18] = -math.inf
        x[18] = math.nan                       # not looked at
        scores[20:24] = -math.inf              # all dead
        x[24:28] = 1.5                         # ties within and between beams
        scores[24:28] = -1.0
        x[28:32] = torch.where(torch.rand(4, vocab, generator=g, device="cuda") < 0.5, -0.0, 0.0)
        scores[28:32] = torch.tensor([-0.0, 0.0, 0.0, -0.0])
        check(H, x, scores, 4, ended)
        big = x.clone()
        big[24:28] = torch.randn(4, vocab, generator=g, device="cuda") * 1e30
        scores[24:28] = torch.tensor([-3e38, 3e38, 1e20, -1e-40])
        check(H, big, scores, 4, ended)
    assert H.device_status() == 0


def test_rows_at_any_address_strides_in_place_and_graphs(H):
    g = torch.Generator(device="cuda").manual_seed(9)
    flat = torch.randn(12 * 1111 + 5, generator=g, device="cuda")
    scores = -torch.rand(12, generator=g, device="cuda")
    for off in range(4):
        for ld, vocab in ((1111, 1111), (1111, 1001), (1109, 1109)):
            x = flat[off:].as_strided((12, vocab), (ld, 1))
            check(H, x, scores, 3)
    x = torch.randn(12, 30001, generator=g, device="cuda")
    ws = H.beam_select_workspace(4, 3, 30001)
    first = [t.clone() for t in H.beam_select(x, scores, 3, workspace=ws)]
    ws.fill_(255)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    other = H.beam_select(x, scores, 3, stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = H.beam_select(x, scores, 3, workspace=ws)
    graph.replay()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    scores.copy_(first[0])
    want = H.beam_select(x, scores, 3)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    # the scores may be written over
    par, tok = torch.empty(12, dtype=torch.int32, device="cuda"), torch.empty(12, dtype=torch.int32, device="cuda")
    assert H.lib().hesa_cuda_beam_select(x.data_ptr(), 30001, 4, 3, 30001, scores.data_ptr(), None, scores.data_ptr(), par.data_ptr(), tok.data_ptr(),
                                         ws.data_ptr(), ws.numel(), None) == 0
    torch.cuda.synchronize()
    assert torch.equal(scores, want[0]) and torch.equal(par, want[1]) and torch.equal(tok, want[2])


# ---- reordering ----

class Pages:
    """The tables of a cache on the host."""

    def __init__(self, page, n_pages, table, lens, refs):
        self.page, self.n_pages = page, n_pages
        self.table, self.lens, self.refs = [list(r) for r in table], list(lens), list(refs)

    def used(self, n):
        return -(-n // self.page)

    def reorder(self, slots, parents, width):
        """The page copies (from, to, places), in order, or None where the pool is too small (nothing has changed then)."""
        page = self.page
        source = [slots[i - i % width + p] for i, p in enumerate(parents)]
        refs, table, lens = list(self.refs), [list(r) for r in self.table], list(self.lens)
        for s in slots:
            if s not in source:
                for p in self.table[s][: self.used(self.lens[s])]:
                    refs[p] -= 1
        free, copies, seen = [p for p in range(self.n_pages) if refs[p] == 0], [], set()
        for s, a in zip(slots, source):
            n = self.lens[a]
            row = self.table[a][: self.used(n)]
            if a in seen:
                for p in row[: n // page]:
                    refs[p] += 1
                if n % page:
                    if not free:
                        return None
                    new = free.pop(0)
                    refs[new] = 1
                    copies.append((row[-1], new, n % page))
                    row[-1] = new
            seen.add(a)
            for j, p in enumerate(row):
                table[s][j] = p
            for j in range(len(row), self.used(self.lens[s])):
                table[s][j] = -1
            lens[s] = n
        self.refs, self.table, self.lens = refs, table, lens
        return copies


def random_cache(H, r, kind, n_slots, page, layers=2, n_kv=2, hd=64, most=60, spare=None, gap=0):
    """A cache in use: some slots share the pages of others as forks do."""
    width = -(-most // page) + 1
    lens, rows, refs_of = [], [], {}
    next_page = [0]

    def fresh():
        next_page[0] += 1
        return next_page[0] - 1
    for s in range(n_slots):
        if s and r.random() < 0.4:
            a = r.randrange(s)
            n = lens[a]
            row = rows[a][: n // page] + ([fresh()] if n % page else [])
        else:
            n = r.choice((0, r.randrange(1, most), page * r.randrange(1, max(2, most // page))))
            n = min(n, most)
            row = [fresh() for _ in range(-(-n // page))]
        lens.append(n)
        rows.append(row)
    n_pages = next_page[0] + (spare if spare is not None else r.randrange(0, 2 * n_slots))
    n_pages = max(n_pages, 1)
    perm = list(range(n_pages))
    r.shuffle(perm)
    rows = [[perm[p] for p in row] for row in rows]
    refs = [0] * n_pages
    for row in rows:
        for p in row:
            refs[p] += 1
    table = [row + [-1] * (width - len(row)) for row in rows]
    t = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (table, lens, refs)]
    g = torch.Generator(device="cuda").manual_seed(r.randrange(1 << 30))
    if kind == "kv4":
        pools = kv4_model.pools(layers, n_pages, page, n_kv, hd, gap=gap)
        for p in pools:
            p.copy_(torch.randint(0, 256, p.shape, generator=g, device="cuda", dtype=torch.uint8) if p.dtype == torch.uint8
                    else torch.randn(p.shape, generator=g, device="cuda").half())
        cache = H.PagedKV4(*pools, *t)
    else:
        pools = [torch.randn(layers, n_pages, page, n_kv, hd, generator=g, device="cuda").half() for _ in range(2)]
        cache = H.PagedKV(*pools, *t)
    return cache, pools, t, Pages(page, n_pages, table, lens, refs)


def same_tables(t, m):
    assert t[0].tolist() == m.table and t[1].tolist() == m.lens and t[2].tolist() == m.refs


@pytest.mark.parametrize("kind", ["fp16", "kv4"])
@pytest.mark.parametrize("seed", range(12))
def test_reorder(H, kind, seed):
    r = random.Random(seed)
    width = r.choice((1, 2, 3, 4, 8, 11, 32))
    groups = r.randrange(1, 5)
    n_slots = groups * width + r.randrange(0, 4)
    page = r.choice((1, 4, 7, 16))
    cache, pools, t, m = random_cache(H, r, kind, n_slots, page, n_kv=r.choice((1, 2, 3)), hd=r.choice((64, 128)), gap=r.choice((0, 8)), most=r.choice((5, 60, 200)))
    for step in range(4):
        slots = r.sample(range(n_slots), groups * width)
        parents = [r.randrange(width) for _ in slots] if step != 2 else r.sample(range(width), width) * groups
        before, tables = [p.clone() for p in pools], [x.clone() for x in t]
        copies = m.reorder(slots, parents, width)
        H.kv_reorder(cache, torch.tensor(slots, dtype=torch.int32, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda"), width)
        if copies is None:
            assert H.device_status() == 5
            H.clear_device_status()
            assert all(torch.equal(a, b) for a, b in zip(t, tables))
            copies = []
        assert H.device_status() == 0
        same_tables(t, m)
        for p, b in zip(pools, before):
            want = b.clone()
            for frm, to, places in copies:
                want[:, to, :places] = b[:, frm, :places]
            assert torch.equal(p, want)


def test_reorder_of_many_slots(H):
    """More slots than the planning block has threads, groups that lie across its ends, pages beyond a thousand."""
    r = random.Random(77)
    for width, groups in ((7, 400), (32, 70), (1, 1500)):
        n = width * groups
        cache, pools, t, m = random_cache(H, r, "kv4", n, 4, layers=1, n_kv=1, most=23, spare=n)
        slots = r.sample(range(n), n)
        for step in range(2):
            parents = [r.randrange(width) for _ in slots]
            before = [p.clone() for p in pools]
            copies = m.reorder(slots, parents, width)
            assert copies is not None
            H.kv_reorder(cache, torch.tensor(slots, dtype=torch.int32, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda"), width)
            assert H.device_status() == 0
            same_tables(t, m)
            for p, b in zip(pools, before):
                want = b.clone()
                for frm, to, places in copies:
                    want[:, to, :places] = b[:, frm, :places]
                assert torch.equal(p, want)
        # the last slot of all is not sound: nothing changes
        kept = [x.clone() for x in t]
        t[1][slots[-1]] = 10 ** 6
        now = [x.clone() for x in t]
        H.kv_reorder(cache, torch.tensor(slots, dtype=torch.int32, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda"), width)
        assert H.device_status() == 3 and all(torch.equal(a, b) for a, b in zip(t, now))
        H.clear_device_status()
        for x, k in zip(t, kept):
            x.copy_(k)


@pytest.mark.parametrize("width,groups,most,page", [(12, 1, 300, 1), (5, 4, 300, 1), (12, 4, 300, 1), (32, 1, 900, 1), (2, 40, 333, 2), (1, 30, 400, 1), (7, 3, 4097, 3)])
def test_reorder_of_long_rows(H, width, groups, most, page):
    """Rows that several warps share, and enough entries for several blocks; then a row that is not sound, and too few pages."""
    r = random.Random(most + width)
    n = width * groups
    cache, pools, t, m = random_cache(H, r, "kv4", n + 3, page, layers=2, n_kv=1, most=most, spare=2 * n)
    slots = r.sample(range(n + 3), n)

    def call(parents):
        H.kv_reorder(cache, torch.tensor(slots, dtype=torch.int32, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda"), width)
    for step in range(3):
        parents = [r.randrange(width) for _ in slots]
        before = [p.clone() for p in pools]
        copies = m.reorder(slots, parents, width)
        assert copies is not None
        call(parents)
        assert H.device_status() == 0
        same_tables(t, m)
        for p, b in zip(pools, before):
            want = b.clone()
            for frm, to, places in copies:
                want[:, to, :places] = b[:, frm, :places]
            assert torch.equal(p, want)
    slot = max(slots, key=lambda x: m.lens[x])   # the last page of the longest row
    at = m.used(m.lens[slot]) - 1
    kept = t[0][slot, at].item()
    for bad in (-1, cache.n_pages):
        t[0][slot, at] = bad
        now = [x.clone() for x in t]
        call([0] * n)
        assert H.device_status() == 3 and all(torch.equal(a, b) for a, b in zip(t, now))
        H.clear_device_status()
    t[0][slot, at] = kept
    if page > 1 and width > 1:   # pages are partly filled, and none is free
        first = slots[0]
        t[1][first] -= 1 if m.lens[first] % page != 1 else 0
        t[2].add_(1)
        now = [x.clone() for x in t]
        call([0] * n)
        lens = [t[1][x].item() for x in slots]
        assert any(x % page for x in lens[::width])
        assert H.device_status() == (3 if min(lens) < 0 else 5) and all(torch.equal(a, b) for a, b in zip(t, now))
        H.clear_device_status()
        slot = max(slots, key=lambda x: m.lens[x])   # the same with no length below zero
        t[1][first] = m.lens[first]
        t[1][slot] -= 1 if m.lens[slot] % page != 1 else 0
        now = [x.clone() for x in t]
        call([slots.index(slot) % width] * n)
        assert H.device_status() == 5 and all(torch.equal(a, b) for a, b in zip(t, now))
        H.clear_device_status()


@pytest.mark.parametrize("kind", ["fp16", "kv4"])
def test_reorder_refusals_change_nothing(H, kind):
    r = random.Random(3)
    cache, pools, t, m = random_cache(H, r, kind, 9, 4, spare=0, most=30)

    def call(slots, parents, width):
        H.kv_reorder(cache, torch.tensor(slots, dtype=torch.int32, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda"), width)
        got = H.device_status()
        H.clear_device_status()
        return got
    for slots, parents, width in (([0, 0], [0, 1], 2), ([0, 9], [0, 1], 2), ([0, -1], [0, 1], 2), ([0, 1], [0, 2], 2), ([0, 1], [-1, 0], 2),
                                  ([0, 1, 2, 1], [0, 0, 0, 0], 2)):
        assert call(slots, parents, width) == 3
        same_tables(t, m)
    for x, at, bad in ((t[1], 4, -1), (t[1], 4, 10 ** 6), (t[0], (4, 0), -1), (t[0], (4, 0), cache.n_pages)):
        slot4 = t[1][4].item()
        if slot4 == 0:
            t[1][4] = 1
        kept = [y.clone() for y in t]
        x[at] = bad
        now = [y.clone() for y in t]
        assert call([3, 4, 5], [0, 0, 0], 3) == 3
        assert all(torch.equal(a, b) for a, b in zip(t, now))
        for y, k in zip(t, kept):
            y.copy_(k)
        t[1][4] = slot4
    # a page with fewer references than slots that hold it
    a = next(i for i in range(9) if m.lens[i] >= 4)
    b = (a + 1) % 9
    t[0][b, 0], t[1][b] = t[0][a, 0], 4
    now = [y.clone() for y in t]
    c = next(i for i in range(9) if i not in (a, b))
    t[2][int(t[0][a, 0])] = 1
    now = [y.clone() for y in t]
    assert call([a, b, c], [2, 2, 2], 3) == 3
    assert all(torch.equal(x, y) for x, y in zip(t, now))
    # no pages for the copies: as it was
    cache, pools, t, m = random_cache(H, r, kind, 3, 4, spare=0, most=30)
    t[1].copy_(torch.tensor([3, 3, 3]))
    n = cache.n_pages
    if n >= 3:
        t[0][:, 0] = torch.arange(3)
        t[2].fill_(1)
        now = [y.clone() for y in t]
        t[2][0:3] = 2     # held by somebody else too, so nothing comes free
        now = [y.clone() for y in t]
        assert call([0, 1, 2], [1, 1, 1], 3) == 5
        assert all(torch.equal(x, y) for x, y in zip(t, now))


def test_reorder_in_a_captured_graph(H):
    r = random.Random(8)
    cache, pools, t, m = random_cache(H, r, "kv4", 8, 4, spare=30)
    slots, parents = torch.arange(8, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    ws = H.kv_pages_workspace(cache)
    H.kv_reorder(cache, slots, torch.arange(4, dtype=torch.int32, device="cuda").repeat(2), 4, workspace=ws)   # everything stays in its place
    same_tables(t, m)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        H.kv_reorder(cache, slots, parents, 4, workspace=ws)
    for step in range(3):
        p = [r.randrange(4) for _ in range(8)]
        parents.copy_(torch.tensor(p, dtype=torch.int32))
        ws.fill_(255)
        graph.replay()
        assert m.reorder(list(range(8)), p, 4) is not None
        torch.cuda.synchronize()
        same_tables(t, m)
    assert H.device_status() == 0


def test_page_operations_of_a_cache_in_4_bits(H):
    """Reserve, free, fork, compact and copy give both kinds of cache the same tables, and every slot keeps its codes and scales."""
    r = random.Random(21)
    for gap, n_kv, hd, page in ((0, 2, 64, 4), (8, 1, 64, 3), (0, 3, 128, 16)):
        a, ap, at, m = random_cache(H, r, "kv4", 6, page, n_kv=n_kv, hd=hd, spare=40, gap=gap)
        bt = [x.clone() for x in at]
        bp = [torch.zeros(1, a.n_pages, page, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
        b = H.PagedKV(*bp, *bt)

        def held():
            out = []
            for s in range(6):
                j = torch.arange(int(at[1][s]), device="cuda")
                out.append([p[:, at[0][s][j // page].long(), j % page].clone() for p in ap])
            return out

        def ints(*v):
            return torch.tensor(v, dtype=torch.int32, device="cuda")
        before = held()
        for x in (a, b):
            H.kv_free(x, ints(1, 4))
            H.kv_fork(x, ints(0, 2), ints(1, 4))
        now = held()
        for s, src in ((0, 0), (1, 0), (2, 2), (3, 3), (4, 2), (5, 5)):
            assert all(torch.equal(p, q) for p, q in zip(now[s], before[src]))
        live = [ints(0), ints(0)]
        for x, n in ((a, live[0]), (b, live[1])):
            H.kv_compact(x, n_live=n)
        assert torch.equal(*live)
        after = held()
        assert all(torch.equal(p, q) for s in range(6) for p, q in zip(now[s], after[s]))
        for x in (a, b):
            H.kv_reserve(x, ints(0, 3), ints(5, 1))
        assert all(torch.equal(x, y) for x, y in zip(at, bt))
        was = [p.clone() for p in ap]
        src, dst = ints(0, 1), ints(a.n_pages - 1, a.n_pages - 2)
        H.kv_copy_pages(a, src, dst)
        for p, w in zip(ap, was):
            w[:, dst.long()] = w[:, src.long()]
            assert torch.equal(p, w)
    assert H.device_status() == 0


# ---- a whole search ----

@pytest.mark.parametrize("kind", ["fp16", "kv4"])
def test_a_beam_search(H, kind):
    """Two sequences with five beams each over a small model of one attention layer: prompts as chunks, then steps of
    select, reorder, reserve, write and attend. The reference keeps each beam's tokens and computes everything anew in
    64 bits from the keys and values that the format makes of them; it goes on with the choices that were made. Scores are off by 16 steps' errors of the logits: an attention
    result's 2^-18 of its norm (paged_bounds) and fp32 products of 128 terms (128 2^-24 2 sqrt 128 at the most), 2e-4 for
    logits of norm 12 a step."""
    width, n_head, n_kv, hd, vocab, page, eos = 5, 4, 2, 64, 61, 4, 60
    g = torch.Generator(device="cuda").manual_seed(31)

    def rand(*s):
        return torch.randn(*s, generator=g, device="cuda", dtype=torch.float32)
    d = 32
    emb, wq, wk, wv, wo = rand(vocab, d), rand(d, n_head * hd) / d ** 0.5, rand(d, n_kv * hd) / d ** 0.5, rand(d, n_kv * hd) / d ** 0.5, rand(n_head * hd, vocab) / 6
    table = torch.from_numpy(H.rope_table(64, hd)).cuda()
    prompts = [[3, 17, 5, 9, 22, 41, 8], [12, 7]]
    n = 2 * width
    cls = H.PagedKV4 if kind == "kv4" else H.PagedKV
    cache = cls.empty(1, 200, page, n_kv, hd, n, 16)

    def project(tokens):
        x = emb[tokens]
        return [(x.double() @ w.double()).float() for w in (wq, wk, wv)]

    def step(batch, tokens):
        q, k, v = project(tokens)
        H.rope_kv_paged(cache, 0, batch, q, k, v, n_head, rope_table=table)
        return H.paged_attention(cache, 0, batch, q, n_head)

    def rope(x, pos):
        a, b = x[..., : hd // 2], x[..., hd // 2:]
        c, s = table[pos, : hd // 2][:, None], table[pos, hd // 2:][:, None]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    def reference(tokens):
        """The last token's logits in 64 bits."""
        t = torch.tensor(tokens, device="cuda")
        q, k, v = project(t)
        pos = torch.arange(len(tokens), device="cuda")
        q, k, v = rope(q.view(-1, n_head, hd), pos)[-1].double(), rope(k.view(-1, n_kv, hd), pos), v.view(-1, n_kv, hd)
        k, v = [kv4_model.values(*kv4_model.quantize(x)).double() if kind == "kv4" else x.half().double() for x in (k, v)]
        k, v = k.repeat_interleave(n_head // n_kv, 1), v.repeat_interleave(n_head // n_kv, 1)
        p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) / hd ** 0.5, 1)
        return torch.einsum("hn,nhd->hd", p, v).reshape(-1) @ wo.double()

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")
    # prompts into the first beam's slot; the other beams are copies of it
    first = ints([0, width])
    H.kv_reserve(cache, first, ints([len(p) for p in prompts]))
    batch = H.TokenBatch(ints([0, 7, 9]), 9, 7, 60, slots=first)
    out = step(batch, torch.tensor(prompts[0] + prompts[1], device="cuda"))
    H.kv_fork(cache, ints([0] * 4 + [width] * 4), ints([1, 2, 3, 4, 6, 7, 8, 9]))
    rows = out[[6, 8]].double() @ wo.double()
    logits = rows.float().repeat_interleave(width, 0)
    scores = torch.full((n,), -math.inf, device="cuda")
    scores[[0, width]] = 0.0
    ended = torch.zeros(n, dtype=torch.int32, device="cuda")
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    hist = [list(prompts[i // width]) for i in range(n)]
    want_scores, want_ended = [0.0 if i % width == 0 else -math.inf for i in range(n)], [False] * n
    for it in range(16):
        scores, parents, tokens = H.beam_select(logits, scores, width, ended=ended)
        # every choice is a candidate of its own, with its score, and as good as the reference's choice at its place
        par, tok, tol = parents.tolist(), tokens.tolist(), 2e-4 * (it + 1)
        new_hist, new_scores, new_ended = [], [], []
        for s0 in (0, width):
            cand = {}
            for b in range(width):
                if want_ended[s0 + b]:
                    cand[b, -1] = want_scores[s0 + b]
                elif want_scores[s0 + b] > -math.inf:
                    lp = torch.log_softmax(reference(hist[s0 + b]), 0).tolist()
                    cand.update({(b, t): want_scores[s0 + b] + lp[t] for t in range(vocab)})
            best = sorted(cand.values(), reverse=True)
            mine = list(zip(par[s0: s0 + width], tok[s0: s0 + width]))
            assert len(set(mine)) == width
            for i, c in enumerate(mine):
                assert abs(float(scores[s0 + i]) - cand[c]) <= tol, f"step {it}"
                assert cand[c] >= best[i] - 2 * tol, f"step {it}"
                b, t = c
                new_hist.append(hist[s0 + b] + ([t] if t >= 0 else []))
                new_scores.append(cand[c])
                new_ended.append(t in (-1, eos))
        hist, want_scores, want_ended = new_hist, new_scores, new_ended
        H.kv_reorder(cache, slots, parents, width)
        on = (tokens >= 0).int()
        ended = ((tokens < 0) | (tokens == eos)).int()
        H.kv_reserve(cache, slots, on)
        starts = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), on.cumsum(0).int()])
        m = int(starts[-1])
        out = step(H.TokenBatch(starts, m, 1, 60), tokens[tokens >= 0].long())
        logits = torch.zeros(n, vocab, device="cuda")
        logits[tokens >= 0] = (out.double() @ wo.double()).float()
        assert cache.seq_len.tolist() == [len(h) for h in hist]
        assert H.device_status() == 0
    refs = cache.page_refs.tolist()
    held = [p for s in range(n) for p in cache.table[s, : -(-len(hist[s]) // page)].tolist()]
    assert refs == [held.count(p) for p in range(200)]


def test_two_host_threads_at_once(H):
    """Writes, reads, attention, selection and reordering from two threads, each on a stream of its own with a cache of its own."""
    import threading
    r = random.Random(5)
    work = []
    for i in range(2):
        kv, hd, page, vocab = ((2, 64, 4, 5003), (1, 128, 16, 40))[i]
        n, width = 8, 4
        cache, pools, t, m = random_cache(H, r, "kv4", n, page, layers=1, n_kv=kv, hd=hd, most=40, spare=40)
        t[1].fill_(1)
        t[0].fill_(-1)
        t[0][:, 0] = torch.arange(n, dtype=torch.int32)
        t[2].fill_(0)
        t[2][:n] = 1
        first = [x.clone() for x in t]
        for p in pools:   # values that are sound
            p.zero_()
        g = torch.Generator(device="cuda").manual_seed(i)
        batch = H.TokenBatch(torch.arange(n + 1, dtype=torch.int32, device="cuda"), n, 1, 20)
        work.append(dict(cache=cache, pools=pools, t=t, first=first, batch=batch, n=n, width=width, kv=kv, hd=hd, vocab=vocab, slots=torch.arange(n, dtype=torch.int32, device="cuda"),
                         one=torch.ones(n, dtype=torch.int32, device="cuda"), x=torch.randn(12, 3, n, kv * hd, generator=g, device="cuda"),
                         logits=torch.randn(12, n, vocab, generator=g, device="cuda")))

    def search(w):
        for a, b in zip(w["t"], w["first"]):
            a.copy_(b)
        for p in w["pools"]:
            p.zero_()
        scores, seen = torch.zeros(w["n"], device="cuda"), []
        for step in range(12):
            scores, parents, tokens = H.beam_select(w["logits"][step], scores, w["width"])
            H.kv_reorder(w["cache"], w["slots"], parents, w["width"])
            H.kv_reserve(w["cache"], w["slots"], w["one"])
            q, k, v = w["x"][step]
            H.rope_kv_paged(w["cache"], 0, w["batch"], None, k, v, w["kv"])
            seen += [scores, parents, tokens, *H.kv_read(w["cache"], 0, w["batch"]), H.paged_attention(w["cache"], 0, w["batch"], q, w["kv"])]
        return [x.clone() for x in seen + w["t"]]
    want = [search(w) for w in work]
    assert H.device_status() == 0
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(15):
                got = search(work[i])
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and H.device_status() == 0


# The branches of the selection's dispatch: a cluster a sequence, two kernels with blocks of eight warps, and with blocks
# of two; each with parts that a block reads in one pass, and longer ones whose largest values it reads again.
BRANCHES = [
    (3, 8, 4000), (2, 3, 5001), (5, 5, 3999), (3, 8, 20001), (2, 3, 40002), (74, 4, 9003),          # clusters
    (10, 16, 4000), (4, 32, 3001), (75, 3, 2002), (20, 16, 9001), (80, 3, 9002), (80, 8, 12003), (5, 32, 20001),   # eight warps
    (100, 3, 1001), (75, 8, 517), (30, 16, 1020), (12, 32, 899), (300, 4, 1021),                    # two warps, one pass
    # short rows that are read again: two warps where there are more than 2 * width sequences
    (80, 5, 1023), (100, 3, 1030), (80, 4, 2050), (76, 8, 1025), (128, 16, 3000), (40, 16, 4095), (100, 32, 4096), (20, 32, 1537),
    (65, 16, 1022), (131, 32, 1537), (64, 16, 1022), (33, 16, 1022), (32, 16, 1022), (65, 32, 1537), (64, 32, 1537), (30, 16, 1024),
]


@pytest.mark.parametrize("n_seq,width,vocab", BRANCHES)
def test_select_of_every_branch(H, n_seq, width, vocab):
    """Rows of odd lengths begin at every alignment. Random values, ascending ones (the largest with the last threads),
    and rows with their largest side by side (all with one thread)."""
    g = torch.Generator(device="cuda").manual_seed(vocab * 33 + width)
    n = n_seq * width
    x = torch.randn(n, vocab, generator=g, device="cuda") * 3
    x[1::3] = torch.linspace(-4, 4, vocab, device="cuda")
    at = int(torch.randint(0, max(1, vocab - 16), (1,), generator=g, device="cuda"))
    x[2::3, at:at + 16] += 9
    scores = -torch.rand(n, generator=g, device="cuda") * 5
    check(H, x, scores, width)
    check(H, x, scores, width, (torch.rand(n, generator=g, device="cuda") < 0.3).int())
    assert H.device_status() == 0
