"""GPU parity of the paged cache's attention against its definition in 64 bits.

Tolerance, per case and derived from its data: a score s = sum_i q_i k_i c has an
absolute error of at most (hd / 16 + 6) 2^-23 c sum_i |q_i k_i| (one rounding for
each 16-wide product added, for the two halves of q and for the scale), a capped
score 2^-21 cap more, a bias 2^-23 |bias| more; p = e^(s - m) gets that error, 2^-21
for the exponential and 2^-21 for its two halves; the output sum p v / sum p is off
by at most twice p's relative error, and 2^-21 for its sums, times the largest |v|.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available()
    import hesa_cuda
    hesa_cuda.lib()
    hesa_cuda.clear_device_status()
    return torch


class Case:
    """A cache whose sequences lie at random pages; every place that no token owns holds NaN."""

    def __init__(self, T, n_head, n_kv, hd, page, lens, news, seed=0, layers=1, slots=None, spare=2):
        import hesa_cuda as H
        g = T.Generator(device="cuda").manual_seed(seed)
        self.T, self.H, self.n_head, self.n_kv, self.hd, self.page = T, H, n_head, n_kv, hd, page
        self.lens, self.news, self.n_seq = lens, news, len(lens)
        self.slot_of = slots or list(range(len(lens)))
        n_slots = max(self.slot_of) + 1
        width = max(1, max(-(-n // page) for n in lens))
        n_pages = sum(-(-n // page) for n in lens) + spare
        self.k = T.full((layers, n_pages, page, n_kv, hd), math.nan, dtype=T.float16, device="cuda")
        self.v = self.k.clone()
        order = T.randperm(n_pages, generator=g, device="cuda").tolist()
        table = T.full((n_slots, width), -1, dtype=T.int32)
        seq_len = T.zeros(n_slots, dtype=T.int32)
        self.keys, self.values = [], []
        at = 0
        for i, n in enumerate(lens):
            np_ = -(-n // page)
            pages = order[at:at + np_]
            at += np_
            table[self.slot_of[i], :np_] = T.tensor(pages, dtype=T.int32)
            seq_len[self.slot_of[i]] = n
            kk = T.randn(n, n_kv, hd, generator=g, device="cuda").half()
            vv = T.randn(n, n_kv, hd, generator=g, device="cuda").half()
            for j, p in enumerate(pages):
                m = min(page, n - j * page)
                self.k[layers - 1, p, :m] = kk[j * page:j * page + m]
                self.v[layers - 1, p, :m] = vv[j * page:j * page + m]
            self.keys.append(kk)
            self.values.append(vv)
        self.layer = layers - 1
        self.cache = H.PagedKV(self.k, self.v, table.cuda(), seq_len.cuda())
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        self.starts, self.n_tokens = starts, starts[-1]
        self.q_start = T.tensor(starts, dtype=T.int32, device="cuda")
        self.slots = T.tensor(self.slot_of, dtype=T.int32, device="cuda") if slots else None
        self.q = T.randn(self.n_tokens, n_head * hd, generator=g, device="cuda") * 1.3
        self.batch = H.TokenBatch(self.q_start, self.n_tokens, max(news), max(lens), slots=self.slots)

    def run(self, **kw):
        return self.H.paged_attention(self.cache, self.layer, self.batch, self.q, self.n_head, **kw)

    def exact(self, scale=None, softcap=0.0, window=0, slopes=None, prefix=None):
        """(definition in 64 bits, tolerance)"""
        T = self.T
        scale = scale or 1.0 / math.sqrt(self.hd)
        out = T.zeros(self.n_tokens, self.n_head, self.hd, dtype=T.float64, device="cuda")
        q = self.q.view(self.n_tokens, self.n_head, self.hd).double()
        worst_s, worst_b, vmax = 0.0, 0.0, 1e-30
        for i in range(self.n_seq):
            lo, hi, n = self.starts[i], self.starts[i + 1], self.lens[i]
            if hi == lo or n == 0:
                continue
            pos = T.arange(n - (hi - lo), n, device="cuda")[:, None]
            j = T.arange(n, device="cuda")[None, :]
            see = j <= pos
            if window:
                see &= j > pos - window
            if prefix is not None:
                see |= j < int(prefix[i])
            for h in range(self.n_head):
                kk, vv = self.keys[i][:, h * self.n_kv // self.n_head].double(), self.values[i][:, h * self.n_kv // self.n_head].double()
                s = q[lo:hi, h] @ kk.T * scale
                worst_s = max(worst_s, float((q[lo:hi, h].abs() @ kk.abs().T).max()) * scale)
                if softcap:
                    s = softcap * T.tanh(s / softcap)
                if slopes is not None:
                    b = float(slopes[h]) * (pos - j).abs().double()
                    worst_b = max(worst_b, float((b * see).max()))
                    s = s - b
                s = s.masked_fill(~see, -math.inf)
                m = s.amax(1, keepdim=True)
                p = T.exp(s - T.where(m == -math.inf, T.zeros_like(m), m))
                z = p.sum(1, keepdim=True)
                out[lo:hi, h] = T.where(z > 0, (p @ vv) / z, T.zeros_like(z))
                vmax = max(vmax, float(vv.abs().max()))
        e = (self.hd / 16 + 6) * 2.0 ** -23 * worst_s + 2.0 ** -21 * softcap + 2.0 ** -23 * worst_b + 2 * 2.0 ** -21
        return out.view(self.n_tokens, -1), (2 * e + 2.0 ** -21) * vmax


def check(c, **opts):
    ref, tol = c.exact(**opts)
    out = c.run(**opts)
    assert c.T.isfinite(out).all()
    err = float((out.double() - ref).abs().max())
    assert err <= tol, f"max error {err:.3e} over {tol:.3e}"
    assert c.H.device_status() == 0
    return out


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens", [
    (32, 32, 128, 16, [2048]),              # the 7B layout
    (64, 8, 128, 16, [1, 17, 300, 5, 1023]),
    (8, 2, 64, 5, [37, 1, 160]),            # pages that end inside a block of keys
    (4, 4, 256, 24, [300, 33]),
    (12, 2, 128, 1, [65, 2]),               # a page for each token, groups of six
    (32, 2, 64, 128, [129, 128, 127]),      # groups of sixteen: two tiles of rows
    (8, 1, 128, 64, [20011, 3]),            # split over the keys
    (2, 1, 256, 48, [9001]),
])
def test_next_token(T, n_head, n_kv, hd, page, lens):
    check(Case(T, n_head, n_kv, hd, page, lens, [1] * len(lens), seed=n_head + hd))


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens,news", [
    (4, 4, 128, 16, [512], [512]),                     # a whole prompt
    (8, 2, 128, 16, [700, 50, 33, 257], [130, 50, 0, 1]),
    (16, 4, 64, 24, [301, 7, 1000], [100, 7, 333]),
    (4, 2, 256, 16, [150, 90], [70, 90]),
    (6, 2, 128, 7, [400, 129], [129, 128]),            # groups of three
    (8, 1, 128, 32, [5000], [40]),                     # few rows, many keys
    (2, 2, 64, 16, [1, 1, 2], [1, 1, 2]),
    (64, 8, 128, 64, [2100], [200]),
    (4, 1, 256, 16, [700, 64, 260], [70, 64, 255]),
    (16, 2, 256, 64, [3000], [100]),
    (8, 8, 256, 8, [1, 190, 65], [1, 190, 30]),
    (4, 2, 256, 20, [150, 500], [70, 21]),             # wide heads in pages that are no multiple of 8
])
def test_chunk(T, n_head, n_kv, hd, page, lens, news):
    check(Case(T, n_head, n_kv, hd, page, lens, news, seed=hd + len(lens)))


OPTIONS = [dict(softcap=20.0), dict(window=1), dict(window=33), dict(window=100, softcap=5.0), dict(slopes=True),
           dict(prefix=True), dict(prefix=True, window=40), dict(slopes=True, prefix=True, window=64, softcap=30.0), dict(scale=0.3)]


@pytest.mark.parametrize("opts", OPTIONS, ids=lambda o: "-".join(o))
@pytest.mark.parametrize("shape", [(8, 2, 64, 24, [300, 41, 129], [1, 1, 1]), (8, 2, 128, 16, [400, 150, 31], [170, 150, 5]),
                                   (4, 4, 256, 16, [200, 66], [77, 1]), (8, 1, 128, 16, [6000, 700], [2, 1])], ids=("next", "chunk", "wide", "split"))
def test_options(T, shape, opts):
    c = Case(T, *shape, seed=7)
    opts = dict(opts)
    if opts.get("slopes"):
        opts["slopes"] = T.exp2(-8.0 * T.arange(1, c.n_head + 1, device="cuda") / c.n_head)
    if opts.get("prefix"):
        opts["prefix"] = T.tensor([min(n, 90) if i != 1 else 0 for i, n in enumerate(c.lens)], dtype=T.int32, device="cuda")
    check(c, **opts)


@pytest.mark.parametrize("seed", range(100))
def test_random_batches(T, seed):
    """Ragged batches of all head layouts, with empty sequences, more new tokens than tokens, and any mask."""
    import random
    r = random.Random(1000 + seed)
    n_kv = r.choice([1, 2, 3, 4, 5, 6, 8, 9, 12, 17])
    group = r.choice([1, 1, 2, 3, 4, 7, 8, 16])
    hd = r.choice([64, 128, 128, 256])
    page = r.choice([1, 3, 8, 16, 24, 40, 64, 128, 200])
    n_seq = r.choice([1, 2, 5, 23])
    most = r.choice([40, 300, 3000]) if n_seq > 5 else r.choice([40, 700, 6000])
    lens = [r.choice([0, 1, r.randrange(0, most), most]) for _ in range(n_seq)]
    lens[0] = max(1, lens[0])
    top = r.choice([1, 1, 3, 60])
    news = [r.randrange(0, min(top, n + 2) + 1) for n in lens]
    news[0] = max(1, news[0])
    c = Case(T, n_kv * group, n_kv, hd, page, lens, news, seed=seed)
    opts = {}
    if r.random() < 0.4:
        opts["window"] = r.choice([1, 5, 16, 130, 1000])
    if r.random() < 0.3:
        opts["softcap"] = r.choice([2.0, 30.0])
    if r.random() < 0.3:
        opts["slopes"] = T.exp2(-4.0 * T.rand(c.n_head, device="cuda"))
    if r.random() < 0.3:
        opts["prefix"] = T.tensor([r.randrange(0, n + 1) for n in lens], dtype=T.int32, device="cuda")
    check(c, **opts)


@pytest.mark.parametrize("n_head,n_kv,hd,news", [(8, 1, 64, [1]), (16, 8, 64, [1]), (34, 17, 64, [20, 0, 9])])
def test_many_sequences(T, n_head, n_kv, hd, news):
    """More tiles than one launch sums up (1024), and more than are worth splitting (4096 with their kv heads)."""
    n = 1300
    lens = [1 + (i * 37) % 61 for i in range(n)]
    check(Case(T, n_head, n_kv, hd, 16, lens, [min(news[i % len(news)], lens[i]) for i in range(n)], seed=n_head))


def test_rows_that_see_nothing_are_zero(T):
    """More new tokens than tokens: rows of negative positions see no key (or the prefix alone)."""
    c = Case(T, 4, 2, 64, 8, [5, 20], [9, 3], seed=3)
    out = check(c)
    assert not out[:4].any() and out[4:].abs().sum(1).min() > 0
    check(c, prefix=T.tensor([2, 0], dtype=T.int32, device="cuda"))


@pytest.mark.parametrize("new,hd", [(1, 128), (40, 128), (200, 128), (200, 64), (200, 256), (1, 256)])
def test_hidden_values_do_not_leak(T, new, hd):
    """NaN and infinities in keys and values that a row does not see leave it as it was."""
    c = Case(T, 8, 2, hd, 16, [333], [new], seed=11)
    window = 50
    ref, tol = c.exact(window=window)
    first = 333 - new
    table = c.cache.table[0]
    for j, bad in ((first - 70, math.nan), (first - 50, math.inf), (3, -math.inf)):   # before the first row's window
        p, s = int(table[j // 16]), j % 16
        c.k[0, p, s] = bad
        c.v[0, p, s] = bad
    out = c.run(window=window)
    assert float((out.double() - ref).abs().max()) <= tol
    if new > 30:
        # token first + 20 is hidden from the first 20 rows and seen by the next
        j = first + 20
        p, s = int(table[j // 16]), j % 16
        d = hd - 59
        c.v[0, p, s, 0, d] = math.nan
        out = c.run(window=window)
        ok = T.ones(new, c.n_head, c.hd, dtype=T.bool, device="cuda")
        ok[20:20 + window, :4, d] = False
        good = ok.view(new, -1)
        assert float((out.double() - ref).abs()[good].max()) <= tol
        assert T.isnan(out[~good]).all()
    assert c.H.device_status() == 0


def test_rows_of_q_that_are_not_finite(T):
    c = Case(T, 4, 2, 64, 16, [100], [20], seed=5)
    ref, tol = c.exact()
    c.q[3, 70] = math.inf
    c.q[9, 0] = math.nan
    out = c.run().view(20, 4, 64)
    assert T.isnan(out[3, 1]).all() and T.isnan(out[9, 0]).all()
    ok = T.ones(20, 4, 64, dtype=T.bool, device="cuda")
    ok[3, 1] = ok[9, 0] = False
    assert float((out.double() - ref.view(20, 4, 64)).abs()[ok].max()) <= tol


@pytest.mark.parametrize("new", [1, 37])
def test_extreme_magnitudes(T, new):
    """Scores far from each other, tiny and huge rows of q: a row's result depends on its own scale alone."""
    c = Case(T, 4, 2, 128, 16, [500], [new], seed=6)
    c.q[0] *= 1e-30
    c.q[-1, :128] *= 2000.0
    ref, tol = c.exact()
    out = c.run()
    assert float((out.double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("news", [[1, 1, 1], [30, 1, 90]])
def test_strides_slots_and_rows_behind_the_batch(T, news):
    """Column slices, a slot map, several layers, and rows after the last sequence's."""
    c = Case(T, 8, 2, 64, 16, [50, 33, 200], news, seed=9, layers=3, slots=[4, 0, 2])
    ref, tol = c.exact()
    n = c.n_tokens + 5
    wide = T.full((n, 8 * 64 + 12), 7.0, device="cuda")
    wide[:c.n_tokens, 4:4 + 512] = c.q
    c.q = wide[:, 4:4 + 512]
    out = T.full((n, 600), -3.0, device="cuda")
    c.batch = c.H.TokenBatch(c.q_start, n, max(news), 200, slots=c.slots)
    c.run(out=out[:, 8:520])
    assert float((out[:c.n_tokens, 8:520].double() - ref).abs().max()) <= tol
    assert (out[c.n_tokens:] == -3.0).all() and (out[:, :8] == -3.0).all() and (out[:, 520:] == -3.0).all()


def test_page_and_layer_strides(T):
    """Pools whose layers are nested inside the pages."""
    c = Case(T, 8, 2, 64, 16, [90, 40], [1, 33], seed=10)
    ref, tol = c.exact()
    both = T.full((c.k.shape[1], 3, 2, 16, 2, 64), math.nan, dtype=T.float16, device="cuda")
    k, v = both[:, :, 0].permute(1, 0, 2, 3, 4), both[:, :, 1].permute(1, 0, 2, 3, 4)
    k[1].copy_(c.k[0])
    v[1].copy_(c.v[0])
    c.cache, c.layer = c.H.PagedKV(k, v, c.cache.table, c.cache.seq_len), 1
    assert float((c.run().double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("news", [[1, 1, 1], [5, 60, 3]])
def test_pages_with_gaps(T, news):
    """A page stride that is no multiple of a token's row."""
    c = Case(T, 4, 2, 128, 16, [50, 200, 70], news, seed=19)
    ref, tol = c.exact()
    n = c.k.shape[1]
    pools = []
    for x in (c.k, c.v):
        wide = T.full((1, n, 16 * 256 + 40), math.nan, dtype=T.float16, device="cuda")
        p = wide.as_strided((1, n, 16, 2, 128), (wide.stride(0), wide.stride(1), 256, 128, 1))
        p.copy_(x)
        pools.append(p)
    c.cache = c.H.PagedKV(pools[0], pools[1], c.cache.table, c.cache.seq_len)
    assert float((c.run().double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("news", [[1, 1, 1], [5, 60, 3]])
def test_unsound_tables_are_skipped(T, news):
    """A page outside the pool, a length over the bound, a slot that is not there: status 3, the others as before."""
    c = Case(T, 8, 2, 64, 16, [50, 200, 70], news, seed=12)
    ref, tol = c.exact()
    last = slice(c.starts[2], c.starts[3])
    for what in ("page", "negative", "length", "slot", "start"):
        table, lens, starts = c.cache.table.clone(), c.cache.seq_len.clone(), c.q_start.clone()
        slots = T.arange(3, dtype=T.int32, device="cuda")
        if what == "page":
            table[1, 2] = c.k.shape[1]
        elif what == "negative":
            table[1, 0] = -7
        elif what == "length":
            lens[1] = 201
        elif what == "slot":
            slots[1] = 3
        else:
            starts[1] = -4
        cache = c.H.PagedKV(c.k, c.v, table, lens)
        batch = c.H.TokenBatch(starts, c.n_tokens, max(news), 200, slots=slots)
        out = c.H.paged_attention(cache, 0, batch, c.q, 8)
        assert c.H.device_status() == 3, what
        c.H.clear_device_status()
        assert float((out.double() - ref)[last].abs().max()) <= tol, what
    assert float((c.run().double() - ref).abs().max()) <= tol   # and the workspace of none is spoilt
    assert c.H.device_status() == 0


@pytest.mark.parametrize("shape", [(8, 1, 128, 16, [4000, 900], [1, 1]), (8, 2, 128, 16, [900, 70], [64, 70])])
def test_captured_and_replayed_with_new_lengths(T, shape):
    """One graph serves every step within its bounds; results are the eager call's, bit for bit."""
    c = Case(T, *shape, seed=13)
    ws = c.H.paged_attention_workspace(c.cache, c.batch, c.n_head)
    out = T.zeros(c.n_tokens, c.n_head * c.hd, device="cuda")
    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(side):
        c.run(out=out, workspace=ws)
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g, stream=side):
            c.run(out=out, workspace=ws)
    T.cuda.synchronize()
    for cut in (0, 5, 64):
        c.cache.seq_len.copy_(T.tensor([n - cut for n in c.lens], dtype=T.int32))
        out.zero_()
        g.replay()
        T.cuda.synchronize()
        eager = c.run()
        assert T.equal(out, eager)
        d = Case.__new__(Case)
        d.__dict__ = dict(c.__dict__, lens=[n - cut for n in c.lens], keys=[k[:len(k) - cut] for k in c.keys], values=[v[:len(v) - cut] for v in c.values])
        ref, tol = d.exact()
        assert float((out.double() - ref).abs().max()) <= tol


def test_workspace_shared_by_shapes_and_streams_of_their_own(T):
    """Calls of different shapes one after another in one workspace; two streams at once, each with its own."""
    a = Case(T, 8, 1, 128, 16, [5000], [1], seed=14)
    b = Case(T, 16, 4, 64, 16, [3000, 20, 4000], [1, 1, 1], seed=15)
    d = Case(T, 8, 2, 128, 16, [900], [300], seed=16)
    ws = max((x.H.paged_attention_workspace(x.cache, x.batch, x.n_head) for x in (a, b, d)), key=lambda t: t.numel())
    want = [x.run() for x in (a, b, d)]
    for _ in range(3):
        for x, w in zip((a, b, d), want):
            assert T.equal(x.run(workspace=ws), w)
    s1, s2 = T.cuda.Stream(), T.cuda.Stream()
    T.cuda.synchronize()
    got1, got2 = [], []
    for _ in range(4):
        got1.append(a.run(stream=s1))
        got2.append(b.run(stream=s2))
    T.cuda.synchronize()
    assert all(T.equal(g, want[0]) for g in got1) and all(T.equal(g, want[1]) for g in got2)


def test_a_batch_without_rows(T):
    """A step in which nothing is new: no error, nothing written."""
    c = Case(T, 4, 2, 64, 16, [50, 3], [1, 1], seed=18)
    none = c.H.TokenBatch(T.zeros(3, dtype=T.int32, device="cuda"), 0, 0, 50)
    k, v = c.k.clone(), c.v.clone()
    q = T.zeros(0, 256, device="cuda")
    assert c.H.paged_attention(c.cache, 0, none, q, 4).shape == (0, 256)
    c.H.rope_kv_paged(c.cache, 0, none, q, q[:, :128], q[:, :128], 4, rope_table=T.zeros(60, 64, device="cuda"))
    assert T.equal(c.k.view(T.int16), k.view(T.int16)) and T.equal(c.v.view(T.int16), v.view(T.int16)) and c.H.device_status() == 0


def test_refusals_of_the_binding(T):
    c = Case(T, 4, 2, 64, 16, [50], [1], seed=17)
    H = c.H
    with pytest.raises(ValueError):
        H.paged_attention(c.cache, 0, c.batch, c.q.cpu(), 4)
    with pytest.raises(ValueError):
        H.paged_attention(c.cache, 0, c.batch, c.q.half(), 4)
    with pytest.raises(ValueError):
        H.paged_attention(c.cache, 0, c.batch, c.q[:, :128], 4)
    with pytest.raises(H.HesaError):
        H.paged_attention(c.cache, 1, c.batch, c.q, 4)      # no such layer
    with pytest.raises(H.HesaError):
        c.run(workspace=T.zeros(64, dtype=T.uint8, device="cuda"))
    with pytest.raises(ValueError):
        H.PagedKV(c.k.float(), c.v.float(), c.cache.table, c.cache.seq_len)
    with pytest.raises(ValueError):
        H.PagedKV(c.k, c.v[:, :1], c.cache.table, c.cache.seq_len)
