"""GPU tests of the paged operators at the edges of what their contract allows."""
import math  # noqa: F401

import pytest

from paged_bounds import RMS, relative
from test_paged_attention_gpu import Case, T  # noqa: F401  (T: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_head,n_kv,hd,before,news", [
    (16, 2, 128, 10, [0, 2, 1] + [0, 1] * 12 + [0] * 3),      # next tokens, a row a group: tiles of 8 rows by q_start
    (3, 3, 64, 61, [1, 16, 0] + [1, 0, 0] * 9),               # groups of one
    (8, 8, 256, 5, [1, 9, 0, 1] + [0, 1] * 13),
    (16, 2, 64, 64, [0, 100, 3, 0, 5, 0]),                    # chunks, the first sequence empty
    (16, 2, 128, 7, [4, 100, 0, 0, 21, 0]),
    (8, 1, 256, 33, [0, 90, 0, 7, 0, 0]),
])
def test_a_batch_that_is_part_of_a_longer_one(T, n_head, n_kv, hd, before, news):
    """q_start that begins behind row 0: its sequences as ever, the rows before them and behind them as they were."""
    n = len(news)
    lens = [max(1, x) + 13 * i % 70 for i, x in enumerate(news)]
    c = Case(T, n_head, n_kv, hd, 16, lens, news, seed=21)
    ref, tol = c.exact()
    rows = before + c.n_tokens + 2
    q = T.full((rows, n_head * hd), math.nan, device="cuda")
    q[before:before + c.n_tokens] = c.q
    out = T.full_like(q, -5.0)
    c.batch = c.H.TokenBatch(c.q_start + before, rows, max(news), max(lens))
    c.q = q
    # more sequences times tiles than rows can fill: tiles are found by q_start
    r = 8 if max(news) * (n_head // n_kv) <= (48 if hd == 256 else 16) else 128
    assert n * -(-max(news) * (n_head // n_kv) // r) > rows * (n_head // n_kv) // r + n
    c.run(out=out)
    assert float((out[before:before + c.n_tokens].double() - ref).abs().max()) <= tol
    assert (out[:before] == -5.0).all() and (out[before + c.n_tokens:] == -5.0).all()
    k = T.randn(rows, 2 * n_kv * hd, device="cuda")
    c.H.rope_kv_paged(c.cache, 0, c.batch, None, k[:, :n_kv * hd], k[:, n_kv * hd:], n_head)
    last = max(i for i, x in enumerate(news) if x)
    p = lens[last] - 1
    at = c.cache.table[last, p // 16].item()
    assert T.equal(c.k[0, at, p % 16].reshape(-1), k[before + c.starts[last + 1] - 1, :n_kv * hd].half())
    assert c.H.device_status() == 0


def test_page_operations_beside_a_busy_stream(T):
    """Scratch for a call on another stream, while the current one still uses memory that it has given back; then by turns
    on three streams, one of them current without being named, and captured."""
    import hesa_cuda as H
    from test_kv_pages_gpu import Model, fresh, ints, same
    _, c, m = fresh(T, n_layer=3, n_pages=60)
    assert isinstance(m, Model)
    k, v = c.k.clone(), c.v.clone()
    lists = {x: ints(T, x) for x in ((0,), (1,), (2,), (3,), (4,), (0, 1), (2, 3), (19, 30), (7,))}

    def copied(pairs):
        for a, b, n in pairs:
            k[:, b, :n] = k[:, a, :n]
            v[:, b, :n] = v[:, a, :n]
    need = H.kv_pages_workspace(c).numel()
    s1, s2 = T.cuda.Stream(), T.cuda.Stream()
    T.cuda.synchronize()
    T.cuda._sleep(20_000_000)                                   # about 10 ms
    gone = [T.full((need,), 255, dtype=T.uint8, device="cuda") for _ in range(8)]   # written behind the sleep
    del gone                                                    # to the allocator, while those writes are queued
    H.kv_reserve(c, lists[0, 1], lists[19, 30], stream=s1)
    H.kv_fork(c, lists[0, 1], lists[2, 3], stream=s1)
    s2.wait_stream(s1)
    with T.cuda.stream(s2):
        H.kv_free(c, lists[1,])
        H.kv_compact(c)
    T.cuda.current_stream().wait_stream(s2)
    H.kv_reserve(c, lists[4,], lists[7,])
    m.reserve([0, 1], [19, 30])
    copied(m.fork([0, 1], [2, 3]))
    m.free([1])
    copied([(a, b, m.page) for a, b in m.compact()[1]])
    m.reserve([4], [7])
    same(c, m)
    assert T.equal(c.k, k) and T.equal(c.v, v)
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):                                       # without a workspace: the graph has its own
        H.kv_free(c, lists[3,])
        H.kv_fork(c, lists[0,], lists[3,])
    g.replay()
    m.free([3])
    copied(m.fork([0], [3]))
    same(c, m)
    assert T.equal(c.k, k) and T.equal(c.v, v) and H.device_status() == 0


@pytest.mark.parametrize("n_seq,n_head,n_kv,hd", [(1024, 32, 32, 128), (1024, 8, 8, 64), (200, 64, 16, 64), (300, 17, 17, 256), (3, 64, 8, 128),
                                                  (5, 8, 2, 128)])
@pytest.mark.parametrize("new", [1, 40])
def test_nobody_has_a_key(T, n_seq, n_head, n_kv, hd, new):
    """New rows of sequences without tokens see nothing: zeros, in every row."""
    n_seq = min(n_seq, 60) if new > 1 else n_seq
    c = Case(T, n_head, n_kv, hd, 16, [0] * n_seq, [new] * n_seq, seed=22)
    out = T.full_like(c.q, 7.0)
    ws = c.H.paged_attention_workspace(c.cache, c.batch, n_head).fill_(255)
    for _ in range(3):
        c.run(out=out, workspace=ws)
        assert not out.any() and c.H.device_status() == 0
        out.fill_(7.0)


@pytest.mark.parametrize("how", ["two slots", "one slot", "with a sound one"])
def test_pages_held_more_often_than_they_have_references(T, how):
    """Freeing what holds a page twice that has one reference: status 3, and nothing has changed."""
    import hesa_cuda as H
    from test_kv_pages_gpu import fresh, ints, same
    _, c, m = fresh(T, n_pages=300, page=4, n_slots=6, max_pages=80)
    H.kv_reserve(c, ints(T, [0, 1, 2, 5]), ints(T, [300, 33, 8, 9]))
    m.reserve([0, 1, 2, 5], [300, 33, 8, 9])
    if how == "one slot":
        m.refs[m.rows[0][70]] = 0
        m.rows[0][70] = m.rows[0][3]
    else:
        m.refs[m.rows[1][8]] = 0
        m.rows[1][8] = m.rows[0][74]
    c.table.copy_(T.tensor(m.rows, dtype=T.int32))
    c.page_refs.copy_(T.tensor(m.refs, dtype=T.int32))
    for _ in range(2):
        H.kv_free(c, ints(T, {"two slots": [1, 0], "one slot": [0], "with a sound one": [2, 0, 5, 1]}[how]))
        assert H.device_status() == 3
        H.clear_device_status()
        same(c, m)
    H.kv_free(c, ints(T, [5, 2]))
    m.free([5, 2])
    same(c, m)
    if how == "two slots":                       # with its second reference it goes
        m.refs[m.rows[0][74]] += 1
        c.page_refs.copy_(T.tensor(m.refs, dtype=T.int32))
        H.kv_free(c, ints(T, [1, 0]))
        m.free([1, 0])
        same(c, m)
    H.kv_compact(c)
    assert H.device_status() == 0


@pytest.mark.parametrize("n_head,n_kv,hd,page", [(8, 2, 128, 16), (8, 2, 64, 7), (4, 4, 256, 16)])
def test_a_capped_row_depends_on_what_it_sees_alone(T, n_head, n_kv, hd, page):
    """Scores far from zero, of hidden keys and of other rows, change no bit of a row whose own are near it."""
    new, n, cap = 150, 400, 30.0
    c = Case(T, n_head, n_kv, hd, page, [n], [new], seed=33)
    was = c.run(softcap=cap)
    j = n - 20
    c.k[0, int(c.cache.table[0, j // page]), j % page] = 3000.0
    out = c.run(softcap=cap)
    assert T.equal(out[:new - 20], was[:new - 20]) and not T.equal(out[new - 20:], was[new - 20:])
    c.q[37] *= 50.0
    again = c.run(softcap=cap)
    assert T.equal(again[:37], was[:37]) and T.equal(again[38:], out[38:]) and not T.equal(again[37], out[37])
    assert T.isfinite(again).all() and c.H.device_status() == 0


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan], ids=("inf", "-inf", "nan"))
@pytest.mark.parametrize("opts", [{}, dict(softcap=20.0), dict(window=60), dict(window=60, softcap=2.0, prefix=True), dict(slopes=True)],
                         ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("n_head,n_kv,hd,page,n,new", [(8, 2, 128, 16, 333, 1), (8, 2, 64, 5, 700, 2), (4, 1, 256, 16, 333, 3), (2, 1, 128, 64, 20011, 1),
                                                       (8, 2, 128, 16, 333, 200), (8, 2, 64, 7, 700, 65), (4, 4, 256, 16, 400, 100), (8, 1, 128, 32, 5000, 40)])
def test_a_key_that_is_not_finite(T, n_head, n_kv, hd, page, n, new, opts, bad):
    """One value of k of either sign: NaN for every row and head that sees its key, and no other row is any different."""
    c = Case(T, n_head, n_kv, hd, page, [n], [new], seed=31)
    opts = dict(opts)
    if opts.get("slopes"):
        opts["slopes"] = T.exp2(-8.0 * T.arange(1, n_head + 1, device="cuda") / n_head)
    if opts.get("prefix"):
        opts["prefix"] = T.tensor([4], dtype=T.int32, device="cuda")
    was = c.run(**opts).view(new, n_head, hd)
    assert T.isfinite(was).all()
    first = n - new
    pos = T.arange(first, n, device="cuda")
    for j, d in ((first - 3, hd - 1), (n - 1, 0), (first + new // 2, 17), (2, 5)):
        p, s = int(c.cache.table[0, j // page]), j % page
        x = c.k[0, p, s, n_kv - 1, d].item()
        c.k[0, p, s, n_kv - 1, d] = bad
        out = c.run(**opts).view(new, n_head, hd)
        c.k[0, p, s, n_kv - 1, d] = x
        sees = (j <= pos) & (j > pos - opts["window"]) if "window" in opts else j <= pos
        if "prefix" in opts:
            sees = sees | (j < 4)
        hit = T.zeros(new, n_head, dtype=T.bool, device="cuda")
        hit[:, n_head - n_head // n_kv:] = sees[:, None]
        assert T.isnan(out[hit]).all() and T.equal(out[~hit], was[~hit]), (j, d)
    assert T.equal(c.run(**opts).view(new, n_head, hd), was) and c.H.device_status() == 0


@pytest.mark.parametrize("news", [[2, 1], [150, 70]])
def test_scores_past_the_range_of_floats_are_no_keys_that_are_not_finite(T, news):
    """Finite q and k whose score is below the lowest float: the weight is 0, as it is for any score far below the best."""
    c = Case(T, 4, 2, 128, 16, [300, 90], news, seed=32)
    c.q.fill_(0.0)
    c.q[:, ::128] = 3e38
    c.k[0, :, :, :, 0] = -40000.0
    for i in range(2):
        c.k[0, int(c.cache.table[i, 0]), 1, :, 0] = 0.0     # the one key of each sequence that counts
    out = c.run().view(-1, 4, 128)
    for i in range(2):
        want = c.values[i][1].float().repeat_interleave(2, 0)
        assert T.equal(out[c.starts[i]:c.starts[i + 1]], want.expand(news[i], 4, 128))
    assert c.H.device_status() == 0


def far_apart(T, pool, stride, buf, at):
    """The pool's pages `stride` values apart in buf, layers side by side in each, from value `at` on."""
    n_layer, n_pages, page, n_kv, hd = pool.shape
    x = buf.as_strided(pool.shape, (page * n_kv * hd, stride, n_kv * hd, hd, 1), at)
    x.copy_(pool)
    return x


@pytest.fixture
def wide(T):
    """2.9e9 values of fp16: offsets that neither 31 nor 32 bits of bytes, nor 31 of values, hold."""
    buf = T.empty(11 * (1 << 28), dtype=T.float16, device="cuda")
    yield buf
    del buf
    T.cuda.empty_cache()


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens,news", [(16, 2, 128, 16, [70, 70], [1, 1]), (8, 2, 64, 7, [33, 29], [2, 1]), (4, 1, 256, 16, [70, 70], [1, 3]),
                                                           (16, 2, 128, 16, [70, 70], [40, 33]), (8, 2, 64, 7, [33, 29], [33, 20]), (4, 1, 256, 16, [75, 70], [60, 70])])
@pytest.mark.parametrize("odd", [0, 8], ids=("rows", "gaps"))
def test_pages_beyond_two_to_the_31(T, wide, n_head, n_kv, hd, page, lens, news, odd):
    """Cache write and attention over pages 2^28 values apart: as over the same pages side by side."""
    c = Case(T, n_head, n_kv, hd, page, lens, news, seed=51, spare=0)
    assert c.k.shape[1] == 10 and int(c.cache.table.max()) == 9
    H, stride = c.H, (1 << 28) + odd
    far = H.PagedKV(far_apart(T, c.k, stride, wide, 0), far_apart(T, c.v, stride, wide, 1 << 27), c.cache.table, c.cache.seq_len)
    kv = T.randn(c.n_tokens, 2 * n_kv * hd, device="cuda")
    got = []
    for cache in (c.cache, far):
        H.rope_kv_paged(cache, 0, c.batch, None, kv[:, :n_kv * hd], kv[:, n_kv * hd:], n_head)
        got.append((H.paged_attention(cache, 0, c.batch, c.q, n_head), cache.k.clone(), cache.v.clone()))
    (a, ka, va), (b, kb, vb) = got
    assert T.equal(ka.view(T.int16), kb.view(T.int16)) and T.equal(va.view(T.int16), vb.view(T.int16))
    if hd == 256 and odd and max(news) > 3:
        # heads of 256 have chunk tiles for pages of whole rows apart only; with gaps tiles of 8 rows serve them: each is within RMS of 64 bits
        assert relative(b, a.double()) <= 2 * RMS
    else:
        assert T.equal(a, b)
    assert T.isfinite(a).all() and H.device_status() == 0


def test_page_operations_beyond_two_to_the_31(T, wide):
    import hesa_cuda as H
    from test_kv_pages_gpu import Model, ints, same
    near = H.PagedKV.empty(2, 11, 8, 2, 64, 6, 6)
    near.k.normal_()
    near.v.normal_()
    far = H.PagedKV(far_apart(T, near.k, 1 << 28, wide, 0), far_apart(T, near.v, 1 << 28, wide, 1 << 27), near.table.clone(), near.seq_len.clone(),
                    near.page_refs.clone())
    m = Model(11, 8, 6, 6)
    m.reserve([0, 1], [30, 35])
    m.fork([1, 0], [2, 3])
    m.free([0])
    m.compact()
    for c in (near, far):
        H.kv_reserve(c, ints(T, [0, 1]), ints(T, [30, 35]))
        H.kv_fork(c, ints(T, [1, 0]), ints(T, [2, 3]))
        H.kv_free(c, ints(T, [0]))
        H.kv_compact(c)
        H.kv_copy_pages(c, ints(T, [1, 10]), ints(T, [9, 8]))
        same(c, m)
    assert T.equal(near.k, far.k) and T.equal(near.v, far.v) and H.device_status() == 0


@pytest.mark.parametrize("window", [1 << 30, 2 ** 31 - 1])
@pytest.mark.parametrize("news", [[9, 3], [70, 150]])
def test_the_widest_window_is_none(T, window, news):
    """Also where positions are negative (more new tokens than tokens)."""
    c = Case(T, 4, 2, 64, 8, [5, 140], news, seed=52)
    assert T.equal(c.run(window=window), c.run()) and c.H.device_status() == 0


@pytest.mark.parametrize("what", ["below", "above", "free", "short", "long"])
def test_freeing_slots_that_are_not_sound_changes_nothing(T, what):
    """Sound slots beside one with a page outside the pool, a page that is free, or a length that its row cannot have."""
    import hesa_cuda as H
    from test_kv_pages_gpu import fresh, ints, same
    _, c, m = fresh(T, n_pages=400, page=4, n_slots=60, max_pages=12)
    slots = list(range(50))
    m.reserve(slots, [1 + 7 * s % 40 for s in slots])
    m.free([20])
    m.reserve([20], [30])
    if what in ("short", "long"):
        m.len[20] = {"short": -1, "long": 49}[what]
    else:
        m.rows[20][5] = {"below": -1, "above": 400, "free": m.refs.index(0)}[what]
    before = [x[:] for x in m.rows], m.refs[:], m.len[:]
    c.table.copy_(T.tensor(m.rows, dtype=T.int32))
    c.page_refs.copy_(T.tensor(m.refs, dtype=T.int32))
    c.seq_len.copy_(T.tensor(m.len, dtype=T.int32))
    H.kv_free(c, ints(T, slots))
    assert H.device_status() == 3
    H.clear_device_status()
    same(c, m)
    assert before == (m.rows, m.refs, m.len)
    rest = [s for s in slots if s != 20]
    H.kv_free(c, ints(T, rest))
    m.free(rest)
    same(c, m)
    assert H.device_status() == 0


def test_two_host_threads_at_once(T):
    """Attention, cache write, log probabilities and page operations from two threads, each on a stream of its own."""
    import threading

    import hesa_cuda as H
    from test_kv_pages_gpu import ints
    shapes = [(16, 2, 128, 16, [900, 70, 3], [1, 2, 1]), (8, 2, 64, 7, [700, 300], [65, 300])]
    cases = [Case(T, *s, seed=61 + i) for i, s in enumerate(shapes)]
    want = [c.run() for c in cases]
    logits = [T.randn(2, 50001, device="cuda"), T.randn(1500, 321, device="cuda")]
    top = [H.token_logprobs(x, top_k=7) for x in logits]
    pages = [H.PagedKV.empty(2, 64, 8, 1, 64, 8, 16) for _ in cases]
    lists = [ints(T, x) for x in ([0, 1], [20, 33], [2, 3], [1])]
    T.cuda.synchronize()
    wrong = []

    def work(i):
        c, cache, s = cases[i], pages[i], T.cuda.Stream()
        with T.cuda.stream(s):
            for _ in range(50):
                out = c.run()
                lp = H.token_logprobs(logits[i], top_k=7)
                H.kv_reserve(cache, lists[0], lists[1])
                H.kv_fork(cache, lists[0], lists[2])
                H.kv_free(cache, lists[3])
                H.kv_compact(cache)
                H.kv_free(cache, ints(T, [0, 2, 3]))
                s.synchronize()
                if not T.equal(out, want[i]) or not all(a is None or T.equal(a, b) for a, b in zip(lp, top[i])) or bool(cache.page_refs.any()):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and H.device_status() == 0
