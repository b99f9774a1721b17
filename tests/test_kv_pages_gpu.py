"""Page operations and cache writes against a host model of the pages, and the
paged operators together: a model run in ragged chunks, with forks, against the
oracle's decode step."""
import math
import random

import numpy as np
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


class Model:
    """The page tables as the definition has them, on the host."""

    def __init__(self, n_pages, page, n_slots, max_pages):
        self.refs, self.page, self.max_pages = [0] * n_pages, page, max_pages
        self.rows, self.len = [[-1] * max_pages for _ in range(n_slots)], [0] * n_slots

    def pages(self, s):
        return -(-self.len[s] // self.page)

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, slots, add):
        for s, a in zip(slots, add):
            have = self.pages(s)
            self.len[s] += a
            for j in range(have, self.pages(s)):
                self.rows[s][j] = self.take()

    def free(self, slots):
        for s in slots:
            for j in range(self.pages(s)):
                self.refs[self.rows[s][j]] -= 1
                self.rows[s][j] = -1
            self.len[s] = 0

    def fork(self, src, dst):
        """The copies made: (page from, page to, places)."""
        made = []
        for a, b in zip(src, dst):
            full, tail = divmod(self.len[a], self.page)
            for j in range(full):
                self.rows[b][j] = self.rows[a][j]
                self.refs[self.rows[a][j]] += 1
            if tail:
                self.rows[b][full] = self.take()
                made.append((self.rows[a][full], self.rows[b][full], tail))
            self.len[b] = self.len[a]
        return made

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        new = dict(zip(movers, holes))
        for s in range(len(self.rows)):
            for j in range(self.pages(s)):
                self.rows[s][j] = new.get(self.rows[s][j], self.rows[s][j])
        for a, b in new.items():
            self.refs[a], self.refs[b] = 0, self.refs[a]
        return live, list(new.items())


def ints(T, v):
    return T.tensor(list(v), dtype=T.int32, device="cuda")


def same(cache, m):
    assert cache.seq_len.tolist() == m.len
    assert cache.page_refs.tolist() == m.refs
    assert cache.table.tolist() == m.rows


def fresh(T, n_layer=2, n_pages=40, page=8, n_kv=2, hd=64, n_slots=6, max_pages=12):
    import hesa_cuda as H
    c = H.PagedKV.empty(n_layer, n_pages, page, n_kv, hd, n_slots, max_pages)
    c.k.normal_()
    c.v.normal_()
    return H, c, Model(n_pages, page, n_slots, max_pages)


@pytest.mark.parametrize("page,n_pages,n_slots,seed", [(8, 40, 6, 0), (1, 300, 9, 1), (5, 2500, 40, 2), (64, 30, 5, 3), (16, 5000, 1500, 4)])
def test_random_histories(T, page, n_pages, n_slots, seed):
    """Long random runs of all operations: tables, references and page contents as the model's."""
    max_pages = 12
    H, c, m = fresh(T, 2, n_pages, page, 1, 64, n_slots, max_pages)
    r = random.Random(seed)
    k, v = c.k.clone(), c.v.clone()

    def copy(pairs):
        for a, b, places in pairs:
            k[:, b, :places] = k[:, a, :places]
            v[:, b, :places] = v[:, a, :places]
    for step in range(60):
        free_pages = sum(x == 0 for x in m.refs)
        used = [s for s in range(n_slots) if m.len[s]]
        empty = [s for s in range(n_slots) if not m.len[s]]
        op = r.choice(("reserve", "reserve", "free", "fork", "compact"))
        if op == "reserve":
            slots = r.sample(range(n_slots), r.randrange(1, n_slots + 1))
            add, left = [], free_pages
            for s in slots:
                a = r.randrange(0, min(max_pages * page - m.len[s], 3 * page) + 1)
                need = -(-(m.len[s] + a) // page) - m.pages(s)
                if need > left:
                    a, need = 0, 0
                left -= need
                add.append(a)
            m.reserve(slots, add)
            H.kv_reserve(c, ints(T, slots), ints(T, add))
        elif op == "free" and used:
            slots = r.sample(used, r.randrange(1, min(len(used), 1 + n_slots // 3) + 1))
            m.free(slots)
            H.kv_free(c, ints(T, slots))
        elif op == "fork" and used and empty:
            dst = r.sample(empty, r.randrange(1, len(empty) + 1))[:free_pages]
            if not dst:
                continue
            src = [r.choice(used) for _ in dst]
            copy(m.fork(src, dst))
            H.kv_fork(c, ints(T, src), ints(T, dst))
        elif op == "compact":
            n = ints(T, [-1])
            live, moves = m.compact()
            H.kv_compact(c, n_live=n)
            copy([(a, b, page) for a, b in moves])
            assert n.item() == live
        same(c, m)
        assert T.equal(c.k, k) and T.equal(c.v, v)
    assert H.device_status() == 0


def test_more_slots_than_a_block_has_threads(T):
    H, c, m = fresh(T, 1, 9000, 4, 1, 64, 3000, 4)
    slots = list(range(2999, -1, -1))
    add = [1 + (s * 7) % 9 for s in slots]
    m.reserve(slots, add)
    H.kv_reserve(c, ints(T, slots), ints(T, add))
    same(c, m)
    gone = slots[::3]
    m.free(gone)
    H.kv_free(c, ints(T, gone))
    same(c, m)
    src = [s for s in slots if s % 3 == 1][:len(gone)]
    k = c.k.clone()
    for a, b, n in m.fork(src, gone[:len(src)]):
        k[:, b, :n] = k[:, a, :n]
    H.kv_fork(c, ints(T, src), ints(T, gone[:len(src)]))
    same(c, m)
    assert T.equal(c.k, k) and H.device_status() == 0


def test_a_call_that_cannot_be_carried_out_changes_nothing(T):
    H, c, m = fresh(T, n_pages=10, page=4, n_slots=4, max_pages=6)
    H.kv_reserve(c, ints(T, [0, 2]), ints(T, [9, 16]))
    m.reserve([0, 2], [9, 16])
    before = c.k.clone()
    for code, call in ((5, lambda: H.kv_reserve(c, ints(T, [1]), ints(T, [13]))),               # 4 pages, 3 are free
                       (3, lambda: H.kv_reserve(c, ints(T, [1, 1]), ints(T, [1, 1]))),          # the same slot twice
                       (3, lambda: H.kv_reserve(c, ints(T, [4]), ints(T, [1]))), (3, lambda: H.kv_reserve(c, ints(T, [-1]), ints(T, [1]))),
                       (3, lambda: H.kv_reserve(c, ints(T, [1]), ints(T, [-1]))), (3, lambda: H.kv_reserve(c, ints(T, [2]), ints(T, [9]))),
                       (3, lambda: H.kv_reserve(c, ints(T, [1]), ints(T, [2 ** 31 - 1]))),
                       (3, lambda: H.kv_free(c, ints(T, [0, 0]))), (3, lambda: H.kv_free(c, ints(T, [7]))),
                       (3, lambda: H.kv_fork(c, ints(T, [0]), ints(T, [2]))),                   # a target in use
                       (3, lambda: H.kv_fork(c, ints(T, [0, 0]), ints(T, [1, 1]))), (3, lambda: H.kv_fork(c, ints(T, [0, 1]), ints(T, [1, 3]))),
                       (3, lambda: H.kv_fork(c, ints(T, [9]), ints(T, [1]))),
                       (3, lambda: H.kv_copy_pages(c, ints(T, [0, 1]), ints(T, [8, 8]))), (3, lambda: H.kv_copy_pages(c, ints(T, [0, 8]), ints(T, [8, 9]))),
                       (3, lambda: H.kv_copy_pages(c, ints(T, [10]), ints(T, [8]))), (3, lambda: H.kv_copy_pages(c, ints(T, [0]), ints(T, [-1])))):
        call()
        assert H.device_status() == code
        H.clear_device_status()
        same(c, m)
    assert T.equal(c.k, before)
    m.reserve([1], [10])                     # what is left is given out
    H.kv_reserve(c, ints(T, [1]), ints(T, [10]))
    same(c, m)
    # a table that holds a page of nobody: compacting and freeing leave it alone
    c.table[1, 0] = 99
    H.kv_compact(c)
    assert H.device_status() == 3
    H.clear_device_status()
    H.kv_free(c, ints(T, [1]))
    assert H.device_status() == 3 and c.page_refs.tolist() == m.refs
    H.clear_device_status()


@pytest.mark.parametrize("handle", [False, True], ids=("object", "handle"))
def test_page_operations_on_another_stream(T, handle):
    """A stream given as torch's object or as a handle, with the cache's own scratch: ordered there, results as ever."""
    H, c, m = fresh(T)
    lists = [ints(T, v) for v in ([0, 3], [20, 9], [3, 0], [1, 4], [3])]
    k = c.k.clone()
    T.cuda.synchronize()
    side = T.cuda.Stream()
    on = side.cuda_stream if handle else side
    H.kv_reserve(c, lists[0], lists[1], stream=on)
    H.kv_fork(c, lists[2], lists[3], stream=on)
    H.kv_free(c, lists[4], stream=on)
    H.kv_compact(c, stream=on)
    side.synchronize()
    m.reserve([0, 3], [20, 9])
    pairs = m.fork([3, 0], [1, 4])
    m.free([3])
    for a, b, n in pairs:
        k[:, b, :n] = k[:, a, :n]
    for a, b in m.compact()[1]:
        k[:, b] = k[:, a]
    same(c, m)
    assert T.equal(c.k, k) and H.device_status() == 0


def test_copy_pages_and_empty_lists(T):
    H, c, _ = fresh(T, n_layer=3, page=5)
    k, v = c.k.clone(), c.v.clone()
    src, dst = [3, 3, 17, 0], [4, 20, 39, 8]
    H.kv_copy_pages(c, ints(T, src), ints(T, dst))
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    H.kv_copy_pages(c, ints(T, []), ints(T, []))
    H.kv_free(c, ints(T, []))
    H.kv_fork(c, ints(T, []), ints(T, []))
    H.kv_reserve(c, ints(T, []), ints(T, []))
    H.kv_compact(c)                            # nothing in use
    H.kv_fork(c, ints(T, [0]), ints(T, [1]))   # a copy of nothing
    H.kv_free(c, ints(T, [2]))
    assert T.equal(c.k, k) and T.equal(c.v, v) and H.device_status() == 0 and not c.page_refs.any()


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens,news", [
    (8, 2, 64, 16, [40, 1, 300], [40, 1, 77]), (4, 4, 128, 5, [12, 900], [0, 700]), (2, 1, 256, 24, [33], [1]),
    (32, 32, 128, 16, [1024, 16], [1000, 16])])
def test_store_matches_rope_and_kv_store(T, n_head, n_kv, hd, page, lens, news):
    """Every row as the one-token kernels write it, bit for bit; every other place and row as it was."""
    import hesa_cuda as H
    n_slots, width = len(lens) + 1, -(-max(lens) // page)
    c = H.PagedKV.empty(2, sum(-(-n // page) for n in lens) + 2, page, n_kv, hd, n_slots, width)
    slots = [len(lens) - i for i in range(len(lens))]
    H.kv_reserve(c, ints(T, slots), ints(T, lens))
    c.k.normal_()
    c.v.normal_()
    k0, v0 = c.k.clone(), c.v.clone()
    starts = [0] + [sum(news[:i + 1]) for i in range(len(news))]
    n = starts[-1] + 3
    qkv = T.randn(n, (n_head + 2 * n_kv) * hd, device="cuda")
    a, b = n_head * hd, (n_head + n_kv) * hd
    was = qkv.clone()
    table = T.from_numpy(H.rope_table(max(lens), hd)).cuda()
    batch = H.TokenBatch(ints(T, starts), n, max(news), max(lens), slots=ints(T, slots))
    H.rope_kv_paged(c, 1, batch, qkv[:, :a], qkv[:, a:b], qkv[:, b:], n_head, rope_table=table)
    rows = c.table.tolist()
    kc, vc = T.zeros(1, n_kv * hd, dtype=T.float16, device="cuda"), T.zeros(1, n_kv * hd, dtype=T.float16, device="cuda")
    want = was.clone()
    for i, s in enumerate(slots):
        for t in range(news[i]):
            if news[i] > 50 and t % 37 and t != news[i] - 1:
                p = lens[i] - news[i] + t      # spot checks of a long chunk; its other places are copied over
                k0[1, rows[s][p // page], p % page] = c.k[1, rows[s][p // page], p % page]
                v0[1, rows[s][p // page], p % page] = c.v[1, rows[s][p // page], p % page]
                want[starts[i] + t] = qkv[starts[i] + t]
                continue
            p, r = lens[i] - news[i] + t, starts[i] + t
            H.rope(want[r, :a], n_head, hd, table, pos=p)
            kk = was[r, a:b].clone()
            H.rope(kk, n_kv, hd, table, pos=p)
            H.kv_store(kk, was[r, b:].clone(), kc, vc, 1, pos=0)
            k0[1, rows[s][p // page], p % page] = kc.view(n_kv, hd)
            v0[1, rows[s][p // page], p % page] = vc.view(n_kv, hd)
    assert T.equal(qkv, want) and T.equal(c.k, k0) and T.equal(c.v, v0)
    assert H.device_status() == 0
    # without a table: k and v as they are, q not looked at
    H.rope_kv_paged(c, 0, batch, None, was[:, a:b], was[:, b:], n_head)
    i, s = len(slots) - 1, slots[-1]
    p = lens[i] - 1
    assert T.equal(c.k[0, rows[s][p // page], p % page].reshape(-1), was[starts[i + 1] - 1, a:b].half())
    assert H.device_status() == 0


def test_store_skips_rows_without_a_place(T):
    import hesa_cuda as H
    c = H.PagedKV.empty(1, 8, 4, 1, 64, 2, 4)
    H.kv_reserve(c, ints(T, [0, 1]), ints(T, [6, 6]))
    c.table[0, 1] = 77                       # its last two tokens have no page
    table = T.from_numpy(H.rope_table(6, 64)).cuda()
    x = T.randn(12, 3 * 64, device="cuda")
    was = x.clone()
    batch = H.TokenBatch(ints(T, [0, 6, 12]), 12, 6, 16)
    H.rope_kv_paged(c, 0, batch, x[:, :64], x[:, 64:128], x[:, 128:], 1, rope_table=table)
    assert H.device_status() == 3
    H.clear_device_status()
    assert T.equal(x[4:6], was[4:6])
    assert T.equal(c.v[0, c.table[1, 0].item(), 0, 0], was[6, 128:].half())
    # more new tokens than tokens: the first rows have negative positions
    c.table[0, 1] = 1
    c.seq_len[0] = 3
    H.rope_kv_paged(c, 0, batch, x[:, :64], x[:, 64:128], x[:, 128:], 1)
    assert H.device_status() == 3
    H.clear_device_status()
    assert T.equal(c.v[0, c.table[0, 0].item(), 2, 0], was[5, 128:].half())


def test_graph_of_a_beam_step(T):
    """Free, fork, reserve, store and attend captured as one graph and replayed: as the eager calls."""
    import hesa_cuda as H

    def start():
        T.manual_seed(3)
        c = H.PagedKV.empty(2, 30, 8, 2, 64, 6, 6)
        c.k.normal_()
        c.v.normal_()
        H.kv_reserve(c, ints(T, [0, 1, 2, 3]), ints(T, [13, 20, 8, 31]))
        return c
    x = T.randn(3, 8 * 64, device="cuda")
    free, src, dst, one = ints(T, [3]), ints(T, [0, 0]), ints(T, [4, 5]), ints(T, [1, 1, 1])
    grow = ints(T, [0, 4, 5])

    def step(c, batch, ws, pws, q, out):
        H.kv_free(c, free, workspace=pws)
        H.kv_fork(c, src, dst, workspace=pws)
        H.kv_reserve(c, grow, one, workspace=pws)
        H.rope_kv_paged(c, 1, batch, q[:, :256], q[:, 256:384], q[:, 384:], 4)
        H.paged_attention(c, 1, batch, q[:, :256], 4, out=out, workspace=ws)
    results = []
    for captured in (False, True):
        c = start()
        batch = H.TokenBatch(ints(T, [0, 1, 2, 3]), 3, 1, 48, slots=grow)
        ws, pws, out = H.paged_attention_workspace(c, batch, 4), H.kv_pages_workspace(c), T.zeros(3, 256, device="cuda")
        if captured:
            H.device_status()
            g = T.cuda.CUDAGraph()
            with T.cuda.graph(g):
                step(c, batch, ws, pws, x, out)
            g.replay()
        else:
            step(c, batch, ws, pws, x, out)
        T.cuda.synchronize()
        results.append((out, c.k, c.v, c.table, c.seq_len, c.page_refs))
    assert all(T.equal(a, b) for a, b in zip(*results)) and H.device_status() == 0
    assert results[0][4].tolist() == [14, 20, 8, 0, 14, 14]


def test_model_in_chunks_matches_the_oracle(T):
    """Two sequences of one two-layer model, run as a chunk, forked, and continued token by token in one batch:
    the logits of every position as the oracle's decode step gives them, and its log probabilities."""
    import hesa_cuda as H
    from oracle import oracle as O
    qt, L, D, NH, NKV, HD, F, V, page = H.Q8_0, 2, 256, 4, 2, 64, 512, 320, 5
    QD, KD = NH * HD, NKV * HD

    def w(n, k, seed):
        return O.quantize(qt, O.gaussian((n, k), 0.05, seed))
    layers = [dict(qkv=w(QD + 2 * KD, D, 10 * i + 1), o=w(D, QD, 10 * i + 2), gu=w(2 * F, D, 10 * i + 3), down=w(D, F, 10 * i + 4),
                   n1=1 + O.gaussian((D,), 0.1, 10 * i + 5), n2=1 + O.gaussian((D,), 0.1, 10 * i + 6)) for i in range(L)]
    out_norm, w_out, emb = 1 + O.gaussian((D,), 0.1, 91), w(V, D, 92), O.gaussian((V, D), 1.0, 93)
    tokens = [[(7 * i + 3) % V for i in range(21)], None]
    tokens[1] = tokens[0][:13] + [(11 * i + 5) % V for i in range(8)]     # the second shares the first 13

    # 64-bit model: fp16 cache, everything else in doubles
    dq = lambda b, k: O.dequantize(qt, b, k).astype(np.float64)  # noqa: E731
    W = [{n: dq(l[n], F if n == "down" else QD if n == "o" else D) for n in ("qkv", "o", "gu", "down")} | {"n1": l["n1"], "n2": l["n2"]} for l in layers]
    rope = H.rope_table(32, HD).astype(np.float64)

    def norm(x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * g

    def rot(x, pos):
        c, s = rope[pos, :HD // 2], rope[pos, HD // 2:]
        a, b = x[..., :HD // 2], x[..., HD // 2:]
        return np.concatenate([a * c - b * s, a * s + b * c], -1)

    def reference(seq):
        x = emb[seq].astype(np.float64)
        for l in W:
            qkv = norm(x, l["n1"]) @ l["qkv"].T
            n = len(seq)
            q = np.stack([rot(qkv[p, :QD].reshape(NH, HD), p) for p in range(n)])
            k = np.stack([rot(qkv[p, QD:QD + KD].reshape(NKV, HD), p) for p in range(n)]).astype(np.float16).astype(np.float64)
            v = qkv[:, QD + KD:].reshape(n, NKV, HD).astype(np.float16).astype(np.float64)
            a = np.zeros((n, NH, HD))
            for p in range(n):
                for h in range(NH):
                    s = k[:p + 1, h * NKV // NH] @ q[p, h] / math.sqrt(HD)
                    e = np.exp(s - s.max())
                    a[p, h] = e @ v[:p + 1, h * NKV // NH] / e.sum()
            x = x + a.reshape(n, QD) @ l["o"].T
            gu = norm(x, l["n2"]) @ l["gu"].T
            g = gu[:, :F]
            x = x + (g / (1 + np.exp(-g)) * gu[:, F:]) @ l["down"].T
        return norm(x, out_norm) @ dq(w_out, D).T

    dev = lambda a: T.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    G = [{n: dev(l[n]) for n in l} for l in layers]
    g_out, g_norm, g_rope = dev(w_out), dev(out_norm.astype(np.float32)), dev(H.rope_table(32, HD))
    cache = H.PagedKV.empty(L, 20, page, NKV, HD, 4, 6)

    def forward(slots, starts, ids):
        n = len(ids)
        x = dev(emb[ids].astype(np.float32))
        batch = H.TokenBatch(ints(T, starts), n, max(b - a for a, b in zip(starts, starts[1:])), 30, slots=ints(T, slots))
        for i, l in enumerate(G):
            qkv = H.qmatvec(qt, l["qkv"], H.rms_norm(x, l["n1"].float()))
            H.rope_kv_paged(cache, i, batch, qkv[:, :QD], qkv[:, QD:QD + KD], qkv[:, QD + KD:], NH, rope_table=g_rope)
            a = H.paged_attention(cache, i, batch, qkv[:, :QD], NH)
            x = H.add(x, H.qmatvec(qt, l["o"], a))
            gu = H.qmatvec(qt, l["gu"], H.rms_norm(x, l["n2"].float()))
            x = H.add(x, H.qmatvec(qt, l["down"], H.silu_mul(gu[:, :F].contiguous(), gu[:, F:].contiguous())))
        return H.qmatvec(qt, g_out, H.rms_norm(x, g_norm))

    got = {0: [], 1: []}
    H.kv_reserve(cache, ints(T, [2]), ints(T, [13]))
    first = forward([2], [0, 13], tokens[0][:13])
    got[0] += list(first)
    got[1] += list(first)
    H.kv_fork(cache, ints(T, [2]), ints(T, [0]))
    H.kv_reserve(cache, ints(T, [3]), ints(T, [9]))        # a third sequence comes and goes, leaving holes
    H.kv_free(cache, ints(T, [3]))
    for t in range(13, 21):
        if t == 16:
            H.kv_compact(cache)
        H.kv_reserve(cache, ints(T, [2, 0]), ints(T, [1, 1]))
        y = forward([2, 0], [0, 1, 2], [tokens[0][t], tokens[1][t]])
        got[0].append(y[0])
        got[1].append(y[1])
    for i in (0, 1):
        ref = reference(tokens[i])
        logits = T.stack(got[i])
        d = logits.cpu().numpy() - ref
        # fp16 roundings of k and v may fall either way where fp32 and 64 bits differ: 2^-11 of single values
        assert np.linalg.norm(d) / np.linalg.norm(ref) <= 1e-4
        lp, ent, top, tlp = H.token_logprobs(logits, ints(T, tokens[i][1:] + [0]), top_k=3)
        x = logits.double()
        want = T.log_softmax(x, 1)
        assert float((lp.double() - want.gather(1, T.tensor(tokens[i][1:] + [0], device="cuda")[:, None])[:, 0]).abs().max()) <= 1e-5
        assert T.equal(top.long(), T.topk(x, 3).indices)
        assert float((ent.double() + (want.exp() * want).sum(1)).abs().max()) <= 1e-5
    assert H.device_status() == 0
