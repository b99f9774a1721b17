"""Attention over a cache in 4 bits against its definition in 64 bits on the values that the cache holds. Those are fp16
numbers exactly, so the bounds of the fp16 cache's attention (paged_bounds) hold: blocks are of 32 keys in two sums of
16, and q is held in 22 bits instead of 21."""
import math

import pytest
import torch

from kv4_model import Case, pools, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def H():
    assert torch.cuda.is_available()
    import hesa_cuda
    hesa_cuda.lib()
    hesa_cuda.clear_device_status()
    return hesa_cuda


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens", [
    (32, 32, 128, 16, [2048]),              # the 7B layout
    (64, 8, 128, 16, [1, 17, 300, 5, 1023]),
    (8, 2, 64, 5, [37, 1, 160]),            # pages that end inside a block of keys
    (4, 4, 256, 24, [300, 33]),
    (12, 2, 128, 1, [65, 2]),               # a page for each token, groups of six
    (32, 2, 64, 128, [129, 128, 127]),      # groups of sixteen: two tiles of rows
    (8, 1, 128, 64, [20011, 3]),            # split over the keys
    (2, 1, 256, 48, [9001]),
    (3, 3, 64, 16, [31, 32, 33, 63, 64, 65]),
    (40, 40, 64, 16, [100]),                # more heads than a CTA has warps
    (9, 9, 256, 16, [40, 1]),
    (1, 1, 64, 7, [1]),
])
def test_next_token(n_head, n_kv, hd, page, lens):
    Case(n_head, n_kv, hd, page, lens, [1] * len(lens), seed=n_head + hd).check()


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens", [
    (32, 32, 128, 16, [2] * 74),            # a CTA for each (sequence, group of heads)
    (32, 32, 128, 16, [1, 2, 3, 40, 33] * 3),
    (32, 32, 64, 16, [7] * 40),
    (32, 32, 128, 16, [9001]),
    (64, 8, 128, 16, [30000]),
    (64, 8, 128, 16, [8000, 3, 300, 77, 1, 5000, 64, 20]),
    (4, 4, 256, 16, [2] * 148),
    (4, 4, 256, 16, [12000]),
    (12, 12, 128, 24, [300, 1, 33]),        # heads that are no power of two, in groups of six and three
    (8, 1, 128, 24, [2, 3, 40]),            # a warp with a block, and fifteen of its head without one
])
def test_groups_of_heads(n_head, n_kv, hd, page, lens):
    Case(n_head, n_kv, hd, page, lens, [1] * len(lens), seed=len(lens) + hd).check()


@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 2, 64), (12, 2, 128), (8, 4, 256)])
def test_scratch_may_hold_anything(H, n_head, n_kv, hd):
    """What the workspace of a chunk holds, NaN among it, changes no bit: places of the fp16 copy that no row sees are zeros."""
    c = Case(n_head, n_kv, hd, 24, [301, 90, 1000, 129], [70, 90, 100, 1], seed=hd)
    ws = H.paged_attention_workspace(c.cache, c.batch, n_head)
    prefix = torch.tensor([3, 0, 200, 40], dtype=torch.int32, device="cuda")
    for o in (dict(), dict(window=40, prefix=prefix), dict(window=1)):
        outs = []
        for byte in (0, 0x7e, 0xfc):   # fp16 0x7e7e is NaN
            ws.fill_(byte)
            outs.append(c.run(workspace=ws, **o).clone())
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and bool(torch.isfinite(outs[0]).all())
    assert H.device_status() == 0


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens,news", [
    (4, 4, 128, 16, [512], [512]),                     # a whole prompt
    (8, 2, 128, 16, [700, 50, 33, 257], [130, 50, 0, 1]),
    (16, 4, 64, 24, [301, 7, 1000], [100, 7, 333]),
    (4, 2, 256, 16, [150, 90], [70, 90]),
    (6, 2, 64, 7, [130, 129, 128], [5, 3, 2]),
    (6, 2, 64, 7, [130, 129, 128], [50, 3, 2]),
    (32, 1, 128, 16, [300, 40], [1, 1]),               # 32 heads on one: four tiles of rows
    (65, 1, 64, 16, [300, 1], [1, 1]),                 # and so many that they are a chunk
    (2, 2, 256, 16, [700, 300], [64, 3]),              # the most rows that are tiles of eight
    (2, 2, 256, 16, [700, 300], [65, 3]),
    (2, 2, 128, 5, [400], [8]),                        # eight new tokens are rows of one tile
    (4, 1, 128, 16, [400, 1], [3, 1]),
])
def test_chunks(n_head, n_kv, hd, page, lens, news):
    Case(n_head, n_kv, hd, page, lens, news, seed=hd + len(lens)).check()


OPTIONS = [dict(softcap=20.0), dict(window=50), dict(window=1), dict(scale=0.3), dict(slopes=True), dict(prefix=[200, 0, 31]),
           dict(softcap=30.0, window=33, slopes=True, prefix=[90, 300, 2])]


@pytest.mark.parametrize("opts", OPTIONS)
@pytest.mark.parametrize("new", [1, 10, 40])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_options(opts, new, hd):
    lens = [333, 300, 41]
    c = Case(8, 2, hd, 12, lens, [new, min(new, 5), new], seed=hd + new)
    o = dict(opts)
    if o.get("slopes"):
        o["slopes"] = torch.exp2(-torch.arange(1, 9, device="cuda", dtype=torch.float32))
    if "prefix" in o:
        o["prefix"] = torch.tensor(o["prefix"], dtype=torch.int32, device="cuda")
    ref = dict(o)
    if "prefix" in ref:   # a prefix ends with the sequence
        ref["prefix"] = torch.minimum(o["prefix"].cpu(), torch.tensor(lens, dtype=torch.int32))
    r, bound = c.exact(**ref)
    out = c.run(**o)
    assert bool(((out.view_as(r).double() - r).abs() <= bound).all())
    assert c.H.device_status() == 0


@pytest.mark.parametrize("new", [1, 7, 64])
def test_layers_strides_slots_and_gaps(new):
    for kw in (dict(layers=3), dict(layers=2, inside=True), dict(gap=24), dict(slots=[4, 0, 2]), dict(layers=2, gap=8, inside=True, slots=[1, 3, 0])):
        c = Case(6, 3, 64, 7, [100, 33, 64], [new, 1, new], seed=new, **kw)
        wide = torch.full((c.n_tokens, c.q.shape[1] + 12), math.nan, device="cuda")
        wide[:, 8:-4] = c.q
        c.q = wide[:, 8:-4]
        out = torch.full((c.n_tokens + 3, c.q.shape[1] + 4), 7.0, device="cuda")
        c.check(run=lambda: c.run(out=out[: c.n_tokens, :-4]))
        assert bool((out[c.n_tokens:] == 7).all()) and bool((out[:, -4:] == 7).all())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 24, 40])
def test_what_is_not_finite_stays_where_it_is_seen(hd, new):
    """A k group with scale NaN makes the rows that see it NaN, a v group its 32 dims of those rows; nothing else."""
    c = Case(4, 2, hd, 16, [100, 70], [new, new], seed=hd)
    ref, bound = c.exact(window=20)
    page = int(c.table[0, 85 // 16])
    for pool, all_dims in ((2, True), (3, False)):
        kept = c.pools[pool].clone()
        c.pools[pool][0, page, 85 % 16, 1, 1] = math.nan     # sequence 0, key 85, kv head 1, dims 32 .. 63
        out = c.run(window=20).view_as(ref)
        c.pools[pool].copy_(kept)
        pos = torch.arange(100 - new, 100, device="cuda")
        sees = torch.zeros(2 * new, 4, hd, dtype=torch.bool, device="cuda")
        rows = torch.nonzero((pos >= 85) & (pos < 105))[:, 0]
        sees[rows, 2:, :] = True
        if not all_dims:
            sees[:, :, :32] = False
            sees[:, :, 64:] = False
        assert bool(torch.isnan(out[sees]).all()) and bool(sees.any())
        assert bool(((out.double() - ref).abs()[~sees] <= bound[~sees]).all())
    # the new tokens' later keys are hidden from the earlier rows
    if new > 1:
        page = int(c.table[0, 99 // 16])
        c.pools[3][0, page, 99 % 16] = math.nan
        out = c.run(window=20).view_as(ref)
        assert bool(torch.isnan(out[new - 1]).all())
        assert bool(((out.double() - ref).abs()[: new - 1] <= bound[: new - 1]).all())


@pytest.mark.parametrize("new", [1, 24, 40])
def test_rows_of_q_that_are_not_finite_and_of_any_size(new):
    c = Case(4, 2, 128, 16, [90, 60], [new, new], seed=3)
    c.q[0] *= 2.0 ** 90
    c.q[1, :128] *= 2.0 ** -120
    c.q[-1, 130] = math.inf
    ref, bound = c.exact()
    out = c.run().view_as(ref)
    assert bool(torch.isnan(out[-1, 1]).all())
    # scores of 2^90 are an argmax, whose bound says nothing, and the infinite row has none
    assert bool(torch.isfinite(out[0]).all())
    some = torch.ones(2 * new, 4, dtype=torch.bool, device="cuda")
    some[0] = some[-1, 1] = False
    assert bool(((out.double() - ref).abs()[some] <= bound[some]).all())


def test_empty_sequences_rows_that_see_nothing_and_parts_of_a_batch(H):
    for new, g in ((1, 2), (20, 2), (20, 8)):
        c = Case(2 * g, 2, 64, 8, [50, 30, 25], [new, 0, new], seed=new)
        c.check()
        # shorter than its new tokens: positions below 0 see nothing and give zeros
        if new > 1:
            c.seq_len[2] = 12
            c.lens, c.keys[2], c.values[2] = [50, 30, 12], c.keys[2][:12], c.values[2][:12]
            out = c.check()
            assert bool((out[new: new + 8] == 0).all())
        # rows in front of the first and behind the last sequence of a part stay
        out = torch.full_like(c.q, 5.0)
        part = H.TokenBatch(c.q_start[2:], c.n_tokens, max(c.news), 50, slots=torch.tensor([2], dtype=torch.int32, device="cuda"))
        H.paged_attention(c.cache, 0, part, c.q, 2 * g, out=out)
        assert bool((out[:new] == 5).all()) and bool((out[new:] != 5).any())
    empty = H.TokenBatch(torch.zeros(2, dtype=torch.int32, device="cuda"), 0, 0, 5)
    assert H.paged_attention(c.cache, 0, empty, c.q[:0], 16).shape == (0, 1024)


@pytest.mark.parametrize("new,g", [(1, 2), (20, 2), (20, 4)])
def test_tables_that_are_not_sound(H, new, g):
    c = Case(2 * g, 2, 64, 8, [50, 30], [new, new], seed=5)
    ref, bound = c.exact()
    good = int(c.table[0, 3])
    for bad in (-1, c.cache.n_pages, 1 << 30):
        c.table[0, 3] = bad
        out = c.run().view_as(ref)
        assert H.device_status() == 3
        H.clear_device_status()
        assert bool(torch.isfinite(out).all())
        assert bool(((out[new:].double() - ref[new:]).abs() <= bound[new:]).all())
        # the page reads as zeros
        keys, vals = c.keys[0].clone(), c.values[0].clone()
        c.keys[0][24:32], c.values[0][24:32] = 0, 0
        r2, b2 = c.exact()
        assert bool(((out.double() - r2).abs() <= b2).all())
        c.keys[0], c.values[0] = keys, vals
    c.table[0, 3] = good
    for bad in (-1, 51, 1 << 29):
        c.seq_len[1] = bad
        out = torch.full_like(c.q, 5.0)
        c.run(out=out)
        assert H.device_status() == 3
        H.clear_device_status()
        assert bool((out[new:] == 5).all()) and bool(((out[:new].view_as(ref[:new]).double() - ref[:new]).abs() <= bound[:new]).all())
        c.seq_len[1] = 30
    c.q_start[1] = c.n_tokens + 1
    c.run()
    assert H.device_status() == 3
    H.clear_device_status()


@pytest.mark.parametrize("new", [1, 20])
def test_a_captured_step_serves_later_lengths(H, new):
    c = Case(8, 2, 128, 16, [300, 200, 80], [new, new, new], seed=8)
    ws = H.paged_attention_workspace(c.cache, c.batch, 8)
    out = torch.empty_like(c.q)
    c.run(out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out, workspace=ws)
    for lens in ([300, 200, 80], [new, 33, 80], [150, 199, 0 if new == 1 else 20]):
        c.seq_len.copy_(torch.tensor(lens, dtype=torch.int32))
        d = Case.__new__(Case)
        d.__dict__.update(c.__dict__)
        d.lens, d.keys, d.values = lens, [k[:n] for k, n in zip(c.keys, lens)], [v[:n] for v, n in zip(c.values, lens)]
        ws.fill_(255)   # scratch need not be set
        graph.replay()
        d.check(run=lambda: out)


def test_streams_repeats_and_shared_workspaces(H):
    """Calls of several shapes on one stream share a workspace; two streams with workspaces of their own agree with it, bit by bit, every time."""
    cs = [Case(64, 8, 128, 16, [900, 30, 411], [1, 1, 1], seed=1), Case(8, 2, 64, 8, [300], [64], seed=2), Case(4, 4, 256, 16, [77, 500], [1, 1], seed=3)]
    n = max(H.paged_attention_workspace(c.cache, c.batch, c.n_head).numel() for c in cs)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    first = [c.run(workspace=ws).clone() for c in cs]
    for _ in range(3):
        for c, f in zip(cs, first):
            assert torch.equal(c.run(workspace=ws), f)
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    outs = [c.run(stream=s) for c, s in zip(cs, streams)]
    torch.cuda.synchronize()
    for o, f in zip(outs, first):
        assert torch.equal(o, f)


def test_more_sequences_than_the_scratch_holds(H):
    """Chunks of sequences whose fp16 copies take more than 1 GB: a few at a time, the workspace bounded."""
    lens = [40000, 3, 39000, 500, 40000, 40000, 1]
    c = Case(16, 16, 128, 64, lens, [2, 3, 70, 70, 0, 1, 1], seed=4)
    nb = H.paged_attention_workspace(c.cache, c.batch, 16).numel()
    assert (1 << 29) < nb < (1 << 30) + (64 << 20)
    slopes = torch.full((16,), 0.01, device="cuda")
    prefix = torch.tensor([0, 1, 50, 0, 7, 3000, 0], dtype=torch.int32, device="cuda")
    c.check(window=3000, slopes=slopes, prefix=prefix)
    c.slots = torch.tensor([6, 5, 4, 3, 2, 1, 0], dtype=torch.int32, device="cuda")
    c.batch = H.TokenBatch(c.q_start, c.n_tokens, 70, 40000, slots=c.slots)
    c.lens, c.keys, c.values = c.lens[::-1], c.keys[::-1], c.values[::-1]
    c.check(window=3000, slopes=slopes)


def test_pools_of_more_than_4_gb(H):
    """Codes and scales whose offsets pass 32 bits, in bytes and in values."""
    n_pages, page, n_kv, hd = 11000, 128, 8, 256
    k, v, ks, vs = pools(4, n_pages, page, n_kv, hd)
    assert k.stride(0) * 3 + k.stride(1) * (n_pages - 1) > 1 << 32
    small = Case(16, n_kv, hd, page, [300, 128], [1, 1], seed=9)
    pages = [n_pages - 1, 5, n_pages - 2, n_pages - 3]
    table = torch.tensor([pages[:3], [pages[3], -1, -1]], dtype=torch.int32, device="cuda")
    for big, few in zip((k, v, ks, vs), small.pools):
        for i in range(3):
            big[3, pages[i]] = few[0, int(small.table[0, i])]
        big[3, pages[3]] = few[0, int(small.table[1, 0])]
    small.cache, small.layer = H.PagedKV4(k, v, ks, vs, table, small.seq_len), 3
    small.check()
    small.news, small.starts, small.n_tokens = [40, 20], [0, 40, 60], 60
    small.q_start.copy_(torch.tensor([0, 40, 60], dtype=torch.int32))
    small.q = torch.randn(60, 16 * hd, device="cuda")
    small.batch = H.TokenBatch(small.q_start, 60, 40, 300)
    small.check()


def test_random_ragged_batches(H):
    import random
    r = random.Random(11)
    for i in range(40):
        kv = r.choice((1, 2, 3, 5, 8, 17))
        g = r.choice((1, 1, 2, 3, 8, 9))
        hd = r.choice((64, 128, 256))
        n = r.randrange(1, 9)
        new = r.choice((1, 1, 2, 7, 33, 66))
        lens = [r.randrange(1, r.choice((3, 70, 900))) for _ in range(n)]
        news = [min(x, r.randrange(0, new + 1)) for x in lens]
        if not any(news):
            news[0] = 1
        o = dict(window=r.choice((0, 0, 1, 30, 500)), softcap=r.choice((0.0, 15.0)))
        Case(kv * g, kv, hd, r.choice((1, 3, 8, 16, 24, 100)), lens, news, seed=100 + i, gap=r.choice((0, 8))).check(**o)


def test_values_are_what_attention_reads(H):
    """One key: the result is its value, to the 22 bits of P's halves."""
    c = Case(2, 2, 128, 16, [1], [1], seed=6)
    out = c.run().view(2, 128)
    assert torch.allclose(out, c.values[0][0], rtol=2.0 ** -21, atol=0)
    assert torch.equal(values(c.pools[0][0, int(c.table[0, 0]), 0], c.pools[2][0, int(c.table[0, 0]), 0]), c.keys[0][0])
