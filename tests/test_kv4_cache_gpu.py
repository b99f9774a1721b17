"""Writing into a cache in 4 bits and reading it back, bit for bit against the format's definition on the host."""
import math

import pytest
import torch

from kv4_model import Case, quantize, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def H():
    assert torch.cuda.is_available()
    import hesa_cuda
    hesa_cuda.lib()
    hesa_cuda.clear_device_status()
    return hesa_cuda


def rotated(x, table, pos):
    """Rotate-half rope of x [n, heads, hd] at positions pos, products and sums rounded one by one."""
    hd = x.shape[-1]
    co, si = table[pos, : hd // 2][:, None], table[pos, hd // 2:][:, None]
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    return torch.cat([a * co - b * si, a * si + b * co], -1)


def stored(c, layer):
    """What the pages hold for each sequence's tokens: (k codes, k scales, v codes, v scales)."""
    out = []
    for i, n in enumerate(c.lens):
        j = torch.arange(n, device="cuda")
        page, place = c.table[c.slot_of[i]][j // c.page].long(), j % c.page
        out.append([c.pools[x][layer, page, place] for x in (0, 2, 1, 3)])
    return out


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens,news,kw", [
    (8, 2, 64, 16, [40, 7, 100], [1, 1, 1], {}),
    (4, 4, 128, 5, [40, 7, 100], [12, 0, 100], dict(layers=2)),
    (6, 3, 256, 1, [9, 4], [5, 4], dict(gap=8)),
    (1, 1, 64, 7, [300], [299], dict(layers=3, inside=True)),
    (5, 5, 128, 24, [50, 20, 30], [20, 20, 7], dict(slots=[2, 0, 5])),
    (32, 32, 128, 16, [700], [650], {}),
])
@pytest.mark.parametrize("rope", [True, False])
def test_write_and_read(H, n_head, n_kv, hd, page, lens, news, kw, rope):
    c = Case(n_head, n_kv, hd, page, lens, news, seed=hd + page, **kw)
    before = [p.clone() for p in c.pools]
    n = c.n_tokens
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(n + 2, (n_head + 2 * n_kv) * hd + 8, generator=g, device="cuda")
    a, b, e = n_head * hd, (n_head + n_kv) * hd, (n_head + 2 * n_kv) * hd
    was = qkv.clone()
    table = torch.from_numpy(H.rope_table(max(lens), hd)).cuda() if rope else None
    x = qkv[:n]
    H.rope_kv_paged(c.cache, c.layer, c.batch, x[:, :a], x[:, a:b], x[:, b:e], n_head, rope_table=table)
    k, v = H.kv_read(c.cache, c.layer, c.batch)
    assert H.device_status() == 0
    pos = torch.cat([torch.arange(m - t, m) for m, t in zip(lens, news)]).cuda()
    q, kk, vv = was[:n, :a].view(n, n_head, hd), was[:n, a:b].view(n, n_kv, hd), was[:n, b:e].view(n, n_kv, hd)
    if rope:
        q, kk = rotated(q, table, pos), rotated(kk, table, pos)
    assert torch.equal(x[:, :a], q.reshape(n, a))
    assert torch.equal(qkv[:, a:], was[:, a:]) and torch.equal(qkv[n:], was[n:])
    kc, ks = quantize(kk)
    vc, vs = quantize(vv)
    assert torch.equal(k.view(n, n_kv, hd), values(kc, ks)) and torch.equal(v.view(n, n_kv, hd), values(vc, vs))
    for i, got in enumerate(stored(c, c.layer)):
        lo, hi = c.starts[i], c.starts[i + 1]
        for x_, want in zip(got, (kc, ks, vc, vs)):
            assert torch.equal(x_[lens[i] - news[i]:], want[lo:hi])
    # nothing else has changed, in any layer
    for i in range(len(lens)):
        j = torch.arange(lens[i] - news[i], lens[i], device="cuda")
        pg, pl = c.table[c.slot_of[i]][j // page].long(), j % page
        for p, w in zip(c.pools, before):
            p[c.layer, pg, pl] = w[c.layer, pg, pl]
    for p, w in zip(c.pools, before):
        assert torch.equal(p.view(torch.uint8) if p.dtype == torch.uint8 else p.view(torch.int16), w.view(torch.uint8) if w.dtype == torch.uint8 else w.view(torch.int16))


def one_row(H, x):
    """x [32 m] as v of one token of one head of 64 dims or more: the scale and codes it gets."""
    hd = x.numel()
    c = Case(1, 1, hd, 4, [1], [1], seed=0)
    H.rope_kv_paged(c.cache, 0, c.batch, None, x.view(1, hd), x.view(1, hd), 1)
    codes, scales, vc, vs = stored(c, 0)[0]
    assert torch.equal(codes, vc) and torch.equal(scales.view(torch.int16), vs.view(torch.int16))
    return codes[0, 0], scales[0, 0]


def test_edges_of_the_format(H):
    f = torch.float32
    r = torch.randn(64, generator=torch.Generator().manual_seed(2))
    rows = [torch.zeros(64), -torch.zeros(64), r * 1e-3, r * 1e-5, r * 2.0 ** -20, r * 1e-7, r * 2.0 ** -140, r * 3000, r * 5000,
            torch.tensor([2.0, -2.0] * 32), torch.tensor([-2.0, 2.0] * 32), torch.full((64,), 1.0), torch.linspace(-1, 1, 64),
            torch.linspace(-8, 8, 64) * 2.0 ** -17, torch.linspace(-8, 7.9, 64) * 2.0 ** -24, torch.full((64,), 21824.0), torch.full((64,), 21824.002),
            torch.full((64,), -21824.0), torch.full((64,), 65504.0), torch.full((64,), 3e38), torch.full((64,), 2.0 ** -149)]
    for bad in (math.nan, math.inf, -math.inf):
        x = r.clone()
        x[40] = bad
        rows.append(x)
        rows.append(torch.full((64,), bad))
    for i, x in enumerate(rows):
        x = x.to(f).cuda()
        codes, scales = one_row(H, x)
        want_c, want_s = quantize(x.view(1, 64))
        assert torch.equal(codes, want_c[0]), i
        same = (scales == want_s[0]) | (torch.isnan(scales) & torch.isnan(want_s[0]))
        assert bool(same.all()), i
        # the promise of the format: every value is an fp16 number
        val = values(codes, scales)
        assert bool(((val.half().float() == val) | torch.isnan(val)).all()), i
    assert H.device_status() == 0


def test_nearest_value_of_the_grid(H):
    """A value is off by half a step of its group's scale, or, at the end away from the largest, by one step, and the
    rounding of 1 / scale, x / scale and the sum (3 times 2^-24 of 16 steps)."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(1, 256, generator=g, device="cuda")
    codes, scales = one_row(H, x)
    val, d = values(codes, scales), scales.float().abs().repeat_interleave(32)
    off = (val - x[0]).abs() / d
    inner = (x[0] / scales.float().repeat_interleave(32)) < 7.5
    assert float(off[inner].max()) <= 0.5 + 8 / 256 + 16 * 3 * 2.0 ** -24 and float(off.max()) <= 1 + 8 / 256
    assert bool((val.half().float() == val).all())


def test_rows_without_a_place(H):
    """Positions outside the rope table or the pool are skipped; reading them gives zeros; rows of no sequence stay."""
    c = Case(2, 1, 64, 4, [10, 6], [3, 2], seed=3)
    x = torch.randn(5, 4 * 64, device="cuda")
    table = torch.from_numpy(H.rope_table(9, 64)).cuda()   # position 9 has no row
    before = [p.clone() for p in c.pools]
    q0 = x[2, :128].clone()
    H.rope_kv_paged(c.cache, 0, c.batch, x[:, :128], x[:, 128:192], x[:, 192:], 2, rope_table=table)
    assert H.device_status() == 3
    H.clear_device_status()
    page, place = int(c.table[0, 9 // 4]), 9 % 4
    assert all(torch.equal(p[0, page, place], w[0, page, place]) for p, w in zip(c.pools, before)) and torch.equal(x[2, :128], q0)
    keep = int(c.table[1, 1])
    c.table[1, 1] = 99
    k = torch.full((5, 64), 3.0, device="cuda")
    kk, vv = H.kv_read(c.cache, 0, c.batch, k=k)
    assert H.device_status() == 3 and bool((kk[3:] == 0).all()) and bool((vv[3:] == 0).all()) and bool((kk[:3] != 0).any())
    H.clear_device_status()
    c.table[1, 1] = keep
    c.seq_len[0] = -5
    k.fill_(3.0)
    H.kv_read(c.cache, 0, c.batch, k=k)
    assert H.device_status() == 3 and bool((k[:3] == 3).all()) and bool((k[3:] != 3).any())
    H.clear_device_status()
    part = H.TokenBatch(c.q_start[1:], 5, 3, 10, slots=torch.tensor([1], dtype=torch.int32, device="cuda"))
    k.fill_(3.0)
    H.kv_read(c.cache, 0, part, k=k)
    assert bool((k[:3] == 3).all()) and H.device_status() == 0


def test_write_in_a_captured_graph_and_on_another_stream(H):
    c = Case(4, 2, 128, 16, [50, 33], [1, 1], seed=4)
    table = torch.from_numpy(H.rope_table(64, 128)).cuda()
    x = torch.randn(2, 8 * 128, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    w = x.clone()
    s.wait_stream(torch.cuda.current_stream())
    H.rope_kv_paged(c.cache, 0, c.batch, w[:, :512], w[:, 512:768], w[:, 768:], 4, rope_table=table, stream=s)
    k, v = H.kv_read(c.cache, 0, c.batch, stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    w2 = x.clone()
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        H.rope_kv_paged(c.cache, 0, c.batch, w2[:, :512], w2[:, 512:768], w2[:, 768:], 4, rope_table=table)
        H.kv_read(c.cache, 0, c.batch, k=k2, v=v2)
    w2.copy_(x)
    graph.replay()
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(w[:, :512], w2[:, :512])
    c.seq_len.copy_(torch.tensor([20, 17], dtype=torch.int32))
    w2.copy_(x)
    graph.replay()
    kk, _ = quantize(rotated(x[:, 512:768].view(2, 2, 128), table, torch.tensor([19, 16], device="cuda")))
    assert torch.equal(c.pools[0][0, int(c.table[0, 1]), 3], kk[0]) and torch.equal(c.pools[0][0, int(c.table[1, 1]), 0], kk[1])
    assert H.device_status() == 0
