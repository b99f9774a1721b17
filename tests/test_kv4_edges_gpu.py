"""Edges of the cache in 4 bits: chunks that take several passes, rows that see nothing, pools of one page,
windows near 2^31, scales at ties."""
import math

import pytest
import torch

import kv4_model
from kv4_model import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def H():
    assert torch.cuda.is_available()
    import hesa_cuda
    hesa_cuda.lib()
    hesa_cuda.clear_device_status()
    return hesa_cuda


def bounded(c, max_len):
    """The case with tables and a batch for sequences of up to max_len tokens."""
    H = c.H
    pages = -(-max_len // c.page)
    c.table = torch.nn.functional.pad(c.table, (0, pages - c.table.shape[1]), value=-1).contiguous()
    c.cache = H.PagedKV4(*c.pools, c.table, c.seq_len, c.refs)
    c.batch = H.TokenBatch(c.q_start, c.n_tokens, max(c.news), max_len, slots=c.slots)
    return c


@pytest.mark.parametrize("n_head,n_kv,hd,max_len,lens,news", [
    (64, 8, 128, 131072, [300, 100, 2111], [100, 100, 100]),                                      # 2 + 1 sequences
    (64, 8, 128, 30000, [500, 64, 70, 90, 64, 333, 80, 64, 1500], [64] * 9),                       # 8 + 1
    (32, 32, 128, 32768, [300, 256, 257, 512, 700], [256, 256, 1, 30, 256]),                       # 2 + 2 + 1
    (64, 8, 128, 16384, [70 + 13 * i for i in range(16)] + [900], [64] * 17),                      # 16 + 1
    (16, 4, 256, 131072, [600, 100, 300], [200, 40, 130]),                                         # 2 + 1, in 64 keys a block
])
def test_the_last_pass_of_a_chunk_is_split_over_more_keys(n_head, n_kv, hd, max_len, lens, news):
    """Sequences whose fp16 copies take more than 1 GB by the host's bound: the last pass has fewer of them, so that their keys
    are split, which needs room in the workspace."""
    c = bounded(Case(n_head, n_kv, hd, 64, lens, news, seed=len(lens)), max_len)
    c.check()
    ws = c.H.paged_attention_workspace(c.cache, c.batch, n_head)
    ws.fill_(0x7e)
    c.check(run=lambda **o: c.run(workspace=ws, **o), window=50)


@pytest.mark.parametrize("n_head,new", [(2, 9), (4, 9), (4, 30), (16, 20)])
def test_a_row_that_sees_nothing_gives_zeros_whatever_its_q(H, n_head, new):
    """Rows of negative positions, some not finite, beside rows of the same tile that see keys."""
    c = Case(n_head, 2, 128, 8, [5, 40], [new, 3], seed=new)
    want = c.run().clone()
    for bad in (math.nan, math.inf, -math.inf):
        c.q[: new - 5: 2, ::7] = bad
        c.q[new - 4, 0] = bad     # this one sees two keys
        for o in (dict(), dict(softcap=9.0), dict(slopes=torch.ones(n_head, device="cuda"))):
            out = c.run(**o)
            assert not bool(out[: new - 5].any())
            assert bool(torch.isnan(out[new - 4, :128]).all()) and bool(torch.isfinite(out[new - 4, 128:]).all())
            assert bool(torch.isfinite(out[new - 3:]).all())
            if not o:
                assert torch.equal(out[new - 3:], want[new - 3:])
    assert H.device_status() == 0


@pytest.mark.parametrize("layers,page,n_kv,hd", [(1, 1, 1, 64), (3, 1, 1, 64), (2, 5, 1, 128), (1, 3, 3, 64), (2, 1, 1, 256)])
@pytest.mark.parametrize("inside", [False, True])
def test_a_pool_of_one_page(H, layers, page, n_kv, hd, inside):
    """Its pages need no stride: a page whose groups are no multiple of 8 is one all the same."""
    c = Case(2 * n_kv, n_kv, hd, page, [page], [1], seed=page, layers=layers, spare=0, inside=inside)
    assert c.cache.n_pages == 1
    c.check()
    for cache in (H.PagedKV4.empty(layers, 1, page, n_kv, hd, 2, 1), c.cache):
        cache.seq_len.zero_()
        cache.page_refs.zero_()
        H.kv_reserve(cache, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), page, dtype=torch.int32, device="cuda"))
        batch = H.TokenBatch(torch.tensor([0, page], dtype=torch.int32, device="cuda"), page, page, page)
        g = torch.Generator(device="cuda").manual_seed(1)
        k, v = (torch.randn(page, n_kv * hd, generator=g, device="cuda") for _ in range(2))
        for layer in range(layers):
            H.rope_kv_paged(cache, layer, batch, None, k, v, 2 * n_kv)
            for got, x in zip(H.kv_read(cache, layer, batch), (k, v)):
                assert torch.equal(got, kv4_model.values(*kv4_model.quantize(x.view(page, n_kv, hd))).view(page, -1))
    assert H.device_status() == 0


@pytest.mark.parametrize("window", [1 << 30, 2 ** 31 - 1])
@pytest.mark.parametrize("n_head,news", [(4, [9, 3]), (4, [70, 150]), (16, [20, 20])])
def test_the_widest_window_is_none(H, window, n_head, news):
    """Also where positions are negative (more new tokens than tokens), whatever scratch holds."""
    c = Case(n_head, 2, 64, 8, [5, 140], news, seed=52)
    ws = H.paged_attention_workspace(c.cache, c.batch, n_head)
    ws.fill_(0x7e)   # fp16 0x7e7e is NaN
    want = c.run()
    assert bool(torch.isfinite(want).all()) and torch.equal(c.run(window=window, workspace=ws), want) and H.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_scales_between_two_numbers_go_to_the_even_one(H, hd):
    """m / -8 half a step above 128 .. 255 in the last of 8 bits, of all sizes; the format's model on the CPU, where powers of
    two are exact."""
    rows = []
    g = torch.Generator().manual_seed(3)
    for e in list(range(-24, 5)) + [-30, -17]:
        for n in (128, 129, 130, 200, 201, 254, 255):
            x = (torch.rand(hd, generator=g) * 1.9 - 0.95) * n * 2.0 ** e
            x[int(torch.randint(0, hd, (1,), generator=g))] = -8 * (n + 0.5) * 2.0 ** e * (1 - 2 * (n & 1))
            x[int(torch.randint(0, hd, (1,), generator=g))] = 8 * (n + 0.5) * 2.0 ** e * (1 - 2 * (n & 1))
            rows.append(x)
    x = torch.stack(rows)
    n = len(rows)
    c = Case(1, 1, hd, 16, [n], [n], seed=0)
    H.rope_kv_paged(c.cache, 0, c.batch, None, x.cuda(), -x.cuda(), 1)
    for got, y in zip(H.kv_read(c.cache, 0, c.batch), (x, -x)):
        # the largest, above 2720, are NaN
        assert torch.allclose(got.cpu(), kv4_model.values(*kv4_model.quantize(y)), rtol=0, atol=0, equal_nan=True)
    assert H.device_status() == 0
