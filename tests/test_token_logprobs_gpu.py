"""Log probabilities, entropy and top alternatives against 64 bits.

Tolerances: e^(x - m) in fp32 has a relative error of 2^-21 plus 2^-23 |x - m| (the
scaled difference is rounded once), the sum over V terms in lanes and trees adds at
most (log2 V + V / 8192) 2^-24; log z then has that absolute error, x - m one
rounding more: at spreads below 60, |error| <= 2^-21 + 60 2^-23 + 2^-20 + 60 2^-24 < 2e-5.
The entropy adds the same relative error of w / z, whose size is below 60: 60 times
2^-21 more, < 6e-5."""
import math

import pytest

pytestmark = pytest.mark.gpu
TOL, ENT = 2e-5, 6e-5


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available()
    import hesa_cuda
    hesa_cuda.lib()
    hesa_cuda.clear_device_status()
    return torch


def check(T, x, tokens, k, **kw):
    import hesa_cuda as H
    lp, ent, ids, top = H.token_logprobs(x, tokens, top_k=k, **kw)
    d = x.double()
    want = T.log_softmax(d, 1)
    t = want.gather(1, tokens.long().clamp(0)[:, None])[:, 0]
    fin = T.isfinite(t)
    assert T.equal(fin, T.isfinite(lp)) and T.equal(lp[~fin], t[~fin].float())
    assert float((lp.double() - t)[fin].abs().max()) <= TOL if fin.any() else True
    h = -(want.exp() * want.masked_fill(want == -math.inf, 0)).sum(1)
    assert float((ent.double() - h).abs().max()) <= ENT
    order = T.sort(d, dim=1, descending=True, stable=True).indices[:, :k]
    assert T.equal(ids.long(), order)
    w = want.gather(1, order)
    ok = T.isfinite(w)
    assert T.equal(T.isfinite(top), ok)
    assert not ok.any() or float((top.double() - w)[ok].abs().max()) <= TOL
    assert H.device_status() == 0
    return lp, ent, ids, top


@pytest.mark.parametrize("n,vocab,k", [(1, 32000, 8), (1, 1, 1), (3, 2, 2), (1, 131071, 32), (7, 33, 32), (5, 4099, 5), (300, 1000, 1),
                                       (2, 262144, 20), (1500, 257, 3), (64, 32001, 0), (1025, 50, 4)])
@pytest.mark.parametrize("spread", [1.0, 6.0])
def test_random_rows(T, n, vocab, k, spread):
    g = T.Generator(device="cuda").manual_seed(n + vocab)
    x = T.randn(n, vocab, generator=g, device="cuda") * spread
    tokens = T.randint(0, vocab, (n,), generator=g, device="cuda", dtype=T.int32)
    check(T, x, tokens, k)


@pytest.mark.parametrize("order", ["up", "down", "same", "steps", "zeros"])
@pytest.mark.parametrize("vocab", [4096, 50001])
def test_orders_and_ties(T, order, vocab):
    """Rows in ascending order (every value enters the list), and rows of equal values: the lower id first."""
    i = T.arange(vocab, device="cuda", dtype=T.float32)
    x = {"up": i * 1e-3 - 20, "down": 20 - i * 1e-3, "same": i * 0 + 2.5, "steps": T.floor(((i * 7919) % vocab) / 300),
         "zeros": T.where(i % 2 == 0, 0.0, -0.0)}[order]
    x = T.stack([x, x.roll(17), x - 3])
    check(T, x, T.tensor([0, vocab - 1, vocab // 2], dtype=T.int32, device="cuda"), 32)


def test_strides_and_alignment(T):
    """Rows of every alignment; columns behind a row's vocabulary are not read."""
    for off in range(4):
        buf = T.full((3, 1007), math.nan, device="cuda")
        x = buf[:, off:off + 1001]
        x.copy_(T.randn(3, 1001, device="cuda"))
        check(T, x, T.tensor([0, 1000, 500], dtype=T.int32, device="cuda"), 6)
    one = T.randn(40000, device="cuda")
    check(T, one[3:33000][None], T.tensor([5], dtype=T.int32, device="cuda"), 4)


def test_ruled_out_tokens_and_lowest_values(T):
    x = T.randn(6, 20000, device="cuda")
    x[0, 1:] = -math.inf
    x[1, ::2] = -math.inf
    x[2, 100:] = T.finfo(T.float32).min
    x[3] = T.finfo(T.float32).min
    x[4, :19998] = -math.inf
    x[5, 5] = 40.0
    lp, ent, ids, top = check(T, x, T.tensor([0, 2, 3, 9, 0, 5], dtype=T.int32, device="cuda"), 5)
    assert ent[0] == 0 and lp[0] == 0 and top[0, 1] == -math.inf and ids[0].tolist() == [0, 1, 2, 3, 4]
    assert lp[1] == -math.inf and lp[4] == -math.inf


def test_rows_without_a_distribution_and_tokens_without_a_place(T):
    import hesa_cuda as H
    for vocab in (1000, 100000):                       # one block, and split rows
        x = T.randn(5, vocab, device="cuda")
        x[0] = -math.inf
        x[1, 7] = math.nan
        x[2, vocab - 1] = math.inf
        lp, ent, ids, top = H.token_logprobs(x, T.tensor([3, 3, 3, -1, 8], dtype=T.int32, device="cuda"), top_k=2)
        assert lp[0] == -math.inf and ent[0] == 0 and ids[0].tolist() == [0, 1] and (top[0] == -math.inf).all()
        assert T.isnan(lp[1:3]).all() and T.isnan(ent[1:3]).all() and T.isnan(top[1:3]).all()
        assert lp[3] == 0 and T.isfinite(lp[4]) and T.isfinite(ent[3:]).all()
        assert H.device_status() == 0
        lp, _, _, _ = H.token_logprobs(x[3:], T.tensor([vocab, -2], dtype=T.int32, device="cuda"))
        assert T.isnan(lp).all() and H.device_status() == 3
        H.clear_device_status()


def test_workspace_stream_and_graph(T):
    """One workspace for shapes of both kinds, a call on another stream, and a captured call on new logits."""
    import hesa_cuda as H
    a, b = T.randn(1, 100000, device="cuda"), T.randn(2000, 500, device="cuda")
    ta, tb = T.tensor([77], dtype=T.int32, device="cuda"), T.zeros(2000, dtype=T.int32, device="cuda")
    ws = H.token_logprobs_workspace(1, 100000, 32)
    for _ in range(3):
        check(T, a, ta, 32, workspace=ws)
        check(T, b, tb, 2, workspace=ws)
        check(T, a, ta, 3, workspace=ws)
    want = H.token_logprobs(a, ta, top_k=9)
    s = T.cuda.Stream()
    T.cuda.synchronize()
    got = H.token_logprobs(a, ta, top_k=9, stream=s)
    T.cuda.synchronize()
    assert all(T.equal(x, y) for x, y in zip(want, got))
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        got = H.token_logprobs(a, ta, top_k=9, workspace=ws)
    for seed in range(3):
        a.normal_()
        g.replay()
        T.cuda.synchronize()
        assert all(T.equal(x, y) for x, y in zip(H.token_logprobs(a, ta, top_k=9), got))


def test_refusals_of_the_binding(T):
    import hesa_cuda as H
    x = T.randn(4, 100, device="cuda")
    t = T.zeros(4, dtype=T.int32, device="cuda")
    for bad in (lambda: H.token_logprobs(x.half(), t), lambda: H.token_logprobs(x.cpu(), t), lambda: H.token_logprobs(x, t.long()),
                lambda: H.token_logprobs(x, t[:3]), lambda: H.token_logprobs(x.t(), t), lambda: H.token_logprobs(x[0], t)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(H.HesaError):
        H.token_logprobs(x, t, top_k=33)
    lp, ent, ids, top = H.token_logprobs(x)
    assert lp is None and ids.shape == (4, 0) and top.shape == (4, 0)


@pytest.mark.parametrize("vocab,k", [(300000, 32), (131072, 7), (9000, 20)])
def test_large_values_side_by_side(T, vocab, k):
    """The largest values of a row all where one thread, or one block of a split row, reads; and everywhere but there."""
    x = T.randn(4, vocab, device="cuda")
    x[0, 128:640] += 50
    x[1, ::256] += 50
    x[2] = T.arange(vocab, device="cuda") % 251
    x[3] = (T.arange(vocab, device="cuda") // 4 % 97).float()
    check(T, x, T.tensor([130, 1, 250, 0], dtype=T.int32, device="cuda"), k)
    wide = x.repeat(300, 1)      # whole rows a block
    check(T, wide, T.zeros(1200, dtype=T.int32, device="cuda"), k)
