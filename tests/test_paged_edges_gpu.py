"""GPU tests of the paged operators at the edges of what their contract allows."""
import math  # noqa: F401

import pytest

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
