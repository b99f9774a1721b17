"""The attention's results value by value, each within a bound of its own row, head and dim, and as a whole to a few
2^-20: what a kernel that held q or P in one half would miss by far."""
import pytest

from paged_bounds import RMS, head, relative
from test_paged_attention_gpu import Case, T  # noqa: F401  (T: the fixture)

pytestmark = pytest.mark.gpu


def definition(T, c, softcap=0.0, window=0, slopes=None, prefix=None, scale=None):
    out = T.zeros(c.n_tokens, c.n_head, c.hd, dtype=T.float64, device="cuda")
    bound = T.zeros_like(out)
    q = c.q.view(c.n_tokens, c.n_head, c.hd)
    for i in range(c.n_seq):
        lo, hi, n = c.starts[i], c.starts[i + 1], c.lens[i]
        pos = T.arange(n - (hi - lo), n, device="cuda")
        for h in range(c.n_head if hi > lo and n else 0):
            kv = h * c.n_kv // c.n_head
            out[lo:hi, h], bound[lo:hi, h] = head(q[lo:hi, h], c.keys[i][:, kv], c.values[i][:, kv], pos, scale, softcap, window,
                                                  0.0 if slopes is None else float(slopes[h]), 0 if prefix is None else int(prefix[i]))
    return out, bound


SHAPES = [
    (8, 2, 64, 5, [700, 33], [1, 2]),                 # tiles of 8 rows
    (8, 8, 128, 16, [2048], [1]),
    (16, 2, 128, 16, [900, 5000], [1, 1]),            # cut over the keys
    (4, 1, 256, 16, [333, 1200], [2, 1]),
    (12, 3, 256, 24, [900], [4]),
    (8, 2, 64, 16, [1000, 64], [100, 64]),            # tiles of 128 rows
    (8, 2, 64, 7, [700], [65]),
    (4, 4, 128, 16, [2048], [130]),
    (8, 1, 128, 32, [5000], [40]),                    # cut over the keys
    (6, 2, 128, 7, [400, 129], [129, 128]),
    (4, 2, 256, 16, [600, 90], [100, 90]),
    (4, 1, 256, 64, [3000], [70]),
]


@pytest.mark.parametrize("opts", [{}, dict(softcap=20.0), dict(softcap=1.5), dict(window=100, prefix=True), dict(slopes=True), dict(scale=0.02)],
                         ids=lambda o: "-".join(map(str, o.items())) or "plain")
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:4])))
def test_every_value_and_the_whole(T, shape, opts):
    c = Case(T, *shape, seed=41)
    opts = dict(opts)
    if opts.get("slopes"):
        opts["slopes"] = T.exp2(-8.0 * T.arange(1, c.n_head + 1, device="cuda") / c.n_head)
    if opts.get("prefix"):
        opts["prefix"] = T.tensor([min(n, 40) for n in c.lens], dtype=T.int32, device="cuda")
    ref, bound = definition(T, c, **opts)
    out = c.run(**opts).view(c.n_tokens, c.n_head, c.hd)
    over = ((out.double() - ref).abs() / bound).max()
    assert float(over) <= 1, f"{float(over):.2f} times its bound"
    rel = relative(out, ref)
    assert rel <= RMS, f"{rel:.2e}"
    assert c.H.device_status() == 0


@pytest.mark.parametrize("shape", [(4, 2, 128, 16, [500], [37]), (4, 2, 64, 7, [500], [1]), (4, 1, 256, 16, [500], [20]), (4, 4, 128, 16, [500], [300])],
                         ids=lambda s: "-".join(map(str, s[:3])))
def test_each_row_has_its_own_scale(T, shape):
    """Rows of q from 1e-38 to 1e4, side by side: each within its own bound, and the small ones to their last bits."""
    c = Case(T, *shape, seed=42)
    q = c.q.view(c.n_tokens, c.n_head, c.hd)
    for i, f in enumerate((1e-38, 1e-30, 1e-3, 2000.0, 1e4)):
        q[i % c.n_tokens, i % c.n_head] *= f
    ref, bound = definition(T, c)
    out = c.run().view(c.n_tokens, c.n_head, c.hd)
    assert ((out.double() - ref).abs() <= bound).all() and c.H.device_status() == 0
    for i in (0, 1, 2):
        r, h = i % c.n_tokens, i % c.n_head
        assert relative(out[r, h], ref[r, h]) <= RMS


@pytest.mark.parametrize("opts", [{}, dict(window=70, prefix=True), dict(slopes=True), dict(scale=1e3)], ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("shape", [(4, 2, 128, 16, [500], [50]), (2, 2, 64, 7, [500, 3], [2, 1]), (4, 1, 256, 16, [500], [40]), (4, 4, 64, 16, [500], [300]),
                                   (8, 1, 128, 16, [4000], [32])], ids=lambda s: "-".join(map(str, s[:3])))
def test_scores_of_any_size(T, shape, opts):
    """Every row's scores at another power of two, up to 2^110: past 2^24 the shift of P and the maximum no longer fit into
    one float. No infinite P and no row without one: every result is a mean of values, within its bound where that says
    something."""
    c = Case(T, *shape, seed=43)
    opts = dict(opts)
    if opts.get("slopes"):
        opts["slopes"] = T.exp2(20 - 8.0 * T.arange(1, c.n_head + 1, device="cuda") / c.n_head)
    if opts.get("prefix"):
        opts["prefix"] = T.tensor([min(n, 40) for n in c.lens], dtype=T.int32, device="cuda")
    q = c.q.view(c.n_tokens * c.n_head, c.hd)
    top = 95 if "scale" in opts else 105
    q *= T.exp2((T.arange(len(q), device="cuda") * 37 % 16 * (top / 15.0)).floor())[:, None] if len(q) < 100 else \
        T.exp2((T.arange(len(q), device="cuda") * 37 % (top + 1)).float())[:, None]
    ref, bound = definition(T, c, **opts)
    out = c.run(**opts).view(c.n_tokens, c.n_head, c.hd)
    assert T.isfinite(out).all()
    small = bound < 8
    assert ((out.double() - ref).abs() <= bound)[small].all()
    vmax = float(max(v.abs().max() for v in c.values if len(v)))
    assert float(out.abs().max()) <= vmax * (1 + 2.0 ** -10)      # always a mean of values
    assert c.H.device_status() == 0


@pytest.mark.parametrize("new", [2, 80])
def test_a_small_cap_on_scores_of_any_size(T, new):
    """Keys of zeros beside scores near a float's end: a capped score of 0 stays 0, the others are the cap. All weights are
    alike to 2^-19 then, and the sums round (n / 16 + 16) 2^-23: 6.1e-6 of values below 8, on both sides of the quotient."""
    cap = 1e-6
    c = Case(T, 4, 2, 128, 16, [300], [new], seed=44)
    for j in (0, 17, 250):
        c.k[0, int(c.cache.table[0, j // 16]), j % 16] = 0
        c.keys[0][j] = 0
    c.q *= 5e37
    assert T.isfinite(c.q).all()
    ref, bound = definition(T, c, softcap=cap)
    out = c.run(softcap=cap).view(c.n_tokens, c.n_head, c.hd)
    assert ((out.double() - ref).abs() <= bound.clamp(max=1e-4)).all() and c.H.device_status() == 0
