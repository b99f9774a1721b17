"""The tolerances of the attention's precision tests, on a model of the kernels: two halves of q and P are within them,
and either's high half alone is not."""
import math

import pytest
import torch

from paged_bounds import RMS, halves, head, high_half, relative


def inputs(rows, n, hd, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(n, hd, generator=g).half(), torch.randn(n, hd, generator=g).half()
    return torch.randn(rows, hd, generator=g) * 1.3, k, v, torch.arange(n - rows, n)


@pytest.mark.parametrize("opts", [{}, dict(softcap=20.0), dict(window=100, prefix=9), dict(slope=0.05)], ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("rows,n,hd", [(1, 333, 64), (3, 333, 256), (1, 2048, 128), (2, 5000, 128), (65, 700, 64), (130, 2048, 128), (100, 600, 256), (40, 5000, 128)])
def test_one_half_is_not_enough(rows, n, hd, opts):
    worst = {}
    for seed in range(8 if rows < 10 else 2):      # as many heads
        q, k, v, pos = inputs(rows, n, hd, 100 * seed + n + hd)
        ref, bound = head(q, k, v, pos, **opts)
        forms = {"both": dict(q_as=lambda x: halves(x, True), p_as=lambda x: halves(x, False)),
                 "no low q": dict(q_as=lambda x: high_half(x, True)), "no low p": dict(p_as=lambda x: high_half(x, False)),
                 "no low q to nearest": dict(q_as=lambda x: x.float().mul(2.0 ** 10).half().double() / 2.0 ** 10),
                 "no low p to nearest": dict(p_as=lambda x: (x.float() * 2.0 ** 14).half().double() / 2.0 ** 14)}
        for name, f in forms.items():
            out, _ = head(q, k, v, pos, **opts, **f)
            worst.setdefault(name, []).append((relative(out, ref), float(((out - ref).abs() / bound).max())))
    both = worst.pop("both")
    assert max(r for r, _ in both) < RMS / 4 and max(b for _, b in both) < 1
    for name, got in worst.items():
        # a call's result is all of its heads together
        assert math.sqrt(sum(r * r for r, _ in got) / len(got)) > 4 * RMS, name


def test_a_row_of_zeros_is_out_of_bounds():
    """A tiny row of q weighs its keys alike; leaving it out is an error, next to rows of any size."""
    q, k, v, pos = inputs(3, 500, 128, 5)
    q[0] *= 1e-30
    q[2] *= 2000.0
    ref, bound = head(q, k, v, pos)
    assert (bound[0] < 1e-5).all() and float((ref[0].abs() / bound[0]).median()) > 1000


def test_the_definition_is_the_loop():
    """Against sums written out, for every mask."""
    q, k, v, pos = inputs(4, 23, 64, 7)
    for opts in ({}, dict(softcap=3.0), dict(window=5, prefix=2), dict(slope=0.3, prefix=23), dict(scale=0.7)):
        out, bound = head(q, k, v, pos, **opts)
        for r in range(4):
            p, ws = int(pos[r]), []
            for j in range(23):
                s = float(q[r].double() @ k[j].double()) * opts.get("scale", 0.125)
                if "softcap" in opts:
                    s = 3.0 * math.tanh(s / 3.0)
                s -= opts.get("slope", 0.0) * abs(p - j)
                seen = (j <= p and ("window" not in opts or j > p - 5)) or j < opts.get("prefix", 0)
                ws.append(math.exp(s) if seen else 0.0)
            want = sum(x * v[j].double() for j, x in enumerate(ws)) / sum(ws)
            assert torch.allclose(out[r], want, rtol=1e-12, atol=1e-13)
        assert (bound > 0).all()


def test_rows_that_see_nothing():
    q, k, v, _ = inputs(2, 10, 64, 9)
    out, bound = head(q, k, v, torch.tensor([-1, -3]))
    assert not out.any() and not bound.any()
