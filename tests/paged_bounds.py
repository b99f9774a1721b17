"""The attention of one head in 64 bits with a bound for every value of its result, and the relative error of a whole
result; for fp32 inputs on any device.

What the kernels round, relative to the sizes in play (half a step of fp32 is 2^-24; a tensor core's running sum is
taken to be cut, 2^-23):

  score    q is held in 21 bits (2^-21 of each |q_i k_i|), and hd / 16 sums of 16 products, the sum of the two halves and
           the scale round numbers no larger than A = scale sum |q_i k_i|: (hd / 16 + 8) 2^-23 A in all
  cap      2^-21 of the capped score, and no more of what came before (the slope of tanh is at most 1)
  bias     its factor and the product: 2^-22 of it
  p        2^-23 (|s| + |s - m|) for the scores in base 2, 2^-19 for the shift by 14 (below 10 2^-24), the exponential
           (2^-22) and the two halves of P (2^-21)
  sums     of p v and p: a rounding for every 16 keys and a few where parts are joined, (n / 16 + 16) 2^-23

And a step of 2^-24 is the last that a half of P has, 2^-38 of the row's largest p, which the shift puts at 2^14: each p
is off by that much beside its relative error (a weight of 10^-20 is none).

A relative error e_j of p_j moves the result by at most sum_j w_j e_j (|v_j| + |out|), w the weights.

Most of these are independent and of either sign, so a whole result is nearer. For scores of standard deviation 2 or
less the roundings of p have an rms of at most sqrt((hd / 16 + 3) (2^-23 2)^2 + (2^-21 2 / sqrt 3)^2 + (20 2^-24)^2 +
(2^-22)^2 + (2^-21)^2), 1.8e-6 with head_dim 256; values v of either sign average as the weights' errors do, and the
sum of p adds as much again: 2.5e-6 of the result's norm. RMS is 2^-18, 3.8e-6. A high half of P or of q alone would
leave errors of 2^-12 in it.
"""
import math

import torch

RMS = 2.0 ** -18


def high_half(x, away):
    """x to 11 bits, away from zero or cut."""
    m, e = torch.frexp(x)
    y = torch.ldexp(m, torch.full_like(e, 11))
    return torch.ldexp((torch.sign(y) * y.abs().ceil() if away else torch.trunc(y)), e - 11)


def halves(x, away):
    """x as the sum of two halves of 11 bits."""
    hi = high_half(x, away)
    low = x - hi
    m, e = torch.frexp(low)
    return hi + torch.ldexp(torch.round(torch.ldexp(m, torch.full_like(e, 11))), e - 11)


def head(q, k, v, pos, scale=None, softcap=0.0, window=0, slope=0.0, prefix=0, q_as=None, p_as=None):
    """(out, bound), [rows, hd] each, of rows q [rows, hd] at positions pos over keys k and values v [n, hd]. q_as and
    p_as stand in for how a kernel would hold q and p (the bound is then of no meaning)."""
    n, hd = k.shape
    scale = scale or 1.0 / math.sqrt(hd)
    q, k, v = q.double(), k.double(), v.double()
    s = (q_as(q) if q_as else q) @ k.T * scale
    e = (hd / 16 + 8) * 2.0 ** -23 * (q.abs() @ k.abs().T) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        e = e + 2.0 ** -21 * s.abs()
    j = torch.arange(n, device=k.device)[None, :]
    p0 = pos[:, None]
    b = slope * (p0 - j).abs().double()
    s, e = s - b, e + 2.0 ** -22 * b
    see = j <= p0
    if window:
        see = see & (j > p0 - window)
    if prefix:
        see = see | (j < prefix)
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(1, keepdim=True)
    d = (s - torch.where(m == -math.inf, torch.zeros_like(m), m)).masked_fill(~see, -math.inf)
    p = torch.exp(d)
    z = p.sum(1, keepdim=True)
    w = torch.where(z > 0, (p_as(p) if p_as else p) / z, torch.zeros_like(p))
    out = w @ v
    e = torch.where(see, e + 2.0 ** -23 * (s.abs() + d.abs()) + 2.0 ** -19, torch.zeros_like(e))
    we = torch.where(see, w * e + 2.0 ** -38 / z, torch.zeros_like(e))
    bound = we @ v.abs() + we.sum(1, keepdim=True) * out.abs() + (n / 16 + 16) * 2.0 ** -23 * (w @ v.abs() + out.abs())
    return out, bound


def relative(out, ref):
    """The error of a whole result, as a share of its norm."""
    return float((out.double() - ref).norm() / ref.norm())
