"""The 4-bit cache's format and its page tables on the host, for the tests: quantization as it is defined, operation by
operation in fp32, a cache laid out with rubbish in every place that no token owns, and its attention in 64 bits."""
import math

import torch

import paged_bounds

GROUP = 32


def quantize(x):
    """(codes uint8 [..., n / 2], scales fp16 [..., n / 32]) of fp32 x [..., n]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    size = g.abs()
    size = torch.where(torch.isfinite(g), size, torch.full_like(size, math.inf))
    first = (size == size.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)
    s = (g.gather(-1, first) / -8.0).double()
    # 8 significant bits, steps of 2^-24 at least; doubles hold every step exactly
    e = torch.floor(torch.log2(s.abs().clamp(min=2.0 ** -149)))
    e = torch.where(2.0 ** e > s.abs(), e - 1, e)
    step = torch.clamp(2.0 ** (e - 7), min=2.0 ** -24)
    d = torch.round(s / step) * step
    d = torch.where(torch.isfinite(size.amax(-1, keepdim=True)) & (d.abs() <= 2720), d, torch.full_like(d, math.nan)).float()
    code = torch.floor(g * (1.0 / d) + 8.5).clamp(0, 15)
    code = torch.where(d.abs() > 0, code, torch.full_like(code, 8.0)).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), d[..., 0].half()


def values(codes, scales):
    """The fp32 values that codes and scales stand for."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    return (n.unflatten(-1, (-1, GROUP)) * scales.float().unsqueeze(-1)).flatten(-2)


def pools(layers, n_pages, page, n_kv, hd, device="cuda", gap=0, inside=False):
    """(k, v, k_scale, v_scale) whose codes are 0xF5 and whose scales are NaN; `gap` groups (a multiple of 8) between
    pages, layers inside pages with `inside`."""
    per = page * n_kv * (hd // GROUP)
    stride = -(-per // 8) * 8 + gap

    def pool(width, dtype, fill):
        shape = (n_pages, layers) if inside else (layers, n_pages)
        flat = torch.full((*shape, stride * width), fill, dtype=dtype, device=device)
        t = flat[:, :, : per * width].unflatten(2, (page, n_kv, hd // GROUP * width))
        return t.transpose(0, 1) if inside else t
    return pool(16, torch.uint8, 0xF5), pool(16, torch.uint8, 0xF5), pool(1, torch.float16, math.nan), pool(1, torch.float16, math.nan)


class Case:
    """Sequences of a cache in 4 bits at random pages; what no token owns is rubbish with NaN scales."""

    def __init__(self, n_head, n_kv, hd, page, lens, news, seed=0, layers=1, slots=None, spare=2, gap=0, inside=False, size=1.3):
        import hesa_cuda as H
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.H, self.n_head, self.n_kv, self.hd, self.page = H, n_head, n_kv, hd, page
        self.lens, self.news, self.n_seq, self.layer = lens, news, len(lens), layers - 1
        self.slot_of = slots or list(range(len(lens)))
        n_slots, width = max(self.slot_of) + 1, max(1, max(-(-n // page) for n in lens))
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + spare
        self.pools = pools(layers, n_pages, page, n_kv, hd, gap=gap, inside=inside)
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        table = torch.full((n_slots, width), -1, dtype=torch.int32)
        seq_len = torch.zeros(n_slots, dtype=torch.int32)
        refs = torch.zeros(n_pages, dtype=torch.int32)
        self.keys, self.values, at = [], [], 0
        for i, n in enumerate(lens):
            pages = order[at:at + need[i]]
            at += need[i]
            table[self.slot_of[i], :need[i]] = torch.tensor(pages, dtype=torch.int32)
            refs[pages] = 1
            seq_len[self.slot_of[i]] = n
            held = []
            for pool, scales in ((self.pools[0], self.pools[2]), (self.pools[1], self.pools[3])):
                codes, sc = quantize(torch.randn(n, n_kv, hd, generator=g, device="cuda"))
                for j, p in enumerate(pages):
                    m = min(page, n - j * page)
                    pool[self.layer, p, :m] = codes[j * page:j * page + m]
                    scales[self.layer, p, :m] = sc[j * page:j * page + m]
                held.append(values(codes, sc))
            self.keys.append(held[0])
            self.values.append(held[1])
        self.table, self.seq_len, self.refs = table.cuda(), seq_len.cuda(), refs.cuda()
        self.cache = H.PagedKV4(*self.pools, self.table, self.seq_len, self.refs)
        self.starts = [0]
        for n in news:
            self.starts.append(self.starts[-1] + n)
        self.n_tokens = self.starts[-1]
        self.q_start = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.slots = torch.tensor(self.slot_of, dtype=torch.int32, device="cuda") if slots else None
        self.q = torch.randn(self.n_tokens, n_head * hd, generator=g, device="cuda") * size
        self.batch = H.TokenBatch(self.q_start, self.n_tokens, max(news), max(lens), slots=self.slots)

    def run(self, **kw):
        return self.H.paged_attention(self.cache, self.layer, self.batch, self.q, self.n_head, **kw)

    def exact(self, **opts):
        """The definition in 64 bits and a bound for each value [n_tokens, n_head, hd]."""
        out = torch.zeros(self.n_tokens, self.n_head, self.hd, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        for i in range(self.n_seq):
            lo, hi, n = self.starts[i], self.starts[i + 1], self.lens[i]
            if hi == lo or n == 0:
                continue
            pos = torch.arange(n - (hi - lo), n, device="cuda")
            o = dict(opts)
            slopes, prefix = o.pop("slopes", None), o.pop("prefix", None)
            for h in range(self.n_head):
                kv = h * self.n_kv // self.n_head
                out[lo:hi, h], bound[lo:hi, h] = paged_bounds.head(
                    self.q[lo:hi].view(hi - lo, self.n_head, self.hd)[:, h], self.keys[i][:, kv], self.values[i][:, kv], pos,
                    slope=0.0 if slopes is None else float(slopes[h]), prefix=0 if prefix is None else int(prefix[i]), **o)
        return out, bound

    def check(self, run=None, **opts):
        ref, bound = self.exact(**opts)
        out = (run or self.run)(**opts)
        assert torch.isfinite(out).all()
        off = (out.view_as(ref).double() - ref).abs()
        assert bool((off <= bound).all()), f"off by {float((off / bound.clamp(min=1e-300)).max()):.2f} of the bound"
        assert float(ref.norm()) == 0 or paged_bounds.relative(out.view_as(ref), ref) <= paged_bounds.RMS
        assert self.H.device_status() == 0
        return out
