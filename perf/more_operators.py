"""Work of the 4-bit paged KV cache and of beam search over a paged cache, as a server on this library issues it.

A 4-bit cache is a pool of codes and a pool of scales for K and for V, in groups of 32 consecutive dims of a head: codes
[layer, page, place, kv head, head_dim / 2] bytes, of which byte b holds dims 2 b (low nibble) and 2 b + 1 (high), and
fp16 scales [layer, page, place, kv head, head_dim / 32]. A value is scale * (code - 8). Tables and batches are those of
the fp16 cache: the pages of each slot, the tokens that it holds, how many slots refer to each page; and the rows of
sequence i are q_start[i] .. q_start[i + 1] - 1, the last tokens of its slot. Activations are fp32.

  store       rotate-half rope of q (in place) and of the new k at each row's position, and the new k and v into their
              pages: a group's scale is m / -8 for m its value of largest magnitude (the first of them), rounded to 8
              significant bits (a multiple of 2^-24 where it is smaller than 2^-17), a code is floor(x / scale + 8.5) in
              0 .. 15 (8 where the scale is 0). What the pages then hold for the new tokens is read back.
  attention   out = softmax(cap(scale q.k) + bias + mask) v over the pages of the row's sequence: key j is seen from
              position p where j <= p and (no window, or j > p - window), or where j < prefix; cap(s) = c tanh(s / c);
              bias = -slope[head] |p - j|. A row that sees nothing gives zeros.
  select      the next beams of each sequence: of all (beam, token), score[beam] + log softmax(logits[beam])[token], and
              of each beam that has ended itself, with its score and token -1, the `width` largest, ties by the lower
              beam and then the lower token; the beam that each comes from, its token and its score.
  reorder     slot b of a group takes over what slot parents[b] of the group held. Full pages are shared. A partly
              filled last page goes to the first slot that takes it over; the others get copies of its filled places.
              What nobody takes over is given back; then new pages are the lowest free ones in the order of the list.
              Table entries behind a slot's pages that were in use become -1.

`own` is set from outside: False computes the plain forms, True calls the library.
"""
import math
import random

import torch

own = False

F16_BYTES, F32_BYTES = 2, 4
GROUP = 32
VALUE_BYTES = 0.5 + F16_BYTES / GROUP   # of a value in 4 bits, with its share of the scale


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attn(name, n_seq, new, min_len, max_len, heads, kv, hd, page, spread, softcap=0.0, window=0, slopes=False, prefix=0):
    return {"name": name, "op": "attention", "n_seq": n_seq, "new": new, "min_len": min_len, "max_len": max_len, "n_head": heads,
            "n_kv_head": kv, "head_dim": hd, "page": page, "spread": spread, "softcap": softcap, "window": window, "slopes": slopes, "prefix": prefix}


def listed():
    return [
        # one user's next token at the context and head layout of the 7B decode step (32 heads of 128, context 2048)
        _attn("kv4_decode_one", 1, 1, 2048, 2048, 32, 32, 128, 16, 0),
        # the next tokens of a serving batch, sequences of all lengths, the 70B head layout (64 heads on 8 kv heads)
        _attn("kv4_decode_batch", 32, 1, 1, 8192, 64, 8, 128, 16, 1),
        # two very long contexts, what a cache in 4 bits is made for: few rows, a long axis
        _attn("kv4_decode_long", 2, 1, 100001, 131072, 64, 8, 128, 64, 2),
        # a prompt's chunk for the 7B layout: 512 new tokens that see 1536 earlier ones
        _attn("kv4_chunk", 1, 512, 2048, 2048, 32, 32, 128, 16, 0),
        # a mixed batch of ragged chunks, with capped scores, distance bias, window and prefix; odd pages, heads of 64
        _attn("kv4_chunk_mixed", 12, 300, 1, 4001, 16, 4, 64, 24, 3, softcap=30.0, window=1024, slopes=True, prefix=70),
        # a long prompt's chunk: 2048 new tokens at 16384, 64 heads on 8 kv heads
        _attn("kv4_chunk_long", 1, 2048, 16384, 16384, 64, 8, 128, 64, 0),
        # rope and cache write of one decode step's batch
        {"name": "kv4_store_step", "op": "store", "n_seq": 32, "new": 1, "min_len": 1, "max_len": 4096, "n_head": 64, "n_kv_head": 8, "head_dim": 128, "page": 16, "spread": 4},
        # rope and cache write of long prompts' chunks
        {"name": "kv4_store_chunk", "op": "store", "n_seq": 5, "new": 2048, "min_len": 1000, "max_len": 5001, "n_head": 32, "n_kv_head": 32, "head_dim": 128, "page": 16, "spread": 5},
        # one sequence's beams, the 7B vocabulary
        {"name": "beam_select_one", "op": "select", "n_seq": 1, "width": 4, "vocab": 32000, "ended": 0.0, "spread": 6},
        # the beams of a serving batch, a large vocabulary of odd size; some have ended, some sequences have just begun
        {"name": "beam_select_batch", "op": "select", "n_seq": 64, "width": 8, "vocab": 131071, "ended": 0.15, "spread": 7},
        # one sequence's beams change places, in all layers
        {"name": "beam_reorder_one", "op": "reorder", "n_layer": 32, "n_seq": 1, "width": 4, "min_len": 700, "max_len": 700, "n_kv_head": 8, "head_dim": 128, "page": 16, "spread": 8},
        # the beams of a serving batch
        {"name": "beam_reorder_batch", "op": "reorder", "n_layer": 32, "n_seq": 32, "width": 4, "min_len": 50, "max_len": 400, "n_kv_head": 8, "head_dim": 128, "page": 16, "spread": 9},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((32, 32, 128), (64, 8, 128), (32, 8, 128), (16, 4, 64), (8, 2, 64), (4, 4, 256), (12, 2, 128), (8, 1, 128))


def _fits(c):
    """No more than the largest listed case costs, here or in the plain form's memory."""
    w = work(c)
    if c["op"] == "attention":
        lens, news = _lens(c)
        top, wide = max(lens), max(max(news), 1)
        return w["flops"] <= 1.0e12 and c["n_seq"] * top * c["n_kv_head"] * c["head_dim"] <= 3e8 and c["n_seq"] * c["n_head"] * wide * top <= 2.2e9
    if c["op"] == "reorder":
        return c["n_layer"] * _pool_pages(c) * c["page"] * c["n_kv_head"] * c["head_dim"] <= 9e8
    return w["bytes"] <= (2.7e8 if c["op"] == "select" else 6.2e8)


def draw(rng):
    while True:
        op = rng.choice(("attention", "attention", "attention", "store", "select", "select", "reorder"))
        h, kv, hd = rng.choice(_HEADS)
        page, spread = rng.choice((8, 16, 16, 24, 32, 64, 128)), rng.randrange(1, 1 << 20)
        if op == "attention":
            new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
            top = max(new, _log(rng, 1, 131072))
            c = _attn("", _log(rng, 1, 64), new, max(1, _log(rng, 1, top)), top, h, kv, hd, page, spread,
                      softcap=rng.choice((0.0, 0.0, 30.0, 50.0)), window=rng.choice((0, 0, 0, _log(rng, 1, 8192))), slopes=rng.random() < 0.25, prefix=rng.choice((0, 0, 0, _log(rng, 1, 400))))
        elif op == "store":
            new = _log(rng, 1, 2048)
            c = {"op": op, "n_seq": _log(rng, 1, 64), "new": new, "min_len": 1, "max_len": max(new, _log(rng, 1, 8192)), "n_head": h, "n_kv_head": kv, "head_dim": hd, "page": page, "spread": spread}
        elif op == "select":
            c = {"op": op, "n_seq": _log(rng, 1, 128), "width": rng.randrange(1, 17), "vocab": _log(rng, 100, 262144), "ended": rng.choice((0.0, 0.15, 0.5)), "spread": spread}
        else:
            top = _log(rng, 20, 2000)
            c = {"op": op, "n_layer": _log(rng, 1, 48), "n_seq": _log(rng, 1, 48), "width": rng.randrange(2, 13), "min_len": _log(rng, 1, top), "max_len": top, "n_kv_head": kv, "head_dim": hd, "page": page, "spread": spread}
        c.pop("name", None)
        if _fits(c):
            return c


def _lens(case):
    """Tokens and new tokens of each sequence: the first has the most of both, the others lengths spread over the range."""
    r = random.Random(case["spread"])
    lens, news = [case["max_len"]], [case["new"]]
    for _ in range(case["n_seq"] - 1):
        lens.append(_log(r, case["min_len"], case["max_len"]))
        news.append(min(lens[-1], case["new"] if case["new"] == 1 else r.randrange(0, case["new"] + 1)))
    return lens, news


def _prefixes(case, lens):
    return [min(case["prefix"], n) if i % 3 != 1 else 0 for i, n in enumerate(lens)]


def _ended(case):
    """For each beam of each sequence whether it has ended; in every fifth sequence, which has just begun, only the first beam counts and none has."""
    r = random.Random(case["spread"])
    begun = [case["n_seq"] > 1 and i % 5 == 4 for i in range(case["n_seq"])]
    return begun, [[not begun[i] and r.random() < case["ended"] for _ in range(case["width"])] for i in range(case["n_seq"])]


def _beams(case):
    """Tokens of each sequence, the same in all of its beams, the pages that its beams share, and each beam's parent: as in a search, the better beams have more children."""
    r = random.Random(case["spread"])
    lens = [case["max_len"]] + [_log(r, case["min_len"], case["max_len"]) for _ in range(case["n_seq"] - 1)]
    shared = [n * 3 // 4 // case["page"] for n in lens]
    parents = [[min(r.randrange(case["width"]), r.randrange(case["width"])) for _ in range(case["width"])] for _ in lens]
    return lens, shared, parents


def _pool_pages(case):
    lens, shared, _ = _beams(case)
    return sum(s + case["width"] * (-(-n // case["page"]) - s) for n, s in zip(lens, shared)) + case["n_seq"] * case["width"] + 5


def _seen(case):
    """Pairs of a row and a key that it sees, over the batch; and the keys that some row sees."""
    lens, news = _lens(case)
    w = case["window"]
    pairs = keys = 0
    for n, t, pre in zip(lens, news, _prefixes(case, lens)):
        if not t:
            continue
        p0 = n - t
        first = max(0, p0 - w + 1) if w else 0
        keys += (n - first) + min(pre, first)
        for p in range(p0, n):
            lo = max(0, p - w + 1) if w else 0
            pairs += (p + 1 - lo) + min(pre, lo) + max(0, pre - (p + 1))
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "attention":
        pairs, keys = _seen(case)
        rows = sum(_lens(case)[1])
        return {"bytes": keys * case["n_kv_head"] * case["head_dim"] * 2 * VALUE_BYTES + 2 * rows * case["n_head"] * case["head_dim"] * F32_BYTES,
                "flops": 4.0 * pairs * case["n_head"] * case["head_dim"]}
    if op == "store":
        # q in and out, k and v in, their codes and scales out and, read back, in; their values out; a row of the angle table
        rows, hd = sum(_lens(case)[1]), case["head_dim"]
        return {"bytes": rows * hd * (2 * case["n_head"] * F32_BYTES + 2 * case["n_kv_head"] * (2 * F32_BYTES + 2 * VALUE_BYTES) + F32_BYTES),
                "flops": 3.0 * rows * hd * (case["n_head"] + case["n_kv_head"])}
    if op == "select":
        rows = sum((1 if b else case["width"]) - sum(e) for b, e in zip(*_ended(case)))
        return {"bytes": rows * case["vocab"] * F32_BYTES + case["n_seq"] * case["width"] * (2 + 3) * 4, "flops": 3.0 * rows * case["vocab"]}
    lens, shared, parents = _beams(case)
    copied = sum((n % case["page"]) * (len(p) - len(set(p))) for n, p in zip(lens, parents))
    entries = sum(-(-n // case["page"]) * case["width"] for n in lens)
    return {"bytes": 2 * copied * case["n_layer"] * case["n_kv_head"] * case["head_dim"] * 2 * F16_BYTES + 2 * 4 * (2 * entries + case["n_seq"] * case["width"]), "flops": 0}


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _quantize(x):
    """Codes and scales of the groups in the last dimension of x."""
    g = x.unflatten(-1, (-1, GROUP))
    m = g.gather(-1, g.abs().argmax(-1, keepdim=True)) / -8.0
    step = ((m.view(torch.int32) & 0x7F800000).view(torch.float32) * 2.0 ** -7).clamp(min=2.0 ** -24)   # of numbers with 8 significant bits
    d = torch.round(m / step) * step
    code = torch.where(d == 0, torch.full_like(g, 8.0), torch.floor(g * (1.0 / d) + 8.5).clamp(0.0, 15.0)).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), d[..., 0].half()


def _values(codes, scales):
    """What codes and scales stand for, in 32 bits."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    return (n.unflatten(-1, (-1, GROUP)) * scales.float().unsqueeze(-1)).flatten(-2)


def _pool4(case, n_pages, g):
    """Codes and scales of normal values, a part of the pages at a time."""
    kv, hd = case["n_kv_head"], case["head_dim"]
    codes = torch.empty(1, n_pages, case["page"], kv, hd // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(1, n_pages, case["page"], kv, hd // GROUP, dtype=torch.float16, device="cuda")
    some = max(1, (1 << 26) // (case["page"] * kv * hd))
    for p in range(0, n_pages, some):
        x = torch.randn(min(some, n_pages - p), case["page"], kv, hd, generator=g, device="cuda")
        codes[0, p: p + some], scales[0, p: p + some] = _quantize(x)
    return codes, scales


def _tables(lens, page, n_pages, width, g):
    """The table, seq_len and refs of slots whose pages lie at random places of the pool."""
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    need = [-(-x // page) for x in lens]
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < _ints(need)[:, None]] = order[: sum(need)]
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[order[: sum(need)].long()] = 1
    return table, _ints(lens), refs


def _views(buf, n_slots, width):
    a, b = n_slots * width, n_slots * width + n_slots
    return buf[:a].view(n_slots, width), buf[a:b], buf[b:]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    st = {"case": case}

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op in ("attention", "store"):
        lens, news = _lens(case)
        h, kv, hd, page = case["n_head"], case["n_kv_head"], case["head_dim"], case["page"]
        width = -(-max(lens) // page)
        n_pages = sum(-(-x // page) for x in lens) + 3
        st["k"], st["ks"] = _pool4(case, n_pages, g)
        st["v"], st["vs"] = _pool4(case, n_pages, g)
        st["table"], st["seq_len"], st["refs"] = _tables(lens, page, n_pages, width, g)
        starts = [0]
        for t in news:
            starts.append(starts[-1] + t)
        st["q_start"] = _ints(starts)
        st.update(n_tokens=starts[-1], max_new=max(news), max_len=max(lens))
        n = starts[-1]
        if op == "attention":
            st["q"] = rand(n, h * hd) * 1.5
            st["out"] = torch.empty(n, h * hd, device="cuda")
            st["slopes_t"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h) if case["slopes"] else None
            st["prefix_t"] = _ints(_prefixes(case, lens)) if case["prefix"] else None
        else:
            # q, k and v are the columns of one joined projection, as the library's joined matvec gives them
            st["qkv"] = rand(n, (h + 2 * kv) * hd)
            st["q_in"] = st["qkv"][:, : h * hd].clone()
            st["k_new"], st["v_new"] = torch.empty(n, kv * hd, device="cuda"), torch.empty(n, kv * hd, device="cuda")
            inv = 10000.0 ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
            ang = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
            st["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
    elif op == "select":
        n, w, vocab = case["n_seq"], case["width"], case["vocab"]
        begun, ended = _ended(case)
        st["logits"] = rand(n * w, vocab) * 3.0
        # a share of the rows has a part of the vocabulary ruled out, as a grammar does
        ruled = (torch.rand(n * w, 1, generator=g, device="cuda") < 0.25) & (torch.rand(n * w, vocab, generator=g, device="cuda") < 0.3)
        st["logits"].masked_fill_(ruled, -math.inf)
        score = -torch.rand(n, w, generator=g, device="cuda").mul_(4.0).cumsum(1) - 20.0
        first = torch.tensor([0.0] + [-math.inf] * (w - 1), device="cuda")
        st["scores"] = torch.where(torch.tensor(begun, device="cuda")[:, None], first, score).flatten().contiguous()
        st["ended"] = _ints([int(e) for row in ended for e in row])
    else:
        lens, shared, parents = _beams(case)
        w, page, n_pages = case["width"], case["page"], _pool_pages(case)
        n_slots, width = case["n_seq"] * w, -(-max(lens) // page) + 1
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        rows, refs, at = [], [0] * n_pages, 0
        for n, s in zip(lens, shared):
            common, at = order[at: at + s], at + s
            for _ in range(w):
                mine, at = order[at: at + -(-n // page) - s], at + -(-n // page) - s
                rows.append(common + mine + [-1] * (width - s - len(mine)))
                for p in common + mine:
                    refs[p] += 1
        st["width"] = width
        st["tables0"] = _ints([p for row in rows for p in row] + [n for n in lens for _ in range(w)] + refs)
        st["tables"] = st["tables0"].clone()
        st["table"], st["seq_len"], st["refs"] = _views(st["tables"], n_slots, width)
        st["slots"] = torch.arange(n_slots, dtype=torch.int32, device="cuda")
        st["parents"] = _ints([p for row in parents for p in row])
        shape = (case["n_layer"], n_pages, page, case["n_kv_head"], case["head_dim"])
        st["k"], st["v"] = torch.empty(shape, dtype=torch.float16, device="cuda"), torch.empty(shape, dtype=torch.float16, device="cuda")
        for i in range(case["n_layer"]):
            st["k"][i].normal_(generator=g)
            st["v"][i].normal_(generator=g)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _rows_of(st):
    """For each row: its sequence and its position."""
    q_start = st["q_start"].long()
    row = torch.arange(st["n_tokens"], device="cuda")
    seq = torch.searchsorted(q_start, row, right=True) - 1
    new = q_start[1:] - q_start[:-1]
    pos = st["seq_len"].long()[seq] - new[seq] + row - q_start[seq]
    return row, seq, pos


def _attention_plain(st):
    c = st["case"]
    h, kv, hd, top = c["n_head"], c["n_kv_head"], c["head_dim"], st["max_len"]
    n_seq, wide = c["n_seq"], st["max_new"]
    row, seq, pos = _rows_of(st)
    at = row - st["q_start"].long()[seq]
    q = torch.zeros(n_seq, wide, h * hd, device="cuda")
    q[seq, at] = st["q"]
    q = q.view(n_seq, wide, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, (h // kv) * wide, hd)
    pages = st["table"].clamp(min=0).long()
    k = _values(st["k"][0][pages], st["ks"][0][pages]).view(n_seq, -1, kv, hd)[:, :top].permute(0, 2, 1, 3)
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    del k
    s = s.view(n_seq, kv, h // kv, wide, top)
    if c["softcap"]:
        s = torch.tanh(s / c["softcap"]) * c["softcap"]
    p = torch.full((n_seq, wide), -1, device="cuda", dtype=torch.long)
    p[seq, at] = pos
    j = torch.arange(top, device="cuda")
    if c["slopes"]:
        dist = (p[:, :, None] - j[None, None, :]).abs().float()
        s = s - st["slopes_t"].view(1, kv, h // kv, 1, 1) * dist[:, None, None]
    see = j[None, None, :] <= p[:, :, None]
    if c["window"]:
        see = see & (j[None, None, :] > p[:, :, None] - c["window"])
    if c["prefix"]:
        see = see | (j[None, None, :] < st["prefix_t"].long()[:, None, None])
    see = see & (j[None, None, :] < st["seq_len"].long()[:, None, None]) & (p[:, :, None] >= 0)
    s = s.masked_fill(~see[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = s.sum(-1, keepdim=True)
    v = _values(st["v"][0][pages], st["vs"][0][pages]).view(n_seq, -1, kv, hd)[:, :top].permute(0, 2, 1, 3)
    o = torch.matmul(s.view(n_seq, kv, (h // kv) * wide, top), v).view(n_seq, kv, h // kv, wide, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(n_seq, wide, h * hd)
    return o[seq, at]


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _store_plain(st):
    c = st["case"]
    h, kv, hd, page = c["n_head"], c["n_kv_head"], c["head_dim"], c["page"]
    row, seq, pos = _rows_of(st)
    cos, sin = st["rope"][pos, : hd // 2][:, None, :], st["rope"][pos, hd // 2:][:, None, :]
    x = st["qkv"]
    n = x.shape[0]
    q, k, v = x[:, : h * hd], x[:, h * hd: (h + kv) * hd], x[:, (h + kv) * hd:]
    q.copy_(_rotate(q.reshape(n, h, hd), cos, sin).view(n, h * hd))
    at, place = st["table"][seq, pos // page].long(), pos % page
    st["k"][0][at, place], st["ks"][0][at, place] = _quantize(_rotate(k.reshape(n, kv, hd), cos, sin))
    st["v"][0][at, place], st["vs"][0][at, place] = _quantize(v.reshape(n, kv, hd))
    return [q, _values(st["k"][0][at, place], st["ks"][0][at, place]).view(n, kv * hd), _values(st["v"][0][at, place], st["vs"][0][at, place]).view(n, kv * hd)]


def _select_plain(st):
    c = st["case"]
    n, w, vocab = c["n_seq"], c["width"], c["vocab"]
    x = st["logits"].double()   # beams whose scores are near to one another need more than 32 bits
    m = x.amax(1, keepdim=True)
    score = st["scores"].double()[:, None] + (x - m) - torch.log(torch.exp(x - m).sum(1, keepdim=True))
    del x
    # what is ruled out is ranked behind all else, what an ended beam does not have behind that
    score = torch.where(score == -math.inf, torch.full_like(score, -1e300), score)
    ended = (st["ended"] != 0)[:, None]
    score = score.masked_fill_(ended, -math.inf)
    itself = torch.where(ended, st["scores"].double()[:, None], torch.full_like(ended, -math.inf, dtype=torch.float64))
    order = torch.cat([itself, score], 1).view(n, w * (vocab + 1))
    del score
    top, at = torch.sort(order, dim=1, descending=True, stable=True)
    top, at = top[:, :w], at[:, :w]
    top = torch.where(top == -1e300, torch.full_like(top, -math.inf), top)
    return [top.float().flatten(), (at // (vocab + 1)).to(torch.int32).flatten(), (at % (vocab + 1) - 1).to(torch.int32).flatten()]


def _reorder_plain(st):
    c = st["case"]
    table, seq_len, refs, page, w = st["table"], st["seq_len"], st["refs"], c["page"], c["width"]
    slots = st["slots"].long()
    n = slots.numel()
    i = torch.arange(n, device="cuda")
    parent = i // w * w + st["parents"].long()
    rows, lens = table[slots], seq_len[slots]
    j = torch.arange(table.shape[1], device="cuda")
    full, used, tail = lens // page, (lens + page - 1) // page, lens % page
    children = torch.zeros(n, dtype=torch.int32, device="cuda").scatter_add_(0, parent, torch.ones(n, dtype=torch.int32, device="cuda"))
    # references: a page of a slot has one more for each child but the first, a partly filled one at most its own
    more = (children - 1)[:, None].expand_as(rows)
    more = torch.where(j[None, :] < full[:, None], more, torch.where(j[None, :] < used[:, None], more.clamp(max=0), torch.zeros_like(more)))
    refs.scatter_add_(0, torch.where(j[None, :] < used[:, None], rows, torch.zeros_like(rows)).long().view(-1), more.reshape(-1))
    first = torch.full((n,), n, device="cuda").scatter_reduce_(0, parent, i, "amin")
    copy = (tail[parent] > 0) & (first[parent] != i)
    fresh = torch.sort((refs > 0).int(), stable=True).indices[torch.cumsum(copy.int(), 0) - copy.int()].to(torch.int32)
    refs.scatter_add_(0, torch.where(copy, fresh, torch.zeros_like(fresh)).long(), copy.int())
    new = torch.where((j[None, :] == full[parent][:, None]) & copy[:, None], fresh[:, None], rows[parent])
    mine = j[None, :] < used[parent][:, None]
    table[slots] = torch.where(mine, new, torch.where(j[None, :] < used[:, None], torch.full_like(rows, -1), rows))
    seq_len[slots] = lens[parent]
    # a slot with nothing to copy copies its first page onto itself
    old = rows[parent].gather(1, full[parent].clamp(max=table.shape[1] - 1).long()[:, None])[:, 0]
    frm, to = torch.where(copy, old, new[:, 0]).long(), torch.where(copy, fresh, new[:, 0]).long()
    filled = (torch.arange(page, device="cuda")[None, :] < torch.where(copy, tail[parent], torch.zeros_like(tail))[:, None])[None, :, :, None, None]
    for pool in (st["k"], st["v"]):
        pool[:, to] = torch.where(filled, pool[:, frm], pool[:, to])
    return [st["tables"], st["k"], st["v"]]


# ---------------------------------------------------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------------------------------------------------
def _library(st):
    """The library and the handles that a server makes once for its cache, its batch and its buffers."""
    if "library" not in st:
        import os
        import sys
        here = os.path.join(os.getcwd(), "hesa-llm_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import hesa_cuda as H
        c, hold = st["case"], {"H": H}
        if "ks" in st:
            hold["cache"] = H.PagedKV4(st["k"], st["v"], st["ks"], st["vs"], st["table"], st["seq_len"], st["refs"])
            hold["batch"] = H.TokenBatch(st["q_start"], st["n_tokens"], st["max_new"], st["max_len"])
        if c["op"] == "attention":
            hold["workspace"] = H.paged_attention_workspace(hold["cache"], hold["batch"], c["n_head"])
        elif c["op"] == "select":
            hold["workspace"] = H.beam_select_workspace(c["n_seq"], c["width"], c["vocab"])
        elif c["op"] == "reorder":
            hold["cache"] = H.PagedKV(st["k"], st["v"], st["table"], st["seq_len"], st["refs"])
            hold["workspace"] = H.kv_pages_workspace(hold["cache"])
        st["library"] = hold
    hold = st["library"]
    return hold["H"], hold.get("cache"), hold.get("batch"), hold.get("workspace")


def _attention_own(st):
    H, cache, batch, ws = _library(st)
    c = st["case"]
    return H.paged_attention(cache, 0, batch, st["q"], c["n_head"], out=st["out"], softcap=c["softcap"], window=c["window"],
                             slopes=st["slopes_t"], prefix=st["prefix_t"], workspace=ws)


def _store_own(st):
    H, cache, batch, _ = _library(st)
    c, x = st["case"], st["qkv"]
    a, b = c["n_head"] * c["head_dim"], (c["n_head"] + c["n_kv_head"]) * c["head_dim"]
    H.rope_kv_paged(cache, 0, batch, x[:, :a], x[:, a:b], x[:, b:], c["n_head"], rope_table=st["rope"])
    return [x[:, :a], *H.kv_read(cache, 0, batch, k=st["k_new"], v=st["v_new"])]


def _select_own(st):
    H, _, _, ws = _library(st)
    return list(H.beam_select(st["logits"], st["scores"], st["case"]["width"], ended=st["ended"], workspace=ws))


def _reorder_own(st):
    H, cache, _, ws = _library(st)
    H.kv_reorder(cache, st["slots"], st["parents"], st["case"]["width"], workspace=ws)
    return [st["tables"], st["k"], st["v"]]


def run(state):
    op = state["case"]["op"]
    if op == "reorder":
        state["tables"].copy_(state["tables0"])   # every pass starts from the same tables; pages that were copied from stay as they are
    elif op == "store":
        state["qkv"][:, : state["q_in"].shape[1]].copy_(state["q_in"])   # q is rotated in place
    if own:
        return {"attention": _attention_own, "store": _store_own, "select": _select_own, "reorder": _reorder_own}[op](state)
    return {"attention": _attention_plain, "store": _store_plain, "select": _select_plain, "reorder": _reorder_plain}[op](state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "reorder":
        return None   # pages are copied, tables are whole numbers
    st = prepare(case, seed)
    return {"attention": _attention_exact, "store": _store_exact, "select": _select_exact}[op](st)


def _sequence(st, i):
    """Where sequence i's rows lie, its first new position, and of a pool and its scales what they hold for it, in 64 bits [len, kv head, head_dim]."""
    c = st["case"]
    page, kv, hd = c["page"], c["n_kv_head"], c["head_dim"]
    n = int(st["seq_len"][i])
    ids = st["table"][i, : -(-n // page)].long()
    lo, hi = int(st["q_start"][i]), int(st["q_start"][i + 1])

    def held(codes, scales):
        byte = codes[0].index_select(0, ids).reshape(-1, kv, hd // 2)[:n].to(torch.int32)
        x = torch.empty(n, kv, hd, dtype=torch.float64, device="cuda")
        x[:, :, 0::2] = (byte % 16 - 8).double()
        x[:, :, 1::2] = (byte // 16 - 8).double()
        return x * scales[0].index_select(0, ids).reshape(-1, kv, hd // GROUP)[:n].double().repeat_interleave(GROUP, 2)

    return n, lo, hi, n - (hi - lo), held


def _attention_exact(st):
    c = st["case"]
    h, kv, hd = c["n_head"], c["n_kv_head"], c["head_dim"]
    out = torch.zeros(st["n_tokens"], h, hd, dtype=torch.float64, device="cuda")
    for i in range(c["n_seq"]):
        n, lo, hi, p0, held = _sequence(st, i)
        if hi == lo:
            continue
        k, v = held(st["k"], st["ks"]), held(st["v"], st["vs"])
        pos = torch.arange(p0, n, device="cuda", dtype=torch.float64)[:, None]
        key = torch.arange(n, device="cuda", dtype=torch.float64)[None, :]
        hidden = key > pos
        if c["window"]:
            hidden |= key <= pos - c["window"]
        if c["prefix"]:
            hidden &= key >= float(st["prefix_t"][i])
        for head in range(h):
            s = st["q"][lo:hi].view(hi - lo, h, hd)[:, head].double() @ k[:, head * kv // h].T / math.sqrt(hd)
            if c["softcap"]:
                s = c["softcap"] * torch.tanh(s / c["softcap"])
            if c["slopes"]:
                s -= float(st["slopes_t"][head]) * (pos - key).abs()
            out[lo:hi, head] = torch.softmax(s.masked_fill_(hidden, -math.inf), 1) @ v[:, head * kv // h]
    return out.view(st["n_tokens"], h * hd)


def _store_exact(st):
    """q's rotation; what k and v are rounded to is the format's affair, not a value of 64 bits."""
    c = st["case"]
    h, hd = c["n_head"], c["head_dim"]
    x = st["qkv"][:, : h * hd].double().view(st["n_tokens"], h, hd)
    for i in range(c["n_seq"]):
        lo, hi = int(st["q_start"][i]), int(st["q_start"][i + 1])
        pos = torch.arange(int(st["seq_len"][i]) - (hi - lo), int(st["seq_len"][i]), device="cuda")
        t = torch.complex(st["rope"][pos, : hd // 2].double(), st["rope"][pos, hd // 2:].double())[:, None, :]
        z = torch.complex(x[lo:hi, :, : hd // 2], x[lo:hi, :, hd // 2:]) * t
        x[lo:hi] = torch.cat([z.real, z.imag], 2)
    return [x.reshape(st["n_tokens"], h * hd), None, None]


def _select_exact(st):
    c = st["case"]
    n, w = c["n_seq"], c["width"]
    best = torch.full((n, w), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(w):   # the best so far and one more beam's
        x = st["logits"][b::w].double()
        score = st["scores"][b::w].double()[:, None]
        lp = score + torch.log_softmax(x, 1)
        ended = (st["ended"][b::w] != 0)[:, None]
        mine = torch.where(ended, torch.full_like(lp, -math.inf), lp).topk(min(w, x.shape[1]), 1).values
        best = torch.cat([best, mine, torch.where(ended, score, torch.full_like(score, -math.inf))], 1).topk(w, 1).values
    return [best.flatten(), None, None]
