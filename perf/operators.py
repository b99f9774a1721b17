"""Work of the paged KV cache operators and of the token log probabilities, as a server on this library issues it.

A cache is a pool of fp16 pages [layer, page, slot, kv head, head_dim] (one pool for K, one for V) and three int32
tables: the pages of each sequence slot [n_slots, max_pages], the tokens that each slot holds, and how many slots
refer to each page (0: the page is free). A batch is n_seq sequences with new tokens each: the rows of q (and of the
new k and v) of sequence i are q_start[i] .. q_start[i + 1] - 1, and its new tokens are the last ones of its slot, so
row q_start[i] + t has position seq_len - new + t. Activations are fp32, as everywhere in the library.

  attention   out = softmax(cap(scale q.k) + bias + mask) v over the pages of the row's sequence: key j is seen from
              position p where j <= p and (no window, or j > p - window), or where j < prefix; cap(s) = c tanh(s / c);
              bias = -slope[head] |p - j|. A row that sees nothing gives zeros.
  store       rotate-half rope of q (in place) and of the new k at each row's position, and the new k and v rounded to
              fp16 into their pages.
  pages       free drops the references of a slot's pages. fork lets a new slot share the full pages of another and
              copies the filled slots of the last, partly filled one into a page of its own. reserve gives a slot the
              pages for n more tokens. New pages are the lowest free ones in the order of the list. compact moves pages
              so that the pages in use are 0 .. n - 1: free pages below n, ascending, take the pages from n on, ascending.
  logprobs    log softmax of each row's token, the entropy of the row, and the k largest log probabilities with their
              ids, ties to the lower id.

`own` is set from outside: False computes the plain forms, True calls the library.
"""
import math
import random

import torch

own = False

F16_BYTES, F32_BYTES = 2, 4


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attn(name, n_seq, new, min_len, max_len, heads, kv, hd, page, spread, softcap=0.0, window=0, slopes=False, prefix=0):
    return {"name": name, "op": "attention", "n_seq": n_seq, "new": new, "min_len": min_len, "max_len": max_len, "n_head": heads,
            "n_kv_head": kv, "head_dim": hd, "page": page, "spread": spread, "softcap": softcap, "window": window, "slopes": slopes, "prefix": prefix}


def listed():
    return [
        # one user's next token at the context and head layout of the 7B decode step (32 heads of 128, context 2048)
        _attn("decode_one_7b", 1, 1, 2048, 2048, 32, 32, 128, 16, 0),
        # the next tokens of a serving batch, sequences of all lengths, the 70B head layout (64 heads on 8 kv heads)
        _attn("decode_batch_gqa", 32, 1, 1, 8192, 64, 8, 128, 16, 1),
        # two very long contexts with their next token: few rows, a long axis
        _attn("decode_long_gqa", 2, 1, 100001, 131072, 64, 8, 128, 64, 2),
        # a prompt's chunk for the 7B layout: 512 new tokens that see 1536 earlier ones
        _attn("chunk_7b", 1, 512, 2048, 2048, 32, 32, 128, 16, 0),
        # a mixed batch of ragged chunks, with capped scores, distance bias, window and prefix; odd pages, heads of 64
        _attn("chunk_mixed_bias", 12, 300, 1, 4001, 16, 4, 64, 24, 3, softcap=30.0, window=1024, slopes=True, prefix=70),
        # a long prompt's chunk: 2048 new tokens at 16384, 64 heads on 8 kv heads
        _attn("chunk_long_gqa", 1, 2048, 16384, 16384, 64, 8, 128, 64, 0),
        # rope and cache write of one decode step's batch
        {"name": "store_step", "op": "store", "n_seq": 32, "new": 1, "min_len": 1, "max_len": 4096, "n_head": 64, "n_kv_head": 8, "head_dim": 128, "page": 16, "spread": 4},
        # rope and cache write of long prompts' chunks
        {"name": "store_chunk", "op": "store", "n_seq": 5, "new": 2048, "min_len": 1000, "max_len": 5001, "n_head": 32, "n_kv_head": 32, "head_dim": 128, "page": 16, "spread": 5},
        # one step of a beam search: the beams that lose are freed, the winners forked, each gets room for a token
        {"name": "pages_beam", "op": "beam", "n_layer": 32, "n_pages": 640, "n_slots": 16, "n_fork": 7, "n_free": 7, "max_len": 700, "n_kv_head": 8, "head_dim": 128, "page": 16, "spread": 6},
        # a pool after many sequences came and went, made dense again
        {"name": "pages_compact", "op": "compact", "n_layer": 32, "n_pages": 1024, "n_slots": 24, "n_free": 12, "max_len": 1250, "n_kv_head": 8, "head_dim": 128, "page": 16, "spread": 7},
        # the sampled token's log probability and the alternatives, one sequence, the 7B vocabulary
        {"name": "logprobs_one", "op": "logprobs", "n_rows": 1, "vocab": 32000, "top_k": 8, "spread": 8},
        # a prompt scored: every token's log probability, a large vocabulary of odd size
        {"name": "logprobs_prompt", "op": "logprobs", "n_rows": 1024, "vocab": 131071, "top_k": 5, "spread": 9},
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
    if c["op"] in ("beam", "compact"):
        return c["n_layer"] * c["n_pages"] * c["page"] * c["n_kv_head"] * c["head_dim"] <= 5.4e8
    return w["bytes"] <= (6.0e8 if c["op"] == "logprobs" else 6.2e8)


def draw(rng):
    while True:
        op = rng.choice(("attention", "attention", "attention", "store", "beam", "compact", "logprobs"))
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
        elif op == "logprobs":
            c = {"op": op, "n_rows": _log(rng, 1, 4096), "vocab": _log(rng, 50, 262144), "top_k": rng.randrange(1, 33), "spread": spread}
        else:
            slots = rng.randrange(4, 64)
            n_free = rng.randrange(1, slots // 2 + 1)
            c = {"op": op, "n_layer": _log(rng, 1, 48), "n_pages": 0, "n_slots": slots, "n_free": n_free, "max_len": _log(rng, 20, 2500), "n_kv_head": kv, "head_dim": hd, "page": page, "spread": spread}
            if op == "beam":
                c["n_fork"] = rng.randrange(1, n_free + 1)
            c["n_pages"] = (slots + 4) * (-(-c["max_len"] // page) + 2)
        c.pop("name", None)
        if c.get("top_k", 0) <= c.get("vocab", 1 << 30) and _fits(c):
            return c


def _lens(case):
    """Tokens and new tokens of each sequence: the first has the most of both, the others lengths spread over the range."""
    r = random.Random(case["spread"])
    lens, news = [case["max_len"]], [case["new"]]
    for _ in range(case["n_seq"] - 1):
        lens.append(_log(r, case["min_len"], case["max_len"]))
        news.append(min(lens[-1], case["new"] if case["new"] == 1 else r.randrange(0, case["new"] + 1)))
    return lens, news


def _slots(case):
    """Tokens of each slot of a cache in use, and the slots that are freed."""
    r = random.Random(case["spread"])
    lens = [_log(r, max(1, case["max_len"] // 8), case["max_len"]) for _ in range(case["n_slots"])]
    lens[0] = case["max_len"]
    return lens, sorted(r.sample(range(1, case["n_slots"]), case["n_free"])), r


def _prefixes(case, lens):
    return [min(case["prefix"], n) if i % 3 != 1 else 0 for i, n in enumerate(lens)]


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
        return {"bytes": keys * case["n_kv_head"] * case["head_dim"] * 2 * F16_BYTES + 2 * rows * case["n_head"] * case["head_dim"] * F32_BYTES,
                "flops": 4.0 * pairs * case["n_head"] * case["head_dim"]}
    if op == "store":
        rows, hd = sum(_lens(case)[1]), case["head_dim"]
        return {"bytes": rows * hd * (2 * case["n_head"] * F32_BYTES + 2 * case["n_kv_head"] * (F32_BYTES + F16_BYTES) + F32_BYTES),
                "flops": 3.0 * rows * hd * (case["n_head"] + case["n_kv_head"])}
    row = case.get("n_kv_head", 0) * case.get("head_dim", 0) * 2 * F16_BYTES
    if op == "beam":
        lens, freed, r = _slots(case)
        parents = _parents(case, freed, r)
        copied = sum(lens[p] % case["page"] for p in parents)
        tables = (case["n_slots"] * (-(-case["max_len"] // case["page"]) + 2) + case["n_slots"] + case["n_pages"]) * 4
        return {"bytes": 2 * copied * row * case["n_layer"] + 2 * tables, "flops": 0}
    if op == "compact":
        tables = (case["n_slots"] * (-(-case["max_len"] // case["page"]) + 2) + case["n_slots"] + case["n_pages"]) * 4
        live = _live(case)
        # pages lie at random: a share (1 - live / n) of the places below live is free, and as many pages move
        return {"bytes": int(2 * live * (1 - live / case["n_pages"])) * case["page"] * row * case["n_layer"] + 2 * tables, "flops": 0}
    return {"bytes": case["n_rows"] * (case["vocab"] * F32_BYTES + 3 * 4 + case["top_k"] * 8), "flops": 4.0 * case["n_rows"] * case["vocab"]}


def _live(case):
    lens, freed, _ = _slots(case)
    return sum(-(-n // case["page"]) for i, n in enumerate(lens) if i not in freed)


def _parents(case, freed, r):
    kept = [i for i in range(case["n_slots"]) if i not in freed]
    return [r.choice(kept) for _ in range(case["n_fork"])]


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(case, n_layer, n_pages, g):
    shape = (n_layer, n_pages, case["page"], case["n_kv_head"], case["head_dim"])
    k = torch.empty(shape, dtype=torch.float16, device="cuda")
    v = torch.empty(shape, dtype=torch.float16, device="cuda")
    for i in range(n_layer):
        k[i].normal_(generator=g)
        v[i].normal_(generator=g)
    return k, v


def _tables(lens, page, n_pages, width, g):
    """One int32 buffer [table | seq_len | refs]: each slot's pages lie at random places of the pool."""
    n = len(lens)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    need = [-(-x // page) for x in lens]
    buf = torch.zeros(n * width + n + n_pages, dtype=torch.int32, device="cuda")
    table, seq_len, refs = _views(buf, n, width)
    table.fill_(-1)
    have = torch.arange(width, device="cuda")[None, :] < _ints(need)[:, None]
    table[have] = order[: sum(need)]
    seq_len.copy_(_ints(lens))
    refs[order[: sum(need)].long()] = 1
    return buf


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
        st["k"], st["v"] = _pool(case, 1, n_pages, g)
        st["tables"] = _tables(lens, page, n_pages, width, g)
        st["table"], st["seq_len"], st["refs"] = _views(st["tables"], len(lens), width)
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
            top = max(lens)
            inv = 10000.0 ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
            ang = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
            st["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
    elif op in ("beam", "compact"):
        lens, freed, r = _slots(case)
        page = case["page"]
        width = -(-case["max_len"] // page) + 2
        st["k"], st["v"] = _pool(case, case["n_layer"], case["n_pages"], g)
        st["width"] = width
        st["tables0"] = _tables(lens, page, case["n_pages"], width, g)
        st["tables"] = st["tables0"].clone()
        st["table"], st["seq_len"], st["refs"] = _views(st["tables"], len(lens), width)
        st["freed"] = _ints(freed)
        if op == "beam":
            st["parents"] = _ints(_parents(case, freed, r))
            st["children"] = _ints(freed[: case["n_fork"]])
            st["one"] = torch.ones(case["n_fork"], dtype=torch.int32, device="cuda")
        else:
            # the sequences that ended have been freed already
            _free_plain(st["table"], st["seq_len"], st["refs"], st["freed"], page)
            st["tables0"].copy_(st["tables"])
            st["n_live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        n, vocab = case["n_rows"], case["vocab"]
        st["logits"] = rand(n, vocab) * 3.0
        # a share of the rows has a part of the vocabulary ruled out, as a grammar does
        ruled = (torch.rand(n, 1, generator=g, device="cuda") < 0.25) & (torch.rand(n, vocab, generator=g, device="cuda") < 0.3)
        st["logits"].masked_fill_(ruled, -math.inf)
        st["tokens"] = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
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
    h, kv, hd, page, top = c["n_head"], c["n_kv_head"], c["head_dim"], c["page"], st["max_len"]
    n_seq, wide = c["n_seq"], st["max_new"]
    row, seq, pos = _rows_of(st)
    at = row - st["q_start"].long()[seq]
    q = torch.zeros(n_seq, wide, h * hd, device="cuda")
    q[seq, at] = st["q"]
    q = q.view(n_seq, wide, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, (h // kv) * wide, hd)
    pages = st["table"].clamp(min=0).long()
    k = st["k"][0][pages].reshape(n_seq, -1, kv, hd)[:, :top].permute(0, 2, 1, 3).float()
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
    v = st["v"][0][pages].reshape(n_seq, -1, kv, hd)[:, :top].permute(0, 2, 1, 3).float()
    v = v.masked_fill((j[None, :] >= st["seq_len"].long()[:, None])[:, None, :, None], 0.0)
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
    at = st["table"][seq, pos // page].long()
    st["k"][0][at, pos % page] = _rotate(k.reshape(n, kv, hd), cos, sin).half()
    st["v"][0][at, pos % page] = v.reshape(n, kv, hd).half()
    return [q, st["k"], st["v"]]


def _free_plain(table, seq_len, refs, slots, page):
    s = slots.long()
    j = torch.arange(table.shape[1], device="cuda")
    used = j[None, :] < ((seq_len[s] + page - 1) // page)[:, None]
    rows = table[s]
    refs.scatter_add_(0, torch.where(used, rows, 0).long().view(-1), -used.int().view(-1))
    table[s] = torch.where(used, -1, rows)
    seq_len[s] = 0


def _lowest_free(refs):
    return torch.sort((refs > 0).int(), stable=True).indices


def _fork_plain(st, src, dst):
    table, seq_len, refs, page = st["table"], st["seq_len"], st["refs"], st["case"]["page"]
    a, b = src.long(), dst.long()
    n = seq_len[a]
    rows, j = table[a], torch.arange(table.shape[1], device="cuda")
    full, tail = n // page, n % page
    order = _lowest_free(refs)
    shared = j[None, :] < full[:, None]
    refs.scatter_add_(0, torch.where(shared, rows, 0).long().view(-1), shared.int().view(-1))
    split = tail > 0
    fresh = order[torch.cumsum(split.int(), 0) - split.int()].int()
    old = rows.gather(1, full.clamp(max=table.shape[1] - 1).long()[:, None])[:, 0]
    last = (j[None, :] == full[:, None]) & split[:, None]
    table[b] = torch.where(shared, rows, torch.where(last, fresh[:, None], table[b]))
    refs.scatter_add_(0, torch.where(split, fresh, 0).long(), split.int())
    seq_len[b] = n
    # a fork with nothing to copy copies its first page onto itself
    frm = torch.where(split, old, rows[:, 0]).long()
    to = torch.where(split, fresh, rows[:, 0]).long()
    filled = (torch.arange(page, device="cuda")[None, :] < torch.where(split, tail, 0)[:, None])[None, :, :, None, None]
    for pool in (st["k"], st["v"]):
        pool[:, to] = torch.where(filled, pool[:, frm], pool[:, to])


def _reserve_plain(st, slots, count):
    table, seq_len, refs, page = st["table"], st["seq_len"], st["refs"], st["case"]["page"]
    s = slots.long()
    have = (seq_len[s] + page - 1) // page
    want = (seq_len[s] + count + page - 1) // page
    need = want - have
    start = torch.cumsum(need, 0) - need
    j = torch.arange(table.shape[1], device="cuda")
    new = (j[None, :] >= have[:, None]) & (j[None, :] < want[:, None])
    nth = (start[:, None] + j[None, :] - have[:, None]).clamp(0, refs.numel() - 1)
    pages = _lowest_free(refs)[nth.long()].int()
    table[s] = torch.where(new, pages, table[s])
    refs.scatter_add_(0, torch.where(new, pages, 0).long().view(-1), new.int().view(-1))
    seq_len[s] = seq_len[s] + count


def _beam_plain(st):
    _free_plain(st["table"], st["seq_len"], st["refs"], st["freed"], st["case"]["page"])
    _fork_plain(st, st["parents"], st["children"])
    _reserve_plain(st, st["children"], st["one"])
    return [st["tables"], st["k"], st["v"]]


def _compact_plain(st):
    table, refs, page = st["table"], st["refs"], st["case"]["page"]
    used = refs > 0
    live = used.sum()
    i = torch.arange(refs.numel(), device="cuda")
    to = (~used & (i < live)).nonzero()[:, 0]
    frm = (used & (i >= live)).nonzero()[:, 0]
    new_of = i.to(torch.int32)
    new_of[frm] = to.to(torch.int32)
    have = torch.arange(table.shape[1], device="cuda")[None, :] < ((st["seq_len"] + page - 1) // page)[:, None]
    table.copy_(torch.where(have, new_of[table.clamp(min=0).long()], table))
    for pool in (st["k"], st["v"]):
        pool[:, to] = pool[:, frm]
    refs[to] = refs[frm]
    refs[frm] = 0
    st["n_live"].copy_(live.to(torch.int32).view(1))
    return [st["tables"], st["n_live"], st["k"], st["v"]]


def _logprobs_plain(st):
    x, k = st["logits"], st["case"]["top_k"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    token = x.gather(1, st["tokens"].long()[:, None]) - lse
    # the entropy is lse - sum p x; what is ruled out adds nothing
    entropy = torch.log(z) - (e * torch.where(e > 0, x - m, torch.zeros_like(x))).sum(1, keepdim=True) / z
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    return [token[:, 0], entropy[:, 0], ids[:, :k].to(torch.int32), top[:, :k] - lse]


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
        if "table" in st:
            hold["cache"] = H.PagedKV(st["k"], st["v"], st["table"], st["seq_len"], st["refs"])
        if "q_start" in st:
            hold["batch"] = H.TokenBatch(st["q_start"], st["n_tokens"], st["max_new"], st["max_len"])
        if c["op"] == "attention":
            hold["workspace"] = H.paged_attention_workspace(hold["cache"], hold["batch"], c["n_head"])
        elif c["op"] in ("beam", "compact"):
            hold["workspace"] = H.kv_pages_workspace(hold["cache"])
        elif c["op"] == "logprobs":
            hold["workspace"] = H.token_logprobs_workspace(c["n_rows"], c["vocab"], c["top_k"])
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
    return [x[:, :a], st["k"], st["v"]]


def _beam_own(st):
    H, cache, _, ws = _library(st)
    H.kv_free(cache, st["freed"])
    H.kv_fork(cache, st["parents"], st["children"], workspace=ws)
    H.kv_reserve(cache, st["children"], st["one"])
    return [st["tables"], st["k"], st["v"]]


def _compact_own(st):
    H, cache, _, ws = _library(st)
    H.kv_compact(cache, n_live=st["n_live"], workspace=ws)
    return [st["tables"], st["n_live"], st["k"], st["v"]]


def _logprobs_own(st):
    H, _, _, ws = _library(st)
    return list(H.token_logprobs(st["logits"], st["tokens"], top_k=st["case"]["top_k"], workspace=ws))


def run(state):
    op = state["case"]["op"]
    if op in ("beam", "compact"):
        state["tables"].copy_(state["tables0"])   # every pass starts from the same tables; pages that were copied from stay as they are
    elif op == "store":
        state["qkv"][:, : state["q_in"].shape[1]].copy_(state["q_in"])   # q is rotated in place
    if own:
        return {"attention": _attention_own, "store": _store_own, "beam": _beam_own, "compact": _compact_own, "logprobs": _logprobs_own}[op](state)
    return {"attention": _attention_plain, "store": _store_plain, "beam": _beam_plain, "compact": _compact_plain, "logprobs": _logprobs_plain}[op](state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "attention":
        return _attention_exact(st)
    if op == "store":
        return _store_exact(st)
    if op == "logprobs":
        x = st["logits"].double()
        lp = torch.log_softmax(x, 1)
        some = lp.masked_fill(lp == -math.inf, 0.0)
        order = torch.argsort(-x, dim=1, stable=True)[:, : case["top_k"]]
        return [lp.gather(1, st["tokens"].long()[:, None])[:, 0], -(lp.exp() * some).sum(1), order.to(torch.int32), lp.gather(1, order)]
    return None   # pages are copied, tables are whole numbers


def _sequence(st, i):
    """K and V of sequence i in 64 bits [len, kv head, head_dim], where its rows lie, and its new tokens' first position."""
    page = st["case"]["page"]
    n = int(st["seq_len"][i])
    ids = st["table"][i, : -(-n // page)].long()
    lo, hi = int(st["q_start"][i]), int(st["q_start"][i + 1])
    flat = lambda pool: torch.cat(list(pool[0][ids]), 0)[:n].double()  # noqa: E731
    return n, lo, hi, n - (hi - lo), flat


def _attention_exact(st):
    c = st["case"]
    h, kv, hd = c["n_head"], c["n_kv_head"], c["head_dim"]
    out = torch.zeros(st["n_tokens"], h, hd, dtype=torch.float64, device="cuda")
    for i in range(c["n_seq"]):
        n, lo, hi, p0, flat = _sequence(st, i)
        if hi == lo:
            continue
        k, v = flat(st["k"]), flat(st["v"])
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
    c = st["case"]
    h, kv, hd, page = c["n_head"], c["n_kv_head"], c["head_dim"], c["page"]
    x = st["qkv"].double().view(st["n_tokens"], h + 2 * kv, hd)
    k, v = st["k"].double(), st["v"].double()
    for i in range(c["n_seq"]):
        _, lo, hi, p0, _ = _sequence(st, i)
        pos = torch.arange(p0, p0 + hi - lo, device="cuda")
        t = torch.complex(st["rope"][pos, : hd // 2].double(), st["rope"][pos, hd // 2:].double())[:, None, :]
        z = torch.complex(x[lo:hi, : h + kv, : hd // 2], x[lo:hi, : h + kv, hd // 2:]) * t
        x[lo:hi, : h + kv] = torch.cat([z.real, z.imag], 2)
        ids = st["table"][i][pos // page].long()
        k[0, ids, pos % page] = x[lo:hi, h: h + kv]
        v[0, ids, pos % page] = x[lo:hi, h + kv:]
    return [x[:, :h].reshape(st["n_tokens"], h * hd), k, v]
