"""The decode step's model over a paged cache: three sequences in ragged chunks, one of them forked from another, in
joint batches, against the oracle's decode step token by token."""
import numpy as np
import pytest

from oracle import oracle as O
from test_decode_step_gpu import CFG_HD128, CFG, build_model, rel_l2, to_device
from test_kv_pages_gpu import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt,cfg,page", [(O.Q8_0, CFG, 5), (O.Q4_K, CFG_HD128, 16)], ids=("64", "128"))
def test_ragged_chunks_match_the_oracles_decode_step(qt, cfg, page):
    import torch as T
    import hesa_cuda as H
    H.clear_device_status()
    c, layers, out_norm, w_out, emb = build_model(qt, seed=11, prefill=0, cfg=cfg)
    g = to_device(c, layers, out_norm, w_out, joined=True)
    n, fork, V = 30, 12, c["vocab"]
    tokens = [[(29 * i + 3) % V for i in range(n)], [(31 * i + 7) % V for i in range(n)]]
    tokens.append(tokens[0][:fork] + [(37 * i + 1) % V for i in range(n - fork)])     # shares the first tokens of sequence 0
    rows = O.dequantize(qt, emb, c["d_model"]).astype(np.float32)
    want = {}
    for s, first in ((0, 0), (2, fork), (1, 0)):      # sequence 2 goes on in the caches that sequence 0 has left
        step = [O.decode_step(c, layers, out_norm, w_out, rows[tokens[s][p]], p).copy() for p in range(first, n)]
        want[s] = np.stack((list(want[0][:first]) if first else []) + step)

    NH, NKV, HD = c["n_head"], c["n_kv_head"], c["head_dim"]
    QD, KD, F = NH * HD, NKV * HD, c["d_ff"]
    # joined weights lie one after another: [wq; wk; wv] and [w_gate; w_up]
    joined = g["keep"]
    cache = H.PagedKV.empty(c["n_layer"], 60, page, NKV, HD, 5, 60 // page + 1)
    emb_d = T.from_numpy(rows).cuda()

    def forward(slots, chunks):
        starts = [0]
        for x in chunks:
            starts.append(starts[-1] + len(x))
        H.kv_reserve(cache, ints(T, slots), ints(T, [len(x) for x in chunks]))
        batch = H.TokenBatch(ints(T, starts), starts[-1], max(map(len, chunks)), n, slots=ints(T, slots))
        x = emb_d[T.tensor(sum(chunks, []), device="cuda")]
        for i, d in enumerate(g["per"]):
            qkv = H.qmatvec(qt, joined[2 * i], H.rms_norm(x, d["attn_norm"]))
            H.rope_kv_paged(cache, i, batch, qkv[:, :QD], qkv[:, QD:QD + KD], qkv[:, QD + KD:], NH, rope_table=g["table"])
            x = H.add(x, H.qmatvec(qt, d["wo"], H.paged_attention(cache, i, batch, qkv[:, :QD], NH)))
            gu = H.qmatvec(qt, joined[2 * i + 1], H.rms_norm(x, d["ffn_norm"]))
            x = H.add(x, H.qmatvec(qt, d["w_down"], H.silu_mul(gu[:, :F].contiguous(), gu[:, F:].contiguous())))
        y = H.qmatvec(qt, g["w_out"], H.rms_norm(x, g["out_norm"])).cpu().numpy()
        return [y[a:b] for a, b in zip(starts, starts[1:])]

    slot, done, got = [3, 1, 0], [0, 0, 0], [[], [], []]

    def advance(news):
        """news: sequence -> tokens that it takes now, in one batch."""
        out = forward([slot[s] for s in news], [tokens[s][done[s]:done[s] + k] for s, k in news.items()])
        for (s, k), y in zip(news.items(), out):
            got[s].append(y)
            done[s] += k
    advance({1: 4, 0: fork})
    H.kv_fork(cache, ints(T, [slot[0]]), ints(T, [slot[2]]))
    done[2] = fork
    got[2].append(got[0][0])
    advance({0: 1, 2: 9, 1: 0})
    advance({2: 1, 1: 20, 0: 3})
    H.kv_compact(cache)
    advance({1: 1, 0: 1, 2: 1})
    advance({0: n - done[0], 2: 2, 1: n - done[1]})
    advance({2: n - done[2]})
    assert done == [n, n, n]
    for s in range(3):
        logits = np.concatenate(got[s])
        worst = max(rel_l2(logits[p], want[s][p]) for p in range(n))
        # fp16 roundings of k and v may fall either way where fp32 sums differ: 2^-11 of single values
        assert worst <= 1e-4, f"sequence {s}: {worst:.2e}"
    assert H.device_status() == 0
