"""CPU tests of the 4-bit cache's and the beam search's entry points: sizes of workspaces, struct layouts and the
refusals that come before any CUDA call; and what the format promises, on the host."""
import ctypes
import subprocess

import pytest
import torch

import hesa_cuda as H
import kv4_model

FAKE = 1 << 20   # non-null, aligned, never read: validation fails first
BIG = 1 << 40


def cache(**kw):
    # pages of 16 places, 2 heads of 64 dims: 64 groups
    d = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, page_stride=64, layer_stride=640, n_layer=2, n_pages=10, page_size=16, n_kv_head=2,
             head_dim=64, table=FAKE, seq_len=FAKE, page_refs=FAKE, n_slots=4, max_pages=8)
    d.update(kw)
    return H.PagedKV4Struct(**d)


def fp16_cache(**kw):
    d = dict(k=FAKE, v=FAKE, page_stride=2048, layer_stride=20480, n_layer=2, n_pages=10, page_size=16, n_kv_head=2, head_dim=64, table=FAKE,
             seq_len=FAKE, page_refs=FAKE, n_slots=4, max_pages=8)
    d.update(kw)
    return H.PagedKVStruct(**d)


def batch(**kw):
    d = dict(slots=None, q_start=FAKE, n_seq=3, n_tokens=7, max_new=4, max_len=100)
    d.update(kw)
    return H.TokenBatchStruct(**d)


def attend(c=None, b=None, layer=0, q=FAKE, ldq=256, out=FAKE, ldo=256, n_head=4, opts=None, ws=FAKE, wsb=1 << 30):
    c, b = c or cache(), b or batch()
    return H.lib().hesa_cuda_paged_attention_kv4(ctypes.byref(c), layer, ctypes.byref(b), q, ldq, out, ldo, n_head,
                                                 None if opts is None else ctypes.byref(H.AttnOptionsStruct(*opts)), ws, wsb, None)


def write(c=None, b=None, layer=0, q=FAKE, ldq=256, k=FAKE, ldk=128, v=FAKE, ldv=128, n_head=4, table=FAKE, rows=100):
    c, b = c or cache(), b or batch()
    return H.lib().hesa_cuda_rope_kv4_paged(ctypes.byref(c), layer, ctypes.byref(b), q, ldq, k, ldk, v, ldv, n_head, table, rows, None)


def read(c=None, b=None, layer=0, k=FAKE, ldk=128, v=FAKE, ldv=128):
    c, b = c or cache(), b or batch()
    return H.lib().hesa_cuda_kv4_read(ctypes.byref(c), layer, ctypes.byref(b), k, ldk, v, ldv, None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=0), 2), (dict(v=0), 2), (dict(k_scale=0), 2), (dict(v_scale=0), 2), (dict(table=0), 2), (dict(seq_len=0), 2), (dict(k=FAKE + 8), 2),
    (dict(v=FAKE + 4), 2), (dict(k_scale=FAKE + 8), 2), (dict(v_scale=FAKE + 2), 2), (dict(table=FAKE + 2), 2), (dict(head_dim=96), 6), (dict(head_dim=32), 6),
    (dict(n_pages=0), 6), (dict(page_size=0), 6), (dict(page_size=65537, page_stride=BIG), 6),
    (dict(page_size=65536, n_kv_head=1024, page_stride=BIG, layer_stride=1 << 45), 6), (dict(n_slots=65537), 6), (dict(max_pages=1 << 27), 6),
    (dict(page_stride=56), 6), (dict(page_stride=68), 6), (dict(page_stride=-64), 6), (dict(layer_stride=64), 6), (dict(layer_stride=636), 6),
    (dict(n_layer=0), 6), (dict(n_kv_head=-1), 6), (dict(page_size=-1), 6), (dict(page_stride=1 << 51), 6), (dict(head_dim=-2 ** 31, page_size=-2 ** 31), 6)])
def test_unsound_caches_are_refused(kw, code):
    c = cache(**kw)
    for rc in (attend(c), write(c), read(c)):
        assert rc == code and H.lib().hesa_cuda_last_error()
    assert H.lib().hesa_cuda_paged_attention_kv4_workspace_size(ctypes.byref(c), ctypes.byref(batch()), 4) == 0
    assert H.lib().hesa_cuda_kv4_pages_workspace_size(ctypes.byref(c)) == 0
    r = ctypes.byref(c)
    for call in (lambda: H.lib().hesa_cuda_kv4_free(r, FAKE, 1, FAKE, BIG, None), lambda: H.lib().hesa_cuda_kv4_reserve(r, FAKE, FAKE, 1, FAKE, BIG, None),
                 lambda: H.lib().hesa_cuda_kv4_fork(r, FAKE, FAKE, 1, FAKE, BIG, None), lambda: H.lib().hesa_cuda_kv4_compact(r, None, FAKE, BIG, None),
                 lambda: H.lib().hesa_cuda_kv4_copy_pages(r, FAKE, FAKE, 1, FAKE, BIG, None),
                 lambda: H.lib().hesa_cuda_kv4_reorder(r, FAKE, FAKE, 2, 2, FAKE, BIG, None)):
        assert call() == code


def test_layers_inside_pages_are_a_sound_layout():
    c = cache(page_stride=128, layer_stride=64)
    assert H.lib().hesa_cuda_paged_attention_kv4_workspace_size(ctypes.byref(c), ctypes.byref(batch()), 4) > 0
    assert attend(cache(page_stride=120, layer_stride=64)) == 6   # two layers' pages overlap


@pytest.mark.parametrize("kw,code", [
    (dict(b=batch(q_start=0)), 2), (dict(b=batch(n_seq=0)), 6), (dict(b=batch(n_seq=5)), 6), (dict(b=batch(n_tokens=-1)), 6),
    (dict(b=batch(max_new=8)), 6), (dict(b=batch(max_len=129)), 6), (dict(b=batch(max_len=-1)), 6), (dict(b=batch(q_start=FAKE + 1)), 2),
    (dict(b=batch(slots=FAKE + 2)), 2), (dict(b=batch(n_tokens=1 << 30, max_new=1)), 6), (dict(layer=2), 2), (dict(layer=-1), 2), (dict(n_head=3), 6),
    (dict(n_head=0), 6), (dict(q=0), 2), (dict(out=0), 2), (dict(ws=0), 2), (dict(q=FAKE + 4), 2), (dict(ldq=255), 6), (dict(ldo=258), 2),
    (dict(ws=FAKE + 8), 2), (dict(wsb=100), 2), (dict(opts=(-1.0, 0.0, 0, None, None)), 2), (dict(opts=(0.0, float("nan"), 0, None, None)), 2),
    (dict(opts=(0.0, 0.0, -1, None, None)), 2), (dict(opts=(0.0, 1e7, 0, None, None)), 2), (dict(opts=(3e38, 0.0, 0, None, None)), 2),
    (dict(opts=(0.0, 0.0, 0, FAKE + 2, None)), 2), (dict(opts=(0.0, 0.0, 0, None, FAKE + 1)), 2)])
def test_attention_refuses(kw, code):
    assert attend(**kw) == code and H.lib().hesa_cuda_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(layer=2), 2), (dict(n_head=5), 6), (dict(k=0), 2), (dict(v=0), 2), (dict(q=0), 2), (dict(ldq=255), 6), (dict(ldk=127), 6), (dict(ldv=120), 6),
    (dict(ldk=130), 2), (dict(ldv=129), 2), (dict(k=FAKE + 4), 2), (dict(table=FAKE + 8), 2), (dict(rows=0), 6), (dict(ldk=1 << 41), 6),
    (dict(b=batch(max_new=8)), 6)])
def test_write_refuses(kw, code):
    assert write(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(layer=-1), 2), (dict(ldk=127), 6), (dict(ldv=0), 6), (dict(ldk=130), 2), (dict(v=FAKE + 8), 2), (dict(ldv=1 << 41), 6), (dict(b=batch(n_seq=9)), 6)])
def test_read_refuses(kw, code):
    assert read(**kw) == code


def test_calls_with_nothing_to_do():
    b = batch(n_tokens=0, max_new=0)
    assert attend(b=b, q=0, out=0, ws=0) == 0 and write(b=b, q=0, k=0, v=0) == 0 and read(b=b, k=0, v=0) == 0
    assert read(k=0, v=0) == 0
    assert attend(b=batch(max_new=0)) == 0
    for lib, c in ((H.lib().hesa_cuda_kv4_reorder, cache()), (H.lib().hesa_cuda_kv_reorder, fp16_cache())):
        assert lib(ctypes.byref(c), None, None, 0, 4, FAKE, BIG, None) == 0
    assert H.lib().hesa_cuda_beam_select(None, 10, 0, 4, 10, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("fn,c", [("hesa_cuda_kv_reorder", fp16_cache()), ("hesa_cuda_kv4_reorder", cache())])
def test_reorder_refuses(fn, c):
    call, r = getattr(H.lib(), fn), ctypes.byref(c)
    for args, code in (((FAKE, FAKE, 2, 0, FAKE, BIG), 6), ((FAKE, FAKE, 2, 33, FAKE, BIG), 6), ((FAKE, FAKE, 3, 2, FAKE, BIG), 6),
                       ((FAKE, FAKE, 5, 5, FAKE, BIG), 6), ((FAKE, FAKE, -2, 2, FAKE, BIG), 6), ((None, FAKE, 2, 2, FAKE, BIG), 2),
                       ((FAKE, None, 2, 2, FAKE, BIG), 2), ((FAKE + 2, FAKE, 2, 2, FAKE, BIG), 2), ((FAKE, FAKE + 1, 2, 2, FAKE, BIG), 2),
                       ((FAKE, FAKE, 2, 2, None, BIG), 2), ((FAKE, FAKE, 2, 2, FAKE + 4, BIG), 2), ((FAKE, FAKE, 2, 2, FAKE, 16), 2)):
        assert call(r, *args, None) == code and H.lib().hesa_cuda_last_error()
    refs = type(c)(**{n: getattr(c, n) for n, _ in c._fields_})
    refs.page_refs = None
    assert call(ctypes.byref(refs), FAKE, FAKE, 2, 2, FAKE, BIG, None) == 2


def test_beam_select_refuses():
    def call(x=FAKE, ld=100, n=2, w=4, vocab=100, scores=FAKE, ended=None, out=FAKE, par=FAKE, tok=FAKE, ws=FAKE, wsb=BIG):
        return H.lib().hesa_cuda_beam_select(x, ld, n, w, vocab, scores, ended, out, par, tok, ws, wsb, None)
    for kw, code in ((dict(w=0), 6), (dict(w=33), 6), (dict(vocab=0), 6), (dict(ld=99), 6), (dict(n=-1), 6), (dict(vocab=1 << 30, ld=1 << 30), 6),
                     (dict(ld=1 << 41), 6), (dict(n=1 << 26), 6), (dict(x=None), 2), (dict(scores=None), 2), (dict(out=None), 2), (dict(par=None), 2),
                     (dict(tok=None), 2), (dict(ws=None), 2), (dict(x=FAKE + 2), 2), (dict(scores=FAKE + 1), 2), (dict(ended=FAKE + 2), 2),
                     (dict(out=FAKE + 2), 2), (dict(ws=FAKE + 8), 2), (dict(wsb=64), 2)):
        assert call(**kw) == code and H.lib().hesa_cuda_last_error(), kw
    size = H.lib().hesa_cuda_beam_select_workspace_size
    assert size(0, 4, 100) == 0 and size(1, 0, 100) == 0 and size(1, 33, 100) == 0 and size(1, 4, 0) == 0
    assert size(1, 4, 32000) >= 4 * (8 + 4 * 8) and 1 <= size(64, 8, 131071) / (512 * (8 + 8 * 8)) <= 64


def test_workspaces_grow_with_the_batch_and_are_bounded():
    size = H.lib().hesa_cuda_paged_attention_kv4_workspace_size
    c = cache(n_slots=64, max_pages=4096, page_size=16, n_pages=100, layer_stride=6400)
    last = 1
    for n in (1, 4, 16, 64):
        b = batch(n_seq=n, n_tokens=n, max_new=1, max_len=60000)
        nb = size(ctypes.byref(c), ctypes.byref(b), 4)
        assert nb >= last
        last = nb
    # chunks: the fp16 copies of as many sequences as fit into 1 GB, one at least
    one = 469 * 128 * 2 * 64 * 4
    for n, held in ((1, 1), (8, 8), (64, (1 << 30) // one)):
        b = batch(n_seq=n, n_tokens=n * 50, max_new=50, max_len=60000)
        nb = size(ctypes.byref(c), ctypes.byref(b), 4)
        assert held * one <= nb < held * one + (256 << 20)
    wide = cache(n_kv_head=64, head_dim=256, page_stride=16 * 64 * 8, layer_stride=160 * 64 * 8, n_slots=2, max_pages=1 << 16, page_size=16)
    b = batch(n_seq=2, n_tokens=200, max_new=100, max_len=1 << 20)
    assert size(ctypes.byref(wide), ctypes.byref(b), 64) >= (1 << 20) * 64 * 256 * 4


def test_struct_layout(tmp_path):
    """The ctypes struct has the layout that the C header gives it."""
    src = tmp_path / "t.c"
    names = [n for n, _ in H.PagedKV4Struct._fields_]
    src.write_text('#include <stdio.h>\n#include "hesa_cuda.h"\nint main(void) { printf("%zu", sizeof(hesa_cuda_paged_kv4));\n'
                   + "".join(f'printf(" %zu", offsetof(hesa_cuda_paged_kv4, {n}));\n' for n in names) + "return 0; }\n")
    import os
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(H.PagedKV4Struct)] + [getattr(H.PagedKV4Struct, n).offset for n in names]


def test_values_are_fp16_numbers():
    g = torch.Generator().manual_seed(0)
    for scale in (1.0, 1e-3, 1e-6, 2.0 ** -21, 3000.0, 5000.0):
        codes, d = kv4_model.quantize(torch.randn(200, 64, generator=g) * scale)
        v = kv4_model.values(codes, d)
        assert bool(((v.half().float() == v) | torch.isnan(v)).all())
        # 24 scales are one too, so that (16 + code) d - 24 d rounds nothing
        m = 24 * d.float()
        assert bool(((m.half().float() == m) | torch.isnan(m)).all())


def test_python_refusals():
    with pytest.raises((ValueError, RuntimeError, AssertionError)):
        H.beam_select(torch.zeros(4, 10), torch.zeros(4), 2)   # not on a GPU


def test_workspaces_hold_every_pass_of_a_chunk():
    """The fp16 copies of as many sequences as fit into 1 GB go at a time, as a cache of pages of 128 tokens; the last pass may
    have fewer, and what the attention over each of them asks for is there."""
    import random
    r = random.Random(5)
    L = H.lib()
    several = more = 0
    for i in range(3000):
        n_kv, hd = r.choice((1, 2, 4, 8, 16, 32, 64)), r.choice((64, 128, 256))
        g = r.choice((1, 2, 4, 8))
        n_seq = r.randrange(1, r.choice((3, 10, 60)))
        max_len = int(2 ** r.uniform(7, 19))
        max_new = min(max_len, r.randrange(1, r.choice((100, 3000))))
        tokens = min(max_new * n_seq, (1 << 31) // (2 * n_kv * g))
        if max_new * g <= 64 or max_new > tokens:
            continue
        c = cache(n_kv_head=n_kv, head_dim=hd, page_stride=16 * n_kv * hd // 32, layer_stride=0, n_layer=1, n_slots=64, max_pages=1 << 15)
        b = batch(n_seq=n_seq, n_tokens=r.randrange(max_new, tokens + 1), max_new=max_new, max_len=max_len)
        size = L.hesa_cuda_paged_attention_kv4_workspace_size(ctypes.byref(c), ctypes.byref(b), n_kv * g)
        pages = -(-max_len // 128)
        token = 4 * n_kv * hd
        at_a_time = max(1, min(n_seq, (1 << 30) // (pages * 128 * token)))
        needs = []
        for n in [at_a_time] * (n_seq // at_a_time) + [n_seq % at_a_time]:
            if n == 0:
                continue
            inner = fp16_cache(n_kv_head=n_kv, head_dim=hd, page_size=128, page_stride=128 * n_kv * hd, layer_stride=0, n_layer=1,
                               n_slots=at_a_time, max_pages=pages, n_pages=at_a_time * pages)
            part = batch(n_seq=n, n_tokens=b.n_tokens, max_new=max_new, max_len=max_len)
            needs.append(L.hesa_cuda_paged_attention_workspace_size(ctypes.byref(inner), ctypes.byref(part), n_kv * g))
            assert needs[-1] > 0
        assert size >= at_a_time * pages * 128 * token + max(needs), (n_kv, hd, g, n_seq, max_len, max_new)
        several += len(needs) > 1
        more += needs[-1] > needs[0]
    assert several > 200 and more > 50


@pytest.mark.parametrize("head_dim", [48, 80, 100, 144, 1])
def test_an_empty_cache_has_whole_groups(head_dim):
    with pytest.raises(ValueError, match="multiple of 32"):
        H.PagedKV4.empty(1, 4, 16, 2, head_dim, 2, 2)
