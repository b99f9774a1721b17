"""CPU tests of the paged cache's and the log probabilities' entry points: sizes
of their workspaces and the refusals that come before any CUDA call."""
import ctypes
import subprocess

import pytest

import hesa_cuda as H

FAKE = 1 << 20   # non-null, aligned, never read: validation fails first


def cache(**kw):
    d = dict(k=FAKE, v=FAKE, page_stride=16 * 2 * 64, layer_stride=10 * 16 * 2 * 64, n_layer=2, n_pages=10, page_size=16,
             n_kv_head=2, head_dim=64, table=FAKE, seq_len=FAKE, page_refs=FAKE, n_slots=4, max_pages=8)
    d.update(kw)
    return H.PagedKVStruct(**d)


def batch(**kw):
    d = dict(slots=None, q_start=FAKE, n_seq=3, n_tokens=7, max_new=4, max_len=100)
    d.update(kw)
    return H.TokenBatchStruct(**d)


def attend(c=None, b=None, layer=0, q=FAKE, ldq=256, out=FAKE, ldo=256, n_head=4, opts=None, ws=FAKE, wsb=1 << 30):
    c, b = c or cache(), b or batch()
    return H.lib().hesa_cuda_paged_attention(ctypes.byref(c), layer, ctypes.byref(b), q, ldq, out, ldo, n_head,
                                             None if opts is None else ctypes.byref(H.AttnOptionsStruct(*opts)), ws, wsb, None)


CACHES = [(dict(k=0), 2), (dict(v=0), 2), (dict(table=0), 2), (dict(seq_len=0), 2), (dict(k=FAKE + 8), 2), (dict(table=FAKE + 2), 2),
          (dict(head_dim=80), 6), (dict(n_pages=0), 6), (dict(page_size=0), 6), (dict(page_size=65537, page_stride=1 << 40), 6),
          (dict(page_size=65536, n_kv_head=1024, page_stride=1 << 40, layer_stride=1 << 45), 6),
          (dict(n_slots=65537), 6), (dict(max_pages=1 << 27), 6), (dict(page_stride=2040), 6), (dict(page_stride=2052), 6),
          (dict(layer_stride=2048), 6), (dict(layer_stride=20484), 6), (dict(n_layer=0), 6), (dict(n_kv_head=-1), 6)]


@pytest.mark.parametrize("kw,code", CACHES)
def test_unsound_caches_are_refused(kw, code):
    c = cache(**kw)
    assert attend(c) == code
    assert H.lib().hesa_cuda_last_error()
    assert H.lib().hesa_cuda_paged_attention_workspace_size(ctypes.byref(c), ctypes.byref(batch()), 4) == 0
    assert H.lib().hesa_cuda_kv_free(ctypes.byref(c), FAKE, 1, FAKE, 1 << 30, None) == code


def test_layers_inside_pages_are_a_sound_layout():
    c = cache(page_stride=2 * 2048, layer_stride=2048)
    assert H.lib().hesa_cuda_paged_attention_workspace_size(ctypes.byref(c), ctypes.byref(batch()), 4) > 0
    assert attend(cache(page_stride=2 * 2048 - 8, layer_stride=2048)) == 6   # two layers' pages overlap


@pytest.mark.parametrize("kw,code", [
    (dict(b=batch(q_start=0)), 2), (dict(b=batch(n_seq=0)), 6), (dict(b=batch(n_seq=5)), 6), (dict(b=batch(n_tokens=-1)), 6),
    (dict(b=batch(max_new=8)), 6), (dict(b=batch(max_len=129)), 6), (dict(b=batch(max_len=-1)), 6),
    (dict(b=batch(n_tokens=1 << 30, max_new=1)), 6), (dict(layer=2), 2), (dict(layer=-1), 2), (dict(n_head=3), 6), (dict(n_head=0), 6),
    (dict(q=0), 2), (dict(out=0), 2), (dict(ws=0), 2), (dict(q=FAKE + 4), 2), (dict(ldq=255), 6), (dict(ldo=258), 2), (dict(ws=FAKE + 8), 2),
    (dict(wsb=100), 2), (dict(opts=(-1.0, 0.0, 0, None, None)), 2), (dict(opts=(0.0, float("nan"), 0, None, None)), 2),
    (dict(opts=(0.0, float("inf"), 0, None, None)), 2), (dict(opts=(0.0, 0.0, -1, None, None)), 2),
    (dict(opts=(0.0, -2.0, 0, None, None)), 2), (dict(opts=(0.0, 1e-9, 0, None, None)), 2)])
def test_attention_refusals(kw, code):
    assert attend(**kw) == code
    assert H.lib().hesa_cuda_last_error()


def test_words_of_the_device_arrays_are_aligned():
    """A list or table of 4-byte words at an odd address is refused by every call that would read it."""
    L, r = H.lib(), ctypes.byref(cache())
    odd = FAKE + 2
    for b in (batch(slots=odd), batch(q_start=odd)):
        assert attend(b=b) == 2 and store(b=b) == 2
    assert attend(opts=(0.0, 0.0, 0, odd, None)) == 2
    assert attend(opts=(0.0, 0.0, 0, None, odd)) == 2
    ws = (FAKE, 1 << 30, None)
    assert L.hesa_cuda_kv_reserve(r, odd, FAKE, 1, *ws) == L.hesa_cuda_kv_reserve(r, FAKE, odd, 1, *ws) == 2
    assert L.hesa_cuda_kv_fork(r, odd, FAKE, 1, *ws) == L.hesa_cuda_kv_fork(r, FAKE, odd, 1, *ws) == 2
    assert L.hesa_cuda_kv_copy_pages(r, odd, FAKE, 1, *ws) == L.hesa_cuda_kv_copy_pages(r, FAKE, odd, 1, *ws) == 2
    assert L.hesa_cuda_kv_free(r, odd, 1, *ws) == L.hesa_cuda_kv_compact(r, odd, *ws) == 2
    for name in ("tokens", "lp", "ent", "ids", "top"):
        assert logprobs(**{name: odd}) == 2


def test_nothing_to_attend_is_no_launch():
    """Nor do tensors without rows, whose pointers are null, make an error."""
    none = batch(n_tokens=0, max_new=0)
    assert attend(b=none) == 0 and attend(b=none, q=0, out=0) == 0
    assert store(b=none, q=0, k=0, v=0) == 0
    assert attend(b=none, layer=2) == 2 and store(b=batch(q_start=0, n_tokens=0, max_new=0)) == 2


def test_attention_workspace_follows_the_cut():
    """Next tokens: the parts of one grid and batch, whatever the lengths. Chunks: parts where the keys are split, few bytes where not."""
    size = lambda **kw: H.lib().hesa_cuda_paged_attention_workspace_size(  # noqa: E731
        ctypes.byref(cache(max_pages=1 << 20)), ctypes.byref(batch(**kw)), 4)
    assert size(n_seq=1, n_tokens=1, max_new=1, max_len=64) == size(n_seq=1, n_tokens=1, max_new=1, max_len=1 << 20) < 16 << 20
    assert size(n_seq=1, n_tokens=64, max_new=64, max_len=256) < size(n_seq=1, n_tokens=64, max_new=64, max_len=1 << 20) < 64 << 20
    assert size(n_seq=3, n_tokens=1 << 16, max_new=1 << 16, max_len=1 << 20) == 16


def store(c=None, b=None, layer=0, q=FAKE, ldq=256, k=FAKE, ldk=128, v=FAKE, ldv=128, n_head=4, table=FAKE, rows=128):
    c, b = c or cache(), b or batch()
    return H.lib().hesa_cuda_rope_kv_paged(ctypes.byref(c), layer, ctypes.byref(b), q, ldq, k, ldk, v, ldv, n_head, table, rows, None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=0), 2), (dict(v=0), 2), (dict(q=0), 2), (dict(ldk=127), 6), (dict(ldv=64), 6), (dict(ldq=252), 6), (dict(rows=0), 6),
    (dict(k=FAKE + 4), 2), (dict(ldv=130), 2), (dict(table=FAKE + 4), 2), (dict(q=FAKE + 8), 2), (dict(layer=5), 2), (dict(n_head=5), 6),
    (dict(b=batch(max_len=200)), 6)])
def test_store_refusals(kw, code):
    assert store(**kw) == code


@pytest.mark.parametrize("kw,code", [(dict(page_refs=0), 2), (dict(page_refs=FAKE + 1), 2), (dict(n_pages=(1 << 20) + 1, layer_stride=1 << 40), 6)])
def test_page_operation_refusals(kw, code):
    L, c = H.lib(), cache(**kw)
    assert L.hesa_cuda_kv_free(ctypes.byref(c), FAKE, 1, FAKE, 1 << 30, None) == code
    assert L.hesa_cuda_kv_compact(ctypes.byref(c), None, FAKE, 1 << 30, None) == code


def test_page_operation_argument_refusals():
    L, c = H.lib(), cache()
    r, big = ctypes.byref(c), 1 << 30
    need = L.hesa_cuda_kv_pages_workspace_size(r)
    assert 0 < need < 4096
    for call in (lambda n, a, w, wb: L.hesa_cuda_kv_reserve(r, a, FAKE, n, w, wb, None), lambda n, a, w, wb: L.hesa_cuda_kv_free(r, a, n, w, wb, None),
                 lambda n, a, w, wb: L.hesa_cuda_kv_fork(r, FAKE, a, n, w, wb, None)):
        assert call(-1, FAKE, FAKE, big) == 6
        assert call(5, FAKE, FAKE, big) == 6      # more than the slots
        assert call(2, 0, FAKE, big) == 2
        assert call(2, FAKE, 0, big) == 2
        assert call(2, FAKE, FAKE + 4, big) == 2
        assert call(2, FAKE, FAKE, need - 1) == 2
    assert L.hesa_cuda_kv_copy_pages(r, FAKE, FAKE, 11, FAKE, big, None) == 6
    assert L.hesa_cuda_kv_copy_pages(r, FAKE, 0, 2, FAKE, big, None) == 2


def logprobs(logits=FAKE, ld=100, n=3, vocab=100, tokens=FAKE, k=5, lp=FAKE, ent=FAKE, ids=FAKE, top=FAKE, ws=FAKE, wsb=1 << 30):
    return H.lib().hesa_cuda_token_logprobs(logits, ld, n, vocab, tokens, k, lp, ent, ids, top, ws, wsb, None)


@pytest.mark.parametrize("kw,code", [
    (dict(logits=0), 2), (dict(logits=FAKE + 2), 2), (dict(ld=99), 6), (dict(n=-1), 6), (dict(vocab=0), 6), (dict(vocab=1 << 30, ld=1 << 30), 6),
    (dict(k=33), 6), (dict(k=-1), 6), (dict(vocab=4, k=5), 6), (dict(tokens=0), 2), (dict(ids=0, top=0), 2), (dict(ws=0), 2),
    (dict(ws=FAKE + 8), 2), (dict(wsb=8), 2)])
def test_logprobs_refusals(kw, code):
    assert logprobs(**kw) == code


def test_no_rows_is_no_launch():
    assert logprobs(n=0) == 0


def test_structs_match_the_header(tmp_path):
    """The ctypes layouts have the sizes that a C compiler gives the header's structs."""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "s.c"
    src.write_text('#include "hesa_cuda.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu\\n", sizeof(hesa_cuda_paged_kv), '
                   'sizeof(hesa_cuda_token_batch), sizeof(hesa_cuda_attn_options)); return 0; }\n')
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    got = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(s) for s in (H.PagedKVStruct, H.TokenBatchStruct, H.AttnOptionsStruct)]
