"""How a ragged batch is cut into tiles, and the bindings' handling of streams, without a GPU."""
import ctypes
import os
import random
import subprocess

import pytest

import hesa_build
import hesa_cuda as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OUT_DIR = os.path.join(ROOT, "tests", "cpp", "_build")


@pytest.fixture(scope="module")
def tiles_of():
    """The kernels' own function that finds a tile's rows, compiled for the host."""
    src, exe = os.path.join(ROOT, "tests", "cpp", "tiles.cu"), os.path.join(OUT_DIR, "tiles")
    deps = [src] + [os.path.join(hesa_build.CSRC, f) for f in ("paged.h", "hesa_common.cuh")]
    if not os.path.exists(exe) or any(os.path.getmtime(d) > os.path.getmtime(exe) for d in deps):
        os.makedirs(OUT_DIR, exist_ok=True)
        res = subprocess.run([hesa_build.NVCC, *hesa_build.ARCH_FLAGS, "-std=c++17", "--expt-relaxed-constexpr", "-cudart", "static", src,
                              "-o", exe], capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-4000:]

    def call(g, r, starts, n_tokens):
        out = subprocess.run([exe, *map(str, (g, r, len(starts) - 1, n_tokens, *starts))], capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return call


@pytest.mark.parametrize("seed", range(40))
def test_every_row_has_one_tile(tiles_of, seed):
    """Whatever row the first sequence starts at: each sequence's rows in tiles, once, and no tile before its first row."""
    rng = random.Random(seed)
    g, r = rng.choice([1, 2, 3, 8, 64]), rng.choice([8, 128])
    starts = [rng.choice([0, 1, 7, 100, 5000])]
    for _ in range(rng.choice([1, 2, 9])):
        starts.append(starts[-1] + rng.choice([0, 1, 1, 3, 40, 200]))
    got = tiles_of(g, r, starts, starts[-1] + rng.choice([0, 5]))
    want = {(s, at) for s in range(len(starts) - 1) for at in range(0, (starts[s + 1] - starts[s]) * g, r)}
    # a tile behind a sequence's rows holds none; one before them would be read and written where it has no business
    assert all(at >= -1 for _, at in got)
    live = [(s, at) for s, at in got if 0 <= at < (starts[s + 1] - starts[s]) * g]
    assert len(live) == len(set(live)) and set(live) == want


def test_starts_that_are_not_sound_stay_in_range(tiles_of):
    for starts in ([-4, 3, 9], [9, 3, 20], [2 ** 31 - 1, 5, 7], [-2 ** 31, -2 ** 31, 2 ** 31 - 1], [0, -4, 9]):
        got = tiles_of(8, 8, starts, 40)
        assert all(0 <= s < len(starts) - 1 and -1 <= at <= 8 * len(got) for s, at in got)


class Streams:
    """torch's streams as the binding uses them: which one is current, which ones capture."""

    def __init__(self, monkeypatch):
        import contextlib

        import torch
        self.now, self.capturing = 100, set()

        @contextlib.contextmanager
        def on(stream):
            was, self.now = self.now, stream.cuda_stream
            yield
            self.now = was
        monkeypatch.setattr(torch.cuda, "stream", on)
        monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
        monkeypatch.setattr(torch.cuda, "default_stream", lambda: Stream(0))
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.now in self.capturing)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: self.now)
        monkeypatch.setattr(H, "_same_device", lambda cache, batch=None: None)
        monkeypatch.setattr(H, "kv_pages_workspace", lambda cache: Scratch(self.now))


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


class Scratch:
    """A buffer that torch's allocator took from the memory of the stream that was current."""

    def __init__(self, home):
        self.home = home

    def record_stream(self, stream):
        pass


class Cache:
    def __init__(self):
        self.scratch, self.workspace, self.device = {}, None, 0


def test_scratch_of_page_operations_comes_from_the_calls_own_stream(monkeypatch):
    """Whatever was current when the cache first needed some, and wherever the next call runs: memory of one stream is
    never handed to kernels of another, and no captured graph shares it with eager calls or with another graph."""
    s, c = Streams(monkeypatch), Cache()
    for stream in (Stream(7), 7, None, Stream(8), 0, None):
        want = s.now if stream is None else stream if isinstance(stream, int) else stream.cuda_stream
        assert H._page_workspace(c, None, stream).home == want
    s.now = 200
    eager = H._page_workspace(c, None, None)
    assert eager.home == 200 and H._page_workspace(c, None, None) is eager
    s.capturing.add(200)
    captured = [H._page_workspace(c, None, None) for _ in range(2)]
    assert captured[0] is not captured[1] and eager not in captured and all(x.home == 200 for x in captured)
    s.capturing.clear()
    assert H._page_workspace(c, None, None) is eager


@pytest.mark.parametrize("n_seq,n_kv,hd", [(1024, 32, 128), (1024, 8, 64), (200, 16, 64), (300, 17, 256), (1, 8, 128)])
def test_lengths_of_no_token_are_cut_like_lengths_of_one(n_seq, n_kv, hd):
    """A batch whose bound says that nobody has a key yet: a block a tile, as where everybody has one. (Cut into groups of
    two heads whatever the number of tiles, the list of what is joined would be longer than its place.)"""
    size = {}
    for max_len in (0, 1, 16):
        kv = H.PagedKVStruct(k=1 << 20, v=1 << 20, page_stride=16 * n_kv * hd, layer_stride=0, n_layer=1, n_pages=4, page_size=16, n_kv_head=n_kv,
                             head_dim=hd, table=1 << 20, seq_len=1 << 20, page_refs=None, n_slots=n_seq, max_pages=4)
        b = H.TokenBatchStruct(slots=None, q_start=1 << 20, n_seq=n_seq, n_tokens=n_seq, max_new=1, max_len=max_len)
        size[max_len] = H.lib().hesa_cuda_paged_attention_workspace_size(ctypes.byref(kv), ctypes.byref(b), n_kv)
    assert 0 < size[0] == size[1] == size[16]


@pytest.mark.parametrize("scale,softcap,code", [(3e38, 0.0, 2), (1e33, 1e-6, 2), (float("inf"), 0.0, 2), (float("nan"), 0.0, 2), (-1.0, 0.0, 2)])
def test_scales_that_no_float_holds_are_refused(scale, softcap, code):
    kv = H.PagedKVStruct(k=1 << 20, v=1 << 20, page_stride=16 * 64, layer_stride=0, n_layer=1, n_pages=4, page_size=16, n_kv_head=1,
                         head_dim=64, table=1 << 20, seq_len=1 << 20, page_refs=None, n_slots=1, max_pages=4)
    b = H.TokenBatchStruct(slots=None, q_start=1 << 20, n_seq=1, n_tokens=1, max_new=1, max_len=20)
    o = H.AttnOptionsStruct(scale, softcap, 0, None, None)
    assert H.lib().hesa_cuda_paged_attention(ctypes.byref(kv), 0, ctypes.byref(b), 1 << 20, 64, 1 << 20, 64, 1, ctypes.byref(o), 1 << 20,
                                             1 << 30, None) == code
    assert H.lib().hesa_cuda_last_error()


def test_pools_with_dimensions_of_one_entry(monkeypatch):
    """Such a dimension's stride says nothing: heads before places, one layer of many, one page, are sound pools."""
    import torch
    monkeypatch.setattr(H, "_want", lambda *a, **k: None)
    table, seq_len = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    def strides(k, v=None):
        s = H.PagedKV(k, k.clone(memory_format=torch.contiguous_format) if v is None else v, table, seq_len).struct
        return s.layer_stride, s.page_stride
    half = dict(dtype=torch.float16)
    assert strides(torch.zeros(2, 5, 16, 4, 64, **half)) == (5 * 16 * 256, 16 * 256)
    assert strides(torch.zeros(2, 5, 1, 16, 64, **half).transpose(2, 3)) == (5 * 16 * 64, 16 * 64)     # one head, heads outside
    assert strides(torch.zeros(2, 5, 4, 1, 64, **half).transpose(2, 3)) == (5 * 256, 256)             # pages of one token
    one = torch.zeros(5, 3, 16, 4, 64, **half).transpose(0, 1)
    assert strides(one[1:2], one[2:3]) == (5 * 3 * 16 * 256, 3 * 16 * 256)                             # one layer of three
    page = torch.zeros(7, 9, 16, 4, 64, **half).permute(1, 0, 2, 3, 4)
    assert strides(page[:, 2:3], page[:, 4:5]) == (16 * 256, 16 * 256)                                 # one page, nine layers
    for k, v in ((torch.zeros(2, 5, 4, 16, 64, **half).transpose(2, 3), None), (one, torch.zeros(3, 5, 16, 4, 64, **half)),
                 (torch.zeros(2, 5, 16, 4, 128, **half)[..., :64], None), (one, one[:, :4])):
        with pytest.raises(ValueError):
            strides(k, v if v is not None else k)
