"""How a ragged batch is cut into tiles, and the bindings' handling of streams, without a GPU."""
import os
import random
import subprocess

import pytest

import hesa_build

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
