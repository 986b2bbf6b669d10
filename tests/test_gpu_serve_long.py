"""Prompts over caches of many steps of 64 keys, whose outputs move from tensor memory to FP32 sums on the way: rows of y on 32, 16
and 4 bytes, maxima that rise and fall along the keys, windows, rows that see their first key late or never, pages that are
none. Tolerances: those of test_gpu_serve_blocks.check."""
import numpy as np
import pytest

import serve_ref as ref
from conftest import rng
from test_gpu_serve import u32
from test_gpu_serve_blocks import Blocks, check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LENGTHS = [(64, 900), (40, 513), (70, 260), (1, 700)]


@pytest.mark.parametrize("y_pad", [0, 4, 3])
@pytest.mark.parametrize("dim", [32, 96, 128, 160, 224, 256])
def test_rows_of_y_on_any_alignment(b2, dim, y_pad):
    b = Blocks(b2, rng(500, dim), LENGTHS, 2, 20, dim, 32)
    assert b.rows * b.n_head >= 6144
    check(b, b.run(pad=2, y_pad=y_pad))


@pytest.mark.parametrize("shape", ["rising", "falling", "peak", "steps"])
@pytest.mark.parametrize("dim", [96, 256])
def test_maxima_that_move_along_the_keys(b2, dim, shape):
    # scores of some 60 (powers of e) from end to end
    r = rng(501, dim)
    u = r.choice([-1.0, 1.0], dim)

    def keys(n):
        x = np.arange(n) / max(n - 1, 1)
        h = {"rising": x, "falling": 1 - x, "peak": 1 - np.abs(2 * x - 1), "steps": np.floor(6 * x) / 6}[shape]
        return (0.3 * r.normal(0, 1, (n, 2, dim)) + 2.5 * h[:, None, None] * u).reshape(n, -1).astype(np.float32)

    b = Blocks(b2, r, LENGTHS, 2, 20, dim, 16, k=keys)
    b.q = (0.2 * b.q + 24.0 / dim ** 0.5 * u).astype(np.float32)
    check(b, b.run())


@pytest.mark.parametrize("window", [65, 300, 640])
@pytest.mark.parametrize("dim", [64, 160])
def test_windows_over_many_steps(b2, dim, window):
    # a tile's first rows see no key of its last steps, its last rows none of the first ones
    b = Blocks(b2, rng(502, dim), [(200, 1100), (64, 513), (1, 700)], 2, 16, dim, 64)
    check(b, b.run(window, y_pad=4), window)


def test_pages_that_are_none_over_many_steps(b2):
    b = Blocks(b2, rng(503), LENGTHS, 2, 20, 160, 16)
    whole = b.run()
    t = b.table.copy()
    gone = [0, 1, 2, 3, 4, 5, 17, 30, 31, 50]  # steps without a key at the start, tiles here and there
    t[0, gone] = ref.NO_SLOT
    got = b.run(table=t)
    assert u32(b.status)[0] == b2.SERVE_PAGE and np.array_equal(got[64:], whole[64:])
    for row, h in ((0, 0), (63, 39), (31, 20)):
        key = np.array([x for x in range(900 - 64 + row + 1) if x // 16 not in gone])
        k, v = (b.p.ref.values(i, b.table[0][key // 16], key % 16)[:, h // 20] for i in (0, 1))
        s = k @ b.q[row, h].astype(np.float64) * b.scale
        p = np.exp(s - s.max())
        p /= p.sum()
        big = np.abs(k * b.q[row, h]).sum(-1).max() * b.scale
        tol = 2.0 ** -17 * (1 + big / 8) * (p @ np.abs(v)) + 900 * 2.0 ** -30 * np.abs(v).max()
        assert (np.abs(got[row, h] - p @ v) <= tol).all()
    t[0, :] = ref.NO_SLOT
    assert (b.run(table=t)[:64] == 0).all()


@pytest.mark.parametrize("dim", [96, 256])
def test_not_a_number_late_in_a_long_cache(b2, dim):
    # V of one token infinite: the rows that see it, its block; K of one token NaN: all dims of the rows that see it
    b = Blocks(b2, rng(504, dim), [(64, 900), (40, 513), (70, 260)], 2, 20, dim, 16)
    at = 880
    slot = b.table[0][at // 16] * 16 + at % 16
    keep = b.p.ref.bytes.copy()
    one = np.ones((1, 2 * dim), np.float32)
    v = one.copy()
    v[0, 70] = np.inf
    b.p.fill([slot], one, v)
    got = b.run()
    first = at - (900 - 64)
    assert np.isnan(got[first:64, :20, 64:96]).all()
    got[first:64, :20, 64:96] = 0
    assert np.isfinite(got).all()
    b.p.ref.bytes[:] = keep
    k = one.copy()
    k[0, dim + 5] = np.nan
    b.p.fill([slot], k, one)
    got = b.run()
    assert np.isnan(got[first:64, 20:]).all()
    got[first:64, 20:] = 0
    assert np.isfinite(got).all()


def test_a_long_prompt_gives_the_same_bits_each_time(b2):
    b = Blocks(b2, rng(505), LENGTHS, 2, 20, 224, 16)
    want = b.run()
    for _ in range(3):
        assert np.array_equal(b.run(stream=torch.cuda.Stream().cuda_stream), want)
