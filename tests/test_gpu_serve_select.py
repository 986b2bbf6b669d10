"""Beam selection where many rows share the GPU: a CTA then takes several chunks of a row after one another and carries its
candidates, their bound, maximum and sum from chunk to chunk."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_serve import SKIP, run_select

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::RuntimeWarning")]

ROWS, VOCAB = 256, 40000  # more than half as many rows as CTAs that run at once: one CTA a row, five chunks of 8192


def one_beam(x, scores, n_out):
    """Per row (scores, tokens) of its best, in 64 bits: the higher logit first, then the lower token."""
    out = []
    for r, row in enumerate(x.astype(np.float64)):
        ok = np.nonzero(row > -np.inf)[0]  # NaN: false
        if not len(ok) or np.isposinf(row[ok]).any() or not np.isfinite(scores[r]):
            out.append((np.zeros(0), np.zeros(0, int)))
            continue
        m = row[ok].max()
        lse = m + np.log(np.exp(row[ok] - m).sum())
        best = ok[np.argsort(-row[ok], kind="stable")[:n_out]]
        out.append((float(scores[r]) + (row[best] - lse), best))
    return out


def check(b2, x, n_out, r, pad=0):
    scores = -r.uniform(0, 9, len(x)).astype(np.float32)
    got = run_select(b2, x, scores, len(x), 1, n_out, pad=pad)
    for i, (s, tok) in enumerate(one_beam(x, scores, n_out)):
        n = len(tok)
        assert np.array_equal(got[2][i, :n], tok) and (got[1][i, :n] == 0).all()
        # A thread adds 8 values in each of four chains a chunk, joins them to its sum, which it multiplies by an exponential
        # when its maximum moves (at most 5 times), and 256 threads join theirs: (8 + 3 + 5 + 8) 2^-24 + (1 + 5 + 2) 2^-22
        # < 2^-18 of the sum, so lse within that; then one rounding.
        assert np.all(np.abs(got[0][i, :n] - s) <= 2.0 ** -18 + np.abs(s) * 2.0 ** -24)
        assert (got[0][i, n:] == -np.inf).all() and (got[1][i, n:] == SKIP).all() and (got[2][i, n:] == SKIP).all()


@pytest.mark.parametrize("n_out", [1, 16, 63, 64])
@pytest.mark.parametrize("kind", ["normal", "rising", "falling", "steps", "ties", "equal", "zeros"])
def test_select_over_several_chunks_of_a_row(b2, kind, n_out):
    r = rng(320, n_out)
    token = np.arange(VOCAB)
    x = {"normal": lambda: r.normal(0, 2, (ROWS, VOCAB)),
         "rising": lambda: np.broadcast_to(token * 1e-3, (ROWS, VOCAB)) + r.uniform(0, 1, (ROWS, 1)),   # every logit of a chunk beats the one before
         "falling": lambda: np.broadcast_to(-token * 1e-3, (ROWS, VOCAB)) + r.uniform(0, 1, (ROWS, 1)),
         "steps": lambda: r.normal(0, 1, (ROWS, VOCAB)) + 0.3 * (token // 8192),                          # some hundreds more a chunk
         "ties": lambda: r.integers(0, 12, (ROWS, VOCAB)),
         "equal": lambda: np.ones((ROWS, VOCAB)),
         "zeros": lambda: np.where(r.integers(0, 2, (ROWS, VOCAB)), 0.0, -0.0)}[kind]().astype(np.float32)
    check(b2, x, n_out, r)


@pytest.mark.parametrize("pad", [0, 1])
def test_select_over_several_chunks_with_masks(b2, pad):
    r = rng(321)
    x = r.normal(0, 2, (ROWS, VOCAB)).astype(np.float32)
    x[0:40, :16384 + 5] = -np.inf             # the first chunks hold nothing
    x[40:80, 9:] = -np.inf                    # the later ones nothing
    for i in range(80, 120):                  # a few logits, spread
        keep = r.choice(VOCAB, int(r.integers(0, 40)), replace=False)
        row = np.full(VOCAB, -np.inf, np.float32)
        row[keep] = x[i, keep]
        x[i] = row
    x[120:160][r.random((40, VOCAB)) < 0.5] = np.nan
    x[160:170] = np.nan
    x[170:180, 30000] = np.inf                # a row that is none
    x[180:190, 0], x[180:190, 39999] = np.finfo(np.float32).max, np.finfo(np.float32).min
    x[190:200, 39999], x[190:200, 5] = np.finfo(np.float32).max, np.finfo(np.float32).min
    x[200:210] = np.float32(1e-45) * r.integers(-3, 4, (10, VOCAB))
    check(b2, x, 32, r, pad)


@pytest.mark.parametrize("rows,vocab", [(64, 70001), (150, 20000), (222, 24577), (223, 24577), (500, 16385), (1100, 8193)])
def test_select_with_other_numbers_of_segments(b2, rows, vocab):
    r = rng(322, rows)
    check(b2, r.normal(0, 3, (rows, vocab)).astype(np.float32), 8, r)
