"""Attention over the 4-bit cache where the 32-dim blocks of a token have scales far from one another, for single tokens and drafts
(units of up to sixteen rows) and for prompts (the tensor-memory kernel): a block's dims are as good as if the others were
not there, whatever lies in them. And sums over many keys, which tensor memory alone would make too small."""
import math

import numpy as np
import pytest

import serve_ref as ref
from conftest import load_package, rng
from test_gpu_serve import Batch, Paged, u32

load_package()
import fpga_llama_gguf_b200.kv4 as kv4  # noqa: E402

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FEW = [(1, 1), (1, 40), (3, 130), (1, 333), (2, 64)]
PROMPTS = [(150, 190), (1, 300), (60, 333), (97, 97)]


def unlike(r, n, n_kv, dim, large, small, kind):
    """Rows [n, n_kv dim] of normal values whose blocks have magnitudes of 2^large and 2^small. kind "blocks": by block, the same
    in every token; "turns": by token and block in turns; "late": small up to the middle, then by block."""
    block, tok = np.arange(dim // 32), np.arange(n)[:, None]
    big = {"blocks": (block % 2 == 0) & (tok >= 0), "turns": (block + tok) % 2 == 0, "late": (block % 2 == 0) & (tok >= n // 2)}[kind]
    x = r.normal(0, 1, (n, n_kv, dim // 32, 32)) * np.where(big, 2.0 ** large, 2.0 ** small)[:, None, :, None]
    return x.reshape(n, -1).astype(np.float32)


class Blocks(Batch):
    """A Batch whose K and V are rows(tokens) of each request (None: normal values). Places that nobody stored hold junk."""

    def __init__(self, b2, r, lengths, n_kv, group, dim, page, k=None, v=None):
        self.b2, self.n_head = b2, n_kv * group
        self.new, self.kv = [a for a, _ in lengths], [b for _, b in lengths]
        held = [-(-n // page) for n in self.kv]
        self.stride = max(held) + 1
        self.p = Paged(b2, r, sum(held) + 2, page, n_kv, dim)
        pages = np.split(r.permutation(self.p.ref.n_pages), np.cumsum(held))
        self.table = r.integers(0, 1 << 31, (len(lengths), self.stride))  # entries behind a request's pages: anything
        for i, n in enumerate(self.kv):
            self.table[i, :held[i]] = pages[i]
            kk, vv = (f(n) if f else r.normal(0, 1, (n, n_kv * dim)).astype(np.float32) for f in (k, v))
            full = n // page  # whole pages packed at once, the tokens behind them one by one
            if full:
                packed = kv4.pack_pages(*(x[:full * page].reshape(-1, n_kv, dim) for x in (kk, vv)), page, full)
                self.p.ref.bytes[pages[i][:full]] = packed.reshape(full, *self.p.ref.bytes.shape[1:])
            if n % page:
                self.p.ref.store(pages[i][full] * page + np.arange(n % page), kk[full * page:], vv[full * page:])
        self.p.gpu.copy_(torch.from_numpy(self.p.ref.bytes))
        self.q_start = np.concatenate([[0], np.cumsum(self.new)])
        self.rows = int(self.q_start[-1])
        self.q = r.normal(0, 1.5, (self.rows, self.n_head, dim)).astype(np.float32)
        self.scale = 1.0 / math.sqrt(dim)


def check(b, got, window=0, q=None):
    """Batch.check's bound, with the largest |v| of the element's own block in the place of that of all dims.
    A weight p d is split into two FP16 numbers, off by at most 2^-25 each; a block's d are lifted so that this is 2^-34 of its
    largest d at most, for d up to 2^4. Above, p's own part counts: 2^-25 / 2^(14 - 8), times d, and what FP16 cannot hold of a d that
    is lowered by at most 2^8, 2^-17 where the largest is 2^15 (2^-23 where it is 2^8): together 2^-30 of the largest. By n keys, and a
    sum of all p of 2^-4 at least: n 2^-30 (n 2^-26) of the largest |v| = 8 d.
    Prompts: P's parts are off by 2^-25 of 2^10 at least, and by 2^3 more where a token's values pass 2^16: n 2^-32 of the block's
    largest |v|. Such a token's d are lowered by up to 2^3: what FP16 drops is 2^-25 2^e where the largest is 2^(12 + e) at
    least, 2^-37 of it."""
    table, page = b.table, b.p.ref.page
    y, mag, big = ref.attention(b.p.ref, b.q if q is None else q, table, b.q_start, b.kv, b.scale, window)
    dim, n_kv, group = b.p.ref.dim, b.p.ref.n_kv, b.n_head // b.p.ref.n_kv
    own, all_ = np.zeros(y.shape), np.zeros(y.shape)
    for i, n in enumerate(b.kv):
        v = np.abs(b.p.ref.values(1, table[i][np.arange(n) // page], np.arange(n) % page)).max(0)  # n_kv, dim
        rows = slice(int(b.q_start[i]), int(b.q_start[i + 1]))
        own[rows] = np.repeat(np.repeat(v.reshape(n_kv, -1, 32).max(-1), 32, -1), group, 0)
        all_[rows] = np.repeat(v.max(-1, keepdims=True), group, 0)
    n = max(b.kv)
    tol = 2.0 ** -17 * (1 + big[:, :, None] / 8) * mag + (mag > 0) * (n * own * np.where(own > 128, 2.0 ** -26, 2.0 ** -30) + np.where(all_ > 65536, 2.0 ** -37, 0) * all_)
    assert np.isfinite(got).all() and u32(b.status)[0] == 0
    bad = (np.abs(got - y) - tol) / (mag + 1e-300)
    assert bad.max(initial=0) <= 0, (bad.max(), np.unravel_index(bad.argmax(), bad.shape))


CASES = [(large, small, "blocks") for large, small in ((0, -12), (3, -13), (0, -20), (10, -18), (13, -11), (12, -2), (15, -9), (15, -17))] + [
    (10, -18, "turns"), (13, -11, "turns"), (15, -9, "turns"), (0, -20, "late"), (10, -18, "late"), (15, -17, "late")]


@pytest.mark.parametrize("large,small,kind", CASES)
@pytest.mark.parametrize("dim,n_kv,group", [(64, 2, 4), (128, 1, 12), (160, 2, 3), (256, 2, 4)])
def test_values_of_unlike_blocks_few_rows(b2, dim, n_kv, group, large, small, kind):
    r = rng(400, dim, 50 + large, -small)
    b = Blocks(b2, r, FEW, n_kv, group, dim, 32, v=lambda n: unlike(r, n, n_kv, dim, large, small, kind))
    check(b, b.run(pad=1))


@pytest.mark.parametrize("large,small,kind", CASES)
@pytest.mark.parametrize("dim,group", [(64, 12), (256, 12)])
def test_values_of_unlike_blocks_prompts(b2, dim, group, large, small, kind):
    r = rng(401, dim, 50 + large, -small)
    b = Blocks(b2, r, PROMPTS, 2, group, dim, 32, v=lambda n: unlike(r, n, 2, dim, large, small, kind))
    assert b.rows * b.n_head >= 6144
    check(b, b.run(pad=1))


@pytest.mark.parametrize("window", [5, 70])
@pytest.mark.parametrize("lengths", [FEW, PROMPTS])
def test_values_of_unlike_blocks_in_windows(b2, lengths, window):
    r = rng(404, window)
    b = Blocks(b2, r, lengths, 2, 12, 96, 16, v=lambda n: unlike(r, n, 2, 96, 10, -14, "turns"))
    check(b, b.run(window), window)


@pytest.mark.parametrize("large,small", [(0, -12), (0, -16), (0, -20), (10, -13), (12, -10)])
@pytest.mark.parametrize("dim,group,lengths", [(128, 8, FEW), (64, 12, PROMPTS), (256, 12, PROMPTS)])
def test_keys_of_unlike_blocks_and_queries_that_are_zero_in_the_large_ones(b2, dim, group, lengths, large, small):
    # the scores come from the small blocks alone
    r = rng(402, dim, group)
    b = Blocks(b2, r, lengths, 2, group, dim, 16, k=lambda n: unlike(r, n, 2, dim, large, small, "blocks"))
    b.q = (b.q * (np.arange(dim) // 32 % 2 == 1)).astype(np.float32)
    b.scale = math.sqrt(2.0 / dim) * 2.0 ** -small
    check(b, b.run())


@pytest.mark.parametrize("large", [12, 20, 24])
@pytest.mark.parametrize("dim,group,lengths", [(64, 4, FEW), (128, 8, FEW), (64, 12, PROMPTS), (256, 12, PROMPTS)])
def test_queries_of_unlike_blocks_and_keys_that_are_zero_in_the_large_ones(b2, dim, group, lengths, large):
    # the scores come from the blocks in which a row of q is 2^large below its largest
    r = rng(405, dim, group)
    small = np.arange(dim) // 32 % 2 == 1
    b = Blocks(b2, r, lengths, 2, group, dim, 16, k=lambda n: (r.normal(0, 1, (n, 2, dim)) * small).reshape(n, -1).astype(np.float32))
    b.q = (b.q * np.where(small, 1.0, 2.0 ** large)).astype(np.float32)
    b.scale = math.sqrt(2.0 / dim)
    check(b, b.run())


@pytest.mark.parametrize("std", [1e-30, 1e36])
@pytest.mark.parametrize("lengths", [FEW, PROMPTS])
def test_queries_near_the_ends_of_fp32(b2, lengths, std):
    b = Blocks(b2, rng(406), lengths, 2, 12, 96, 16)
    b.q = (b.q * std).astype(np.float32)
    b.scale = 1.0 / math.sqrt(96) / std
    check(b, b.run())


@pytest.mark.parametrize("lengths", [FEW, PROMPTS])
def test_values_that_grow_from_token_to_token(b2, lengths):
    # a block's largest scale passes the ones before it again and again, each block at other tokens; some blocks begin with zeros
    r = rng(403)

    def values(n):
        tok, block = np.arange(n)[:, None], np.arange(4)
        e = np.where(tok < 20 * block, -1000.0, np.minimum((tok * (block + 1)) // 13 - 16.0, 12.0))
        return (r.normal(0, 1, (n, 2, 4, 32)) * (2.0 ** e)[:, None, :, None]).reshape(n, -1).astype(np.float32)

    b = Blocks(b2, r, lengths, 2, 16, 128, 16, v=values)
    check(b, b.run())


@pytest.mark.parametrize("dim", range(32, 257, 32))
def test_prompts_over_many_keys_of_one_sign_do_not_come_out_small(b2, dim):
    """Tensor memory's sums drop half of their last bit on average, at each of the 12 products of 16 keys in a step of 64: of values
    of one sign all in one direction. A sum that moves on to FP32 every 4 steps is half of what it ends at on average, and its last
    bit 0.72 2^-23 of it: 12 x 4 / 2 / 2 x 0.72 2^-23 = 1.03 10^-6 too small in the mean (first sums, of up to 7 steps of 40, a
    little more), within 2^-19. Over 32 steps it would be 8 10^-6."""
    r = rng(407, dim)
    new, n, page = 64, 2560, 64
    b = Blocks(b2, r, [(new, n)], 1, 96, dim, page, v=lambda n: (1 + 0.25 * r.normal(0, 1, (n, dim))).astype(np.float32))
    got = b.run()
    key = np.arange(n)
    k, v = (b.p.ref.values(i, b.table[0][key // page], key % page)[:, 0] for i in (0, 1))
    s = b.q.astype(np.float64) @ k.T * b.scale
    s = np.where(key > n - new + np.arange(new)[:, None, None], -np.inf, s)
    p = np.exp(s - s.max(-1, keepdims=True))
    y = p @ v / p.sum(-1, keepdims=True)
    assert abs((got / y - 1).mean()) < 2.0 ** -19
