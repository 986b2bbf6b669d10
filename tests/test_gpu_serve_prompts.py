"""Attention over the 4-bit cache for long prompts (the tensor-core kernel with its accumulators in tensor memory, which calls
with many rows give their long requests to) and for units of up to sixteen rows, against 64 bits: head sizes, groups, windows,
ragged lengths beside single tokens, rows without a key, values that are no numbers, pages that are none, strides, streams and
captured graphs. Tolerances: those of Batch.check."""
import numpy as np
import pytest

import serve_ref as ref
from conftest import rng
from test_gpu_serve import Batch, dev, u32

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::RuntimeWarning")]

# short requests and single tokens between the prompts; a prompt of its own keys alone, one behind others, one whose first
# rows see no key, one that ends in the middle of a tile and of a page
MIXED = [(150, 150), (1, 90), (3, 17), (97, 300), (0, 30), (64, 64), (1, 1), (129, 257), (70, 61), (5, 5)]


@pytest.mark.parametrize("dim", range(32, 257, 32))
@pytest.mark.parametrize("n_kv,group", [(2, 8), (1, 16), (3, 5)])
def test_prompts_beside_single_tokens(b2, dim, n_kv, group):
    b = Batch(b2, rng(300, dim, group), MIXED, n_kv, group, dim, 48)
    assert b.rows * b.n_head >= 6144
    b.check(b.run(pad=3))
    assert u32(b.status)[0] == 0


@pytest.mark.parametrize("window", [1, 16, 63, 64, 65, 200])
@pytest.mark.parametrize("dim", [64, 96, 256])
def test_prompts_with_windows(b2, dim, window):
    b = Batch(b2, rng(301, dim, window), MIXED + [(200, 700)], 2, 8, dim, 16)
    b.check(b.run(window), window)


@pytest.mark.parametrize("group,new", [(64, 6), (1, 400), (7, 150), (33, 61), (128, 30)])
def test_prompts_and_groups_of_heads(b2, group, new):
    # rows (token, head) of a tile that begin and end inside a token; a group larger than a tile of 128 rows
    n_kv = -(-6144 // (group * (new + 1 + new // 2)))
    b = Batch(b2, rng(302, group), [(new, new + 9), (1, 33), (new // 2, new)], n_kv, group, 64, 32)
    assert b.rows * b.n_head >= 6144
    b.check(b.run())


@pytest.mark.parametrize("q_pad,head_pad,y_pad", [(1, 0, 0), (0, 4, 4), (4, 4, 3), (3, 1, 1)])
@pytest.mark.parametrize("dim", [32, 160, 256])
def test_prompts_out_of_and_into_wider_rows(b2, dim, q_pad, head_pad, y_pad):
    b = Batch(b2, rng(303, dim), [(130, 131), (2, 50), (101, 160)], 2, 16, dim, 16)
    b.check(b.run(pad=2, q_pad=q_pad, head_pad=head_pad, y_pad=y_pad))


@pytest.mark.parametrize("k_std,q_std", [(6.0, 6.0), (1e-3, 1.0), (1.0, 1e4)])
def test_prompts_at_other_magnitudes(b2, k_std, q_std):
    b = Batch(b2, rng(304), [(150, 190), (1, 300), (60, 333)], 2, 16, 128, 16, k_std=k_std, q_std=q_std)
    if q_std > 100:
        b.scale /= q_std
    b.check(b.run())


@pytest.mark.parametrize("std", [1e-3, 30.0, 3000.0])
def test_prompts_at_other_magnitudes_of_v(b2, std):
    r = rng(305)
    b = Batch(b2, r, [(150, 190), (1, 300), (60, 333)], 2, 16, 64, 16)
    for i, n in enumerate(b.kv):
        slots = b.table[i][np.arange(n) // 16] * 16 + np.arange(n) % 16
        b.p.fill(slots, r.normal(0, 1, (n, 128)).astype(np.float32), r.normal(0, std, (n, 128)).astype(np.float32))
    b.check(b.run())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_pass_a_nan_on_where_it_is_seen_and_nowhere_else(b2, dim):
    n, at = 150, 70
    b = Batch(b2, rng(306, dim), [(n, n), (1, 90), (100, 150)], 2, 16, dim, 16)
    slot = b.table[0][at // 16] * 16 + at % 16
    keep = b.p.ref.bytes.copy()
    k = np.ones((1, 2 * dim), np.float32)
    k[0, 3] = np.nan                                      # K of one token of request 0, KV head 0
    b.p.fill([slot], k, np.ones((1, 2 * dim), np.float32))
    got = b.run()
    assert np.isnan(got[at:n, :16]).all()                 # every row from its position on
    assert np.isfinite(got[:at]).all() and np.isfinite(got[:, 16:]).all() and np.isfinite(got[n:]).all()
    b.p.ref.bytes[:] = keep
    b.p.gpu.copy_(torch.from_numpy(keep))
    v = np.ones((1, 2 * dim), np.float32)
    v[0, dim + 40] = np.inf                               # V, KV head 1, the dims 32..63
    b.p.fill([slot], np.zeros((1, 2 * dim), np.float32), v)
    got = b.run()
    assert np.isnan(got[at:n, 16:, 32:64]).all()
    rest = got.copy()
    rest[at:n, 16:, 32:64] = 0
    assert np.isfinite(rest).all()
    b.p.ref.bytes[:] = keep
    b.p.gpu.copy_(torch.from_numpy(keep))
    q = b.q.copy()
    q[5, 1, 5], q[n + 20, 31, 0] = np.nan, np.inf
    got = b.run(q=q)
    assert np.isnan(got[5, 1]).all() and np.isnan(got[n + 20, 31]).all()
    rest = got.copy()
    rest[5, 1] = rest[n + 20, 31] = 0
    assert np.isfinite(rest).all()


def test_prompts_leave_out_what_lies_outside_and_say_so(b2):
    b = Batch(b2, rng(307), [(150, 150), (1, 60), (90, 200)], 2, 16, 64, 16)
    whole = b.run()
    b.check(whole)
    got = b.run(max_kv=150)
    assert u32(b.status)[0] == b2.SERVE_REQUEST and (got[151:] == 7).all() and np.array_equal(got[:151], whole[:151])
    got = b.run(max_q=90)
    assert u32(b.status)[0] == b2.SERVE_REQUEST and (got[:150] == 7).all() and np.array_equal(got[150:], whole[150:])
    got = b.run(q_start=[0, 150, 151, 1 << 30], max_q=1 << 20)
    assert u32(b.status)[0] == b2.SERVE_REQUEST and (got[151:] == 7).all()
    # pages that are none: their tokens are left out
    t = b.table.copy()
    t[2, 3], t[2, 7] = b.p.ref.n_pages, ref.NO_SLOT
    got = b.run(table=t)
    assert u32(b.status)[0] == b2.SERVE_PAGE and np.array_equal(got[:151], whole[:151]) and np.isfinite(got).all()
    for row, h in ((0, 0), (0, 31), (40, 17), (89, 5)):
        key = np.array([x for x in range(110 + row + 1) if x // 16 not in (3, 7)])
        k, v = (b.p.ref.values(i, b.table[2][key // 16], key % 16)[:, h // 16] for i in (0, 1))
        s = k @ b.q[151 + row, h].astype(np.float64) * b.scale
        p = np.exp(s - s.max())
        assert np.allclose(got[151 + row, h], p @ v / p.sum(), atol=1e-4)
    t[0, :] = ref.NO_SLOT
    assert (b.run(table=t)[:150] == 0).all()


def test_prompts_give_the_same_bits_in_every_stream_and_from_a_graph(b2):
    b = Batch(b2, rng(308), [(150, 150), (1, 700), (90, 200)], 2, 16, 128, 32)
    want = b.run()
    for _ in range(2):
        assert np.array_equal(b.run(stream=torch.cuda.Stream().cuda_stream), want)
    # a captured call follows the lengths that lie on the device when it is replayed
    nh, dim, n = b.n_head, 128, b.rows
    need = b2.kv4_attn_workspace(0, b.p.h, n, nh, 3, 150, 700)
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    q, table, q_start, kv = dev(b.q), dev(b.table), dev(b.q_start), dev(b.kv)
    y = torch.full((n, nh, dim), 7.0, device="cuda")
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        b2.kv4_attn(0, b.p.h, q.data_ptr(), y.data_ptr(), n, nh, table.data_ptr(), b.stride, q_start.data_ptr(), kv.data_ptr(), 3, 150, 700,
                    b.scale, room.data_ptr(), need, stream=torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(y.cpu().numpy(), want)
    b.new, b.kv = [20, 130, 0], [25, 500, 9]
    b.q_start = np.array([0, 20, 150, 150])
    q_start.copy_(dev(b.q_start))
    kv.copy_(dev(b.kv))
    y.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    assert (got[150:] == 7).all()
    # what request 1 sees behind its first 700 keys was never stored; 500 of them were
    whole, b.q = b.q, b.q[:150]
    b.check(got[:150])
    b.q = whole


@pytest.mark.parametrize("dim", range(32, 257, 32))
@pytest.mark.parametrize("group,new", [(3, 3), (12, 1), (6, 2), (13, 1), (5, 3), (16, 1), (17, 1), (4, 5)])
def test_units_of_nine_to_sixteen_rows(b2, dim, group, new):
    b = Batch(b2, rng(309, dim, group), [(new, 130), (1, 1), (new, new), (1, 65), (new, 1), (0, 5), (new, 333)], 2, group, dim, 32)
    b.check(b.run(pad=1))
    b.check(b.run(window=50), 50)


@pytest.mark.parametrize("dim,y_pad,window", [(32, 0, 0), (64, 1, 0), (32, 0, 2500)])
def test_prompts_on_long_caches(b2, dim, y_pad, window):
    # Sums in tensor memory drop what is below their last bit: over 9000 keys without a break (12 products of 16 keys each a
    # step of 64, half of 2^-23 lost each time) O would come out 2^-24 * 12 * 141 / 2 > 2^-15 too small, four times the bound
    b = Batch(b2, rng(310, dim), [(60, 9000), (30, 4097), (1, 9100), (20, 2048), (18, 2049)], 1, 64, dim, 64)
    b.check(b.run(window, y_pad=y_pad), window)


@pytest.mark.parametrize("dim", [64, 256])
def test_prompts_before_many_values_that_are_no_numbers(b2, dim):
    n, at = 400, 150  # V of every token from `at` on is infinite in block 1 of KV head 0: the rows before it do not see it
    b = Batch(b2, rng(311, dim), [(n, n), (1, 90)], 2, 8, dim, 16)
    tok = np.arange(at, n)
    v = np.ones((len(tok), 2 * dim), np.float32)
    v[:, 40] = np.inf
    b.p.fill(b.table[0][tok // 16] * 16 + tok % 16, np.zeros((len(tok), 2 * dim), np.float32), v)
    got = b.run()
    assert np.isnan(got[at:n, :8, 32:64]).all()
    rest = got.copy()
    rest[at:n, :8, 32:64] = 0
    assert np.isfinite(rest).all()


@pytest.mark.parametrize("n_req", [300, 600])
def test_prompts_among_hundreds_of_single_tokens(b2, n_req):
    # more requests than threads count one by one; the bound on new tokens far above what any request has
    lengths = [(1, 1 + i % 70) for i in range(n_req)]
    lengths[7], lengths[n_req // 2], lengths[-1] = (200, 260), (90, 90), (150, 151)
    b = Batch(b2, rng(312, n_req), lengths, 2, 8, 32, 16)
    b.check(b.run(pad=5, max_q=1 << 20))
    assert u32(b.status)[0] == 0
    got = b.run(q_start=np.concatenate([b.q_start[:n_req // 2 + 1], [0], b.q_start[n_req // 2 + 2:]]))  # the rows of one run backwards
    assert u32(b.status)[0] & b2.SERVE_REQUEST
    # those before it are served (where the line of tiles is cut has moved with its length, and the roundings with it)
    k = n_req // 2
    rows = int(b.q_start[k])
    assert (got[rows:] == 7).all()
    b.q_start, b.kv, b.q = b.q_start[:k + 1], b.kv[:k], b.q[:rows]
    b.check(got[:rows])


@pytest.mark.parametrize("dim,group,prompt", [(32, 2, False), (256, 1, False), (64, 4, True)])
def test_as_many_requests_as_a_call_takes(b2, dim, group, prompt):
    most = 5 if dim == 256 else 23  # keys (quantizing them on the host takes the time here)
    lengths = [(1, 1 + i % most) if i % 5 else (0, i % most) for i in range(4096)]
    if prompt:
        lengths[2000], lengths[4095] = (70, 90), (33, 33)
    b = Batch(b2, rng(313, dim), lengths, 1, group, dim, 16)
    b.check(b.run(pad=1))
    assert u32(b.status)[0] == 0
