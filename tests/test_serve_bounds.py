"""Sizes at the ends of what the calls and commands for several sequences take: steps without rows, and products of sizes
that pass 64 bits. No GPU needed, but for the tests marked so."""
import subprocess
import sys

import pytest

import plan_limits
from conftest import ROOT, load_package

b2 = load_package()


def pool(dim=64, n_kv=2, page=16, n_pages=8):
    return b2.Kv4Pool(4096, n_pages, page, n_kv, dim, 1, 0)


ROOM_OF_NO_ROWS = """
import sys
sys.path.insert(0, "tests")
from conftest import load_package
b2 = load_package()
for dim in range(32, 257, 32):
    for n_head in (2, 4, 64):
        for n_req, max_q, max_kv in ((1, 1, 512), (4096, 1, 1), (7, 1 << 24, 1 << 28), (1, 16, 300)):
            h = b2.Kv4Pool(4096, 8, 16, 2, dim, 1, 0)
            none, one = (b2.kv4_attn_workspace(0, h, rows, n_head, n_req, max_q, max_kv) for rows in (0, 1))
            assert 0 < none <= one, (dim, n_head, n_req, none, one)
"""


def test_the_workspace_of_no_rows():
    """In a process of its own: an integer division by zero would end this one."""
    got = subprocess.run([sys.executable, "-c", ROOM_OF_NO_ROWS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, (got.returncode, got.stderr)


def empty_attention(n_req=2):
    return b2.kv4_attn_cmd(4, 1024, 4096, 0, 4, 64, 128, n_req, 0, 2, 64, 0.125, b2.kv4_geometry(2, 64, 16), 256, 8)


def test_an_attention_of_no_rows_plans():
    assert b2.plan(empty_attention())[0] == 0


@pytest.mark.gpu
def test_an_attention_of_no_rows_runs_in_lists_and_graphs():
    import numpy as np
    cl = b2.cmd_list(b2.add(16, 0, 16, 32), empty_attention(), b2.add(16, 0, 16, 48))
    layer = b2.kv4_page_bytes(16, 2, 64) * 8
    with b2.Context(device=0, weight_bytes=1 << 20, act_floats=8192, state_rows=8, kv_bytes=256 + layer) as ctx:
        act = np.arange(8192, dtype=np.float32)
        ctx.write(0, act)
        want = act.copy()
        want[32:48] = want[48:64] = act[:16] + act[16:32]
        assert ctx.run(cl) == 0
        assert np.array_equal(ctx.read(0, 8192), want)
        ctx.write(0, act)
        g = ctx.graph(cl)
        g.launch()
        ctx.synchronize()
        assert np.array_equal(ctx.read(0, 8192), want)
        g.close()


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    return plan_limits.build(str(tmp_path_factory.mktemp("plan")))


def raw(*slots):
    return b2.cmd_list(*(b2.cmd(*s) for s in slots))


@pytest.mark.parametrize("n_req,beams,rows,layers,step", [
    (32768, 32, 1 << 29, 32768, 0),               # layers x a layer's rows: 2^64
    (8192, 32, 1 << 31, 32768, 0),
    (32768, 32, 1 << 29, 32769, 0),               # 2^64 and a layer more
    (65535, 32, (1 << 32) - 1, 65535, 0),
    (1, 2, 256, 3, 1 << 9), (1, 2, 256, 3, 512), (1, 2, 513, 1, 0), (1, 1, 1, 2, 1024)])
def test_state_rows_behind_the_buffer_are_refused_whatever_their_product(plan, n_req, beams, rows, layers, step):
    assert n_req * beams * rows + (layers - 1) * (step or n_req * beams * rows) > 1024
    for dst in (0, 512):
        assert plan(raw((b2.OP_BEAM_REORDER, n_req, beams, 0, 0, dst, rows, layers), (step,))) == 1


@pytest.mark.parametrize("n_req,beams,rows,layers,step,src,dst", [
    (1, 2, 256, 2, 0, 0, 0), (1, 2, 256, 1, 0, 0, 512), (1, 1, 1, 2, 1023, 0, 0), (4, 4, 8, 8, 128, 0, 0), (1, 1, 1024, 1, 0, 0, 0), (1, 2, 4, 3, 50, 916, 800)])
def test_state_rows_up_to_the_buffers_end_are_taken(plan, n_req, beams, rows, layers, step, src, dst):
    assert plan(raw((b2.OP_BEAM_REORDER, n_req, beams, 0, src, dst, rows, layers), (step,))) == 0


def attention(n_head, n_rows, q_stride, q_head_stride, y=1 << 25):
    # one KV head of 32; q before y
    geo = b2.kv4_geometry(1, 32, 16)
    return raw((b2.OP_KV4_ATTN, n_head, 1 << 20, y, 0, 4, 64, 128), (1, n_rows, 1, 64, 0x3F800000, 0, q_stride, q_head_stride), (geo, 0, 8, 0))


@pytest.mark.parametrize("n_head,n_rows,q_head_stride", [
    (510, 16777124, 2155916975),                   # the last row's place is 2^64 and some 7 million
    (1024, (1 << 24) - 1, (1 << 32) - 1), (1024, 1 << 24, 1 << 30), (512, (1 << 23) + 1, 1 << 31), (1, 2, (1 << 32) - 1)])
def test_queries_behind_the_buffer_are_refused_whatever_their_product(plan, n_head, n_rows, q_head_stride):
    # an act buffer that y fits, and q does not (the planner's arithmetic alone: no GPU holds y where the product wraps)
    act = (1 << 25) + n_rows * n_head * 32
    assert (1 << 20) + ((n_rows - 1) * n_head + n_head - 1) * q_head_stride + 32 > act
    assert plan(attention(n_head, n_rows, 0, q_head_stride), act_floats=act) == 1


def test_queries_up_to_the_buffers_end_are_taken(plan):
    # 3 rows of 4 heads 100 floats apart, the rows 500: the last float of q is the buffer's
    for stride, head, n in ((500, 100, 2 * 500 + 3 * 100 + 32), (0, 100, 2 * 400 + 3 * 100 + 32), (0, 0, 3 * 128)):
        cl = attention(4, 3, stride, head, y=4096)
        assert plan(cl, act_floats=(1 << 20) + n) == 0
        assert plan(cl, act_floats=(1 << 20) + n - 1) == 1


@pytest.mark.parametrize("n_head,q_stride,q_head_stride", [
    (17, 0, 1 << 60),           # 16 x 2^60 floats: a row's width wraps to one head's
    (17, 64, 1 << 60), (16, 0, 1 << 60), (2, 0, (1 << 64) - 64), (2, 0, (1 << 32) + 1), (5, 1 << 33, 1 << 33), (3, (1 << 32) + 1, 64)])
def test_query_strides_beyond_all_memory_are_refused_before_the_device(n_head, q_stride, q_head_stride):
    h = pool(n_kv=1)
    with pytest.raises(b2.B200QError, match="stride"):
        b2.kv4_attn(0, h, 4096, 4096, 2, n_head, 4096, 4, 4096, 4096, 1, 1, 64, 1.0, 4096, 1 << 30, q_stride, q_head_stride)


@pytest.mark.parametrize("k_stride,v_stride", [(1 << 32, 128), (128, 1 << 32), (1 << 32, 0)])
def test_rows_whose_bytes_pass_64_bits_are_refused_before_the_device(k_stride, v_stride):
    n = (1 << 30) + 1  # rows 2^34 bytes apart: the last one lies 2^64 bytes behind the first
    for call in (lambda: b2.kv4_store(0, pool(), 4096, 4096, 4096, n, k_stride, v_stride),
                 lambda: b2.kv4_load(0, pool(), 4096, n, 4096, 4096, k_stride, v_stride)):
        with pytest.raises(b2.B200QError, match="rows and their stride"):
            call()
