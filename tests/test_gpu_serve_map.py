"""Block maps: requests that take thousands of pages beside ones that take few, and table entries whose slots 32 bits cannot count."""
import numpy as np
import pytest

import serve_ref as ref
from conftest import rng
from test_gpu_serve import SKIP, run_map

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_block_map_of_long_requests_beside_short_ones(b2):
    r = rng(340)
    past = r.integers(0, 200, 70)
    fresh = r.integers(0, 160, 70)  # up to eleven pages: on both sides of what a thread takes by itself
    fresh[3], fresh[33], fresh[34], fresh[69] = 70000, 4000, 1, 33000
    page = 16
    stride = int(max(-(-(past + fresh) // page)))
    table = r.integers(0, 1 << 20, (70, stride))
    need = int(sum(-(-(past + fresh) // page) - -(-past // page)))
    free, rows = r.permutation(need + 3), int(fresh.sum())
    for held in (len(free), need - 50):  # the last request runs short
        got = run_map(b2, past, fresh, table, page, free[:held], 2, rows)
        want = ref.block_map(past, fresh, table, page, list(free[:held]), 2, rows)
        for g, w in zip(got[:5], want[:5]):
            assert np.array_equal(np.asarray(g, np.int64), np.asarray(w, np.int64))
        assert got[5] == want[5] and got[6] == (b2.SERVE_SHORT if want[6] else 0)


@pytest.mark.parametrize("page", [16, 48, 4096])
def test_block_map_names_no_slot_of_a_page_that_passes_32_bits(b2, page):
    most = 0xFFFFFFFF // page  # pages 0 .. most - 1 have slots below 2^32 - 1
    got = run_map(b2, [0, 0, 0], [3, 2, 1], np.zeros((3, 1)), page, [most - 1, most, 1 << 31], 0, 6)
    first = (most - 1) * page
    assert [int(x) for x in got[3]] == [first, first + 1, first + 2, SKIP, SKIP, SKIP]
    assert [int(x) for x in got[4]] == [0, 1, 2, 0, 1, 0] and got[6] == b2.SERVE_PAGE
