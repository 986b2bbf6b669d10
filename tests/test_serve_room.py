"""Workspaces of the attention over the 4-bit cache: bounded for prompts of any length (no GPU needed)."""
import pytest


def pool(b2, dim=128, n_kv=8, page=64, n_pages=4096):
    return b2.Kv4Pool(0x1000, n_pages, page, n_kv, dim, 1, 0)


@pytest.mark.parametrize("rows", [2048, 32768, 131072, 1 << 20])
@pytest.mark.parametrize("n_req", [1, 64, 4096])
def test_workspace_does_not_grow_with_the_prompts(b2, rows, n_req):
    # Requests of 64 rows (token, head of a group) and more take none. What is left: 63 rows a request at most, in units of 16,
    # four of each KV head, whose tiles (and 16 more a unit) make a line that is cut into ranges of up to 1024, two CTAs an SM
    # at least: each holds 2 x 16 rows of 128 floats, their maxima and sums, and an edge.
    units = min(4 * n_req, rows * 4 // 16 + min(n_req, rows)) * 8
    line = units * (rows // 16 + 16)
    if line >= 1 << 31:
        with pytest.raises(b2.B200QError):
            b2.kv4_attn_workspace(0, pool(b2), rows, 32, n_req, rows, rows)
    else:
        need = b2.kv4_attn_workspace(0, pool(b2), rows, 32, n_req, rows, rows)
        assert 0 < need <= (line / 1024 + 2 * 148) * (2 * 16 * (128 * 4 + 8) + 32)


def test_workspace_does_not_follow_a_loose_bound_on_new_tokens(b2):
    tight = b2.kv4_attn_workspace(0, pool(b2), 4096, 32, 4, 4096, 4096)
    assert b2.kv4_attn_workspace(0, pool(b2), 4096, 32, 4, 1 << 24, 4096) == tight


def test_more_rows_than_a_launch_counts_are_refused(b2):
    with pytest.raises(b2.B200QError):
        b2.kv4_attn_workspace(0, pool(b2, n_kv=1), 1 << 24, 1024, 1, 1 << 24, 1 << 24)
