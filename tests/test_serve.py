"""The operators that serve several sequences, without a GPU: the restated cache layout, and the refusals that come before
any device is touched."""
import ctypes

import numpy as np
import pytest

import serve_ref as ref
from conftest import rng


@pytest.mark.parametrize("dim", range(32, 257, 32))
@pytest.mark.parametrize("which", [0, 1])
def test_every_code_and_scale_has_a_place_of_its_own(b2, dim, which):
    at, shift = ref.code_place(which, dim)
    place = at * 2 + shift // 4
    assert np.array_equal(np.sort(place.reshape(-1)), np.arange(16 * dim) + which * 16 * dim)
    sp = ref.scale_place(which, dim)
    assert np.array_equal(np.sort(sp.reshape(-1)), 16 * dim + which * dim + 2 * np.arange(dim // 2))
    assert b2.kv4_page_bytes(16, 1, dim) == ref.tile_bytes(dim)
    # a block's bytes are a GGUF Q4_0 block's, word by word: element j < 16 in the low nibble of byte j, j + 16 in the high
    word = at.reshape(16, dim // 32, 2, 4, 4)
    assert np.array_equal(word[:, :, 0], word[:, :, 1]) and np.array_equal(word[..., 1:], word[..., :-1] + 1)


def test_restated_store_gives_the_oracles_q4_0(orc):
    # the quantizer against GGUF blocks dequantized by the same formula, at the edges of rounding
    r = rng(70)
    x = r.normal(0, 1, (4, 64)).astype(np.float32)
    x[0, :32] = 0
    x[1, 5], x[1, 9] = 3.0, -3.0  # a tie: the first gives the sign
    codes, d = ref.quantize(x)
    assert d[0, 0] == 0 and np.all(codes[0, :32] == 8)
    assert codes[1, 5] == 0 and codes[1, 9] == 15 and d[1, 0] == np.float16(-3.0 / 8)
    for i in range(4):
        for b in range(2):
            blk, dd = x[i, 32 * b:32 * b + 32], np.float32(d[i, b])
            back = (codes[i, 32 * b:32 * b + 32].astype(np.float32) - 8) * dd
            # a code is off by at most half a step, but for the end of the range: a whole step (code 16 is cut to 15)
            assert np.all(np.abs(back - blk) <= np.abs(dd) * 1.01 + 1e-6)


def test_page_bytes(b2):
    assert b2.kv4_page_bytes(64, 4, 256) == 64 * 4 * 2 * (256 // 32) * 18  # K and V, 18 bytes a block
    for bad in ((0, 4, 128), (24, 4, 128), (16, 0, 128), (16, 4, 48), (16, 4, 288), (4112, 1, 32)):
        assert b2.kv4_page_bytes(*bad) == 0


def pool_of(b2, **kw):
    a = dict(base=4096, n_pages=4, page_tokens=16, n_kv_head=2, head_dim=64, n_layers=1, layer_bytes=0)
    a.update(kw)
    return b2.Kv4Pool(*a.values())


@pytest.mark.parametrize("kw,why", [
    (dict(head_dim=48), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=288), "head_dim"),
    (dict(page_tokens=24), "page_tokens"), (dict(page_tokens=0), "page_tokens"), (dict(page_tokens=8192), "page_tokens"),
    (dict(n_kv_head=0), "n_kv_head"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 28, page_tokens=64), "n_pages")])
def test_pools_that_no_call_takes(b2, kw, why):
    pool = pool_of(b2, **kw)
    with pytest.raises(b2.B200QError, match=why):
        b2.kv4_store(0, pool, 4096, 4096, 4096, 1)
    with pytest.raises(b2.B200QError, match=why):
        b2.kv4_load(0, pool, 4096, 1, 4096, 4096)
    with pytest.raises(b2.B200QError, match=why):
        b2.kv4_attn(0, pool, 4096, 4096, 1, 2, 4096, 4, 4096, 4096, 1, 1, 16, 1.0, 4096, 1 << 20)
    with pytest.raises(b2.B200QError, match=why):
        b2.kv4_reorder(0, pool, 4096, 4, 4096, 4096, 1, 2)
    with pytest.raises(b2.B200QError):
        b2.kv4_attn_workspace(0, pool, 1, 2, 1, 1, 16)


def test_attention_shapes_that_are_refused(b2):
    pool = pool_of(b2)
    ok = dict(n_rows=1, n_head=4, stride=4, n_req=1, max_q=1, max_kv=64, scale=1.0, q_stride=0, q_head=0, y_stride=0)

    def call(**kw):
        a = dict(ok, **kw)
        b2.kv4_attn(0, pool, 4096, 4096, a["n_rows"], a["n_head"], 4096, a["stride"], 4096, 4096, a["n_req"], a["max_q"], a["max_kv"],
                    a["scale"], 4096, 1 << 30, a["q_stride"], a["q_head"], a["y_stride"])

    for kw, why in ((dict(n_head=3), "n_head"), (dict(n_head=0), "n_head"), (dict(n_req=0), "n_req"), (dict(n_req=65536), "n_req"),
                    (dict(max_q=0), "max_q"), (dict(max_kv=0), "max_kv"), (dict(max_kv=65), "max_kv"), (dict(stride=0), "max_kv"),
                    (dict(q_stride=255), "stride"), (dict(q_head=63), "stride"), (dict(y_stride=255), "stride"),
                    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(n_rows=1 << 25), "n_rows")):
        with pytest.raises(b2.B200QError, match=why):
            call(**kw)
    assert b2.kv4_attn_workspace(0, pool, 1, 4, 1, 1, 64) > 0


def test_map_select_and_reorder_shapes_that_are_refused(b2):
    def map_(n_req=1, stride=4, page=16, rows=4):
        b2.block_map(0, n_req, 4096, 4096, 4096, stride, page, 4096, 4, 4096, 4096, 4096, 4096, 4096, 4096, rows)

    for kw, why in ((dict(n_req=0), "n_req"), (dict(n_req=65536), "n_req"), (dict(stride=0), "table_stride"), (dict(page=17), "page_tokens"),
                    (dict(stride=1 << 28, page=64), "tokens"), (dict(rows=1 << 31), "n_rows")):
        with pytest.raises(b2.B200QError, match=why):
            map_(**kw)

    def select(n_req=1, beams=2, vocab=100, n_out=4, room=1 << 20, stride=0):
        b2.beam_select(0, 4096, vocab, 4096, n_req, beams, n_out, 4096, 4096, 4096, 4096, room, stride)

    for kw, why in ((dict(n_req=0), "n_req"), (dict(beams=0), "beams"), (dict(beams=33), "beams"), (dict(vocab=0), "vocab"),
                    (dict(vocab=(1 << 20) + 1), "vocab"), (dict(n_out=0), "n_out"), (dict(n_out=65), "n_out"), (dict(stride=99), "logits_stride")):
        with pytest.raises(b2.B200QError, match=why):
            select(**kw)
        if "stride" not in kw:
            a = dict(n_req=1, beams=2, vocab=100, n_out=4)
            a.update(kw)
            with pytest.raises(b2.B200QError):
                b2.beam_select_workspace(0, *a.values())

    def reorder(n_req=1, beams=2, row=16, layers=1, sl=0, dl=0, src=4096, dst=8192):
        b2.beam_reorder(0, src, dst, 4096, n_req, beams, row, layers, sl, dl)

    for kw, why in ((dict(n_req=0), "n_req"), (dict(beams=0), "beams"), (dict(beams=33), "beams"), (dict(row=0), "row_bytes"),
                    (dict(layers=0), "n_layers"), (dict(layers=65536), "n_layers"), (dict(sl=31), "layer"), (dict(dl=31), "layer"),
                    (dict(dst=4096, sl=32, dl=64), "in place")):
        with pytest.raises(b2.B200QError, match=why):
            reorder(**kw)
    with pytest.raises(b2.B200QError, match="n_layers"):
        b2.kv4_reorder(0, pool_of(b2, n_layers=0), 4096, 4, 4096, 4096, 1, 2)
    with pytest.raises(b2.B200QError, match="layer_bytes"):
        b2.kv4_reorder(0, pool_of(b2, n_layers=2, layer_bytes=64), 4096, 4, 4096, 4096, 1, 2)


def test_a_null_pool_is_refused(b2):
    err = ctypes.create_string_buffer(256)
    assert b2.lib().b200q_kv4_store(0, None, 4096, 4096, 4096, 1, 0, 0, None, None, err, 256) == -1
    assert b"pool" in err.value


def test_restated_block_map():
    t, kv, qs, sl, pos, cur, short = ref.block_map([0, 15, 16], [17, 1, 0], np.zeros((3, 2)), 16, [9, 8, 7], 1, 20)
    assert not short and kv == [17, 16, 16] and qs == [0, 17, 18, 18] and cur == 3
    assert list(t[0]) == [8, 7] and sl[0] == 8 * 16 and sl[16] == 7 * 16 and sl[17] == 15 and sl[18] == ref.NO_SLOT
