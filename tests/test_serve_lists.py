"""The commands for several sequences (opcodes 18 .. 23) in lists: planning and refusals and the host packing on the CPU; on the
GPU the same bits as the direct calls, a step of several sequences through lists and a captured graph, and the hybrid
decoder with its K and V in the 4-bit cache against the oracle and the restatement."""
import math

import numpy as np
import pytest

import serve_ref as ref
from conftest import load_package, rng

b2 = load_package()
import fpga_llama_gguf_b200.decode as D  # noqa: E402
import fpga_llama_gguf_b200.kv4 as kv4  # noqa: E402

SMALL = D.Shape(hidden=1024, ffn=2048, n_layers=4, vocab=4096, gdn_heads=4, n_head=4, n_kv_head=2, head_dim=128, rope_dims=32, kv_ctx=640, prefill=64,
                head_piece=2048)


@pytest.mark.parametrize("dim,page,n_kv,tokens", [(32, 16, 1, 1), (96, 48, 3, 100), (128, 16, 2, 33), (256, 64, 1, 64), (160, 32, 2, 50)])
def test_packed_pages_are_what_store_writes(dim, page, n_kv, tokens):
    r = rng(110, dim)
    k, v = (r.normal(0, 2, (tokens, n_kv, dim)).astype(np.float32) for _ in range(2))
    k[0, 0, :32] = 0
    n_pages = -(-tokens // page) + 1
    p = ref.Pool(n_pages, page, n_kv, dim)
    at, shift = ref.code_place(0, dim)
    p.store(np.arange(tokens), k.reshape(tokens, -1), v.reshape(tokens, -1))
    got = kv4.pack_pages(k, v, page, n_pages).reshape(p.bytes.shape)
    for which, x in ((0, k), (1, v)):
        t = np.arange(tokens)
        q = ref.Pool(n_pages, page, n_kv, dim)
        q.bytes[:] = got
        assert np.array_equal(q.values(which, t // page, t % page), p.values(which, t // page, t % page))
        rest = np.arange(tokens, n_pages * page)
        assert (q.values(which, rest // page, rest % page) == 0).all()
    with pytest.raises(ValueError):
        kv4.pack_pages(k, v, page, (tokens - 1) // page)


GEO = b2.kv4_geometry(2, 64, 16)


def commands(**kw):
    """A valid command of each kind, 64 floats apart."""
    g = dict(geo=GEO)
    g.update(kw)
    return {
        "map": b2.block_map_cmd(2, 0, 64, 128, 4, 192, 8, 256, 320, 384, 448, 512, 4, 16),
        "store": b2.kv4_store_cmd(3, 1024, 2048, 0, g["geo"], 256, 8),
        "attn": b2.kv4_attn_cmd(4, 1024, 4096, 0, 4, 64, 128, 2, 3, 2, 64, 0.125, g["geo"], 256, 8),
        "select": b2.beam_select_cmd(1, 2, 100, 1024, 0, 4, 64, 128, 192),
        "reorder": b2.beam_reorder_cmd(1, 2, 0, 0, 512, 128, 2),
        "pages": b2.kv4_reorder_cmd(1, 2, 0, 4, 64, 128, g["geo"], 0, 8, 2, 8 * 2 * 18 * 64),
    }


def test_valid_commands_plan_and_take_their_slots():
    cl = b2.cmd_list(*commands().values())
    st, passes = b2.plan(cl)
    assert st == 0 and [p["kind"] for p in passes] == ["ext"] * 6 and [p["count"] for p in passes] == [2, 2, 3, 2, 2, 2]
    for name, c in commands().items():  # cut short: the first slot is named
        st, _ = b2.plan(b2.cmd_list(b2.add(16, 0, 16, 32), c[:-8]))
        assert st == 2, name


@pytest.mark.parametrize("name,word,value", [
    ("map", 1, 0), ("map", 1, 65536), ("map", 5, 0), ("map", 8 + 6, 24), ("map", 8 + 7, 1), ("map", 2, 8), ("map", 8, 128), ("map", 8 + 5, 1 << 31),
    ("store", 7, b2.kv4_geometry(2, 64, 16) & 0xFFFF), ("store", 7, b2.kv4_geometry(0, 64, 16)), ("store", 7, b2.kv4_geometry(2, 320, 16)),
    ("store", 5, 127), ("store", 6, 1), ("store", 9, 0), ("store", 10, 1), ("store", 4, 3),
    ("attn", 1, 3), ("attn", 1, 0), ("attn", 5, 3), ("attn", 8, 0), ("attn", 10, 0), ("attn", 11, 0), ("attn", 12, 0x7F800000), ("attn", 14, 255),
    ("attn", 15, 63), ("attn", 19, 255), ("attn", 20, 1), ("attn", 3, 1024), ("attn", 8, 4097),
    ("select", 1, 0), ("select", 2, 33), ("select", 3, 0), ("select", 5, 99), ("select", 7, 65), ("select", 8, 64 + 16), ("select", 8, 1024), ("select", 11, 1),
    ("reorder", 1, 0), ("reorder", 2, 0), ("reorder", 6, 0), ("reorder", 7, 0), ("reorder", 5, 256), ("reorder", 8, 255), ("reorder", 9, 1),
    ("pages", 2, 33), ("pages", 4, 0), ("pages", 10, 0), ("pages", 11, 1), ("pages", 12, 1), ("pages", 6, 0)])
def test_commands_that_are_refused(name, word, value):
    c = commands()[name].copy()
    c[word] = value
    if (name, word, value) == ("select", 8, 64 + 16):
        c[9] = 64  # two outputs in one place
        c[8] = 64
    st, _ = b2.plan(b2.cmd_list(b2.add(16, 0, 16, 32), c))
    assert st == 2


@pytest.mark.parametrize("page", [16, 64])
def test_the_4bit_decoders_lists_plan(page):
    for shape in (SMALL, D.SHAPE_4B):
        m = D.HybridDecoder(shape, kv4_page=page)
        m.handles = {name: (k + 1) * 256 for k, (name, *_) in enumerate(m.matrices())}
        for cl in m.token_lists():
            assert b2.plan(cl)[0] == 0
    with pytest.raises(ValueError, match="4-bit"):
        m.token_graph()


@pytest.mark.parametrize("world", [2, 4, 8])
def test_the_4bit_decoders_lists_plan_for_every_rank(world):
    for rank in range(world):
        m = D.HybridDecoder(D.SHAPE_4B, kv4_page=64, world=world, rank=rank)
        m.handles = {name: (k + 1) * 256 for k, (name, *_) in enumerate(m.matrices())}
        for cl in m.token_lists():
            assert b2.plan(cl)[0] == 0
        assert m.context_config()["kv_bytes"] == m.kv_bytes() == m.kv4_pool(m.s.n_attn)[0]


def test_a_ranks_pages_hold_its_heads_of_the_whole_cache():
    page, s = 16, SMALL
    whole = D.HybridDecoder(s, seed=9, kv4_page=page)
    raw = whole.initial_kv()
    for rank in range(2):
        m = D.HybridDecoder(s, seed=9, kv4_page=page, world=2, rank=rank)
        mine = m.initial_kv()
        for j in range(s.n_attn):
            (at, n_pages), (at1, n1) = whole.kv4_pool(j), m.kv4_pool(j)
            assert n_pages == n1
            size = n_pages * b2.kv4_page_bytes(page, s.n_kv_head, s.head_dim)
            heads = raw[at:at + size].reshape(n_pages, s.n_kv_head, -1)
            assert np.array_equal(mine[at1:at1 + size // 2].reshape(n1, 1, -1), heads[:, rank:rank + 1])


@pytest.mark.gpu
def test_commands_give_the_direct_calls_bits():
    torch = pytest.importorskip("torch")
    r = rng(111)
    n, n_kv, dim, nh, page, stride, vocab = 5, 2, 96, 4, 32, 4, 300
    width, geo = n_kv * dim, b2.kv4_geometry(n_kv, dim, page)
    n_pages = n * stride
    past = np.array([0, 31, 32, 60, 100])
    fresh = np.array([1, 2, 1, 3, 1])
    rows = int(fresh.sum())
    table = np.zeros((n, stride), np.int64)
    perm = r.permutation(n_pages)
    at = 0
    for i, p in enumerate(past):
        held = -(-p // page)
        table[i, :held] = perm[at:at + held]
        at += held
    free = np.concatenate([perm[at:], np.zeros(n_pages - (n_pages - at), np.int64)])[:n_pages - at]
    offs, top = {}, 0

    def take(name, words):
        nonlocal top
        offs[name] = top
        top += -(-words // 16) * 16

    for name, words in dict(past=n, fresh=n, table=n * stride, free=len(free), cursor=1, kv=n, qs=n + 1, slots=rows + 2, pos=rows + 2, q=(rows + 2) * nh * dim,
                            k=(rows + 2) * width, v=(rows + 2) * width, y=(rows + 2) * nh * dim, logits=6 * vocab, scores=6, out=8, par=8, tok=8).items():
        take(name, words)
    act = np.zeros(top, np.float32)
    words = act.view(np.uint32)
    for name, x in dict(past=past, fresh=fresh, table=table.reshape(-1), free=free).items():
        words[offs[name]:offs[name] + len(x)] = x
    for name in ("q", "k", "v", "logits", "scores"):
        end = offs[name] + dict(q=(rows + 2) * nh * dim, k=(rows + 2) * width, v=(rows + 2) * width, logits=6 * vocab, scores=6)[name]
        act[offs[name]:end] = r.normal(0, 1, end - offs[name])
    pool = 512
    layer = b2.kv4_page_bytes(page, n_kv, dim) * n_pages
    kv0 = kv4.pack_pages(*(r.normal(0, 1, (page * n_pages, n_kv, dim)).astype(np.float32) for _ in range(2)), page, n_pages).reshape(-1)
    state0 = r.normal(0, 1, (2 * 6 * 4, 128)).astype(np.float32)
    o = offs
    cl = b2.cmd_list(
        b2.block_map_cmd(n, o["past"], o["fresh"], o["table"], stride, o["free"], len(free), o["cursor"], o["kv"], o["qs"], o["slots"], o["pos"], rows + 2, page),
        b2.kv4_store_cmd(rows + 2, o["k"], o["v"], o["slots"], geo, pool, n_pages),
        b2.kv4_attn_cmd(nh, o["q"], o["y"], o["table"], stride, o["qs"], o["kv"], n, rows + 2, 3, stride * page, 0.1, geo, pool, n_pages),
        b2.beam_select_cmd(2, 3, vocab, o["logits"], o["scores"], 3, o["out"], o["par"], o["tok"]),
        b2.beam_reorder_cmd(2, 3, o["par"], 0, 0, 4, 2),
    )
    with b2.Context(device=0, weight_bytes=1 << 20, act_floats=top, state_rows=len(state0), kv_bytes=pool + layer) as ctx:
        def reset():
            ctx.write(0, act)
            ctx.write_state(0, state0.reshape(-1))
            ctx.write_kv(pool, kv0)

        reset()
        assert ctx.run(cl) == 0, ctx.last_error()
        first, state1 = ctx.read(0, top), ctx.read_state(0, len(state0))
        reset()
        g = ctx.graph(cl)
        assert g.kernels == 1 + 1 + 2 + 2 + 1
        g.launch()
        ctx.synchronize()
        assert np.array_equal(ctx.read(0, top).view(np.uint32), first.view(np.uint32))
        g.close()
        # what the device finds wrong is reported, and the context goes on
        bad = act.copy()
        bad.view(np.uint32)[o["past"]] = 1000
        ctx.write(0, bad)
        with pytest.raises(b2.B200QError, match="0x8"):
            ctx.run(cl[:16])
        reset()
        assert ctx.run(cl) == 0

    dev = torch.from_numpy(act.copy()).cuda()
    dkv, dst = torch.from_numpy(kv0).cuda(), torch.from_numpy(state0.copy()).cuda()
    p = {name: dev.data_ptr() + 4 * v for name, v in offs.items()}
    h = b2.Kv4Pool(dkv.data_ptr(), n_pages, page, n_kv, dim, 1, 0)
    need = b2.kv4_attn_workspace(0, h, rows + 2, nh, n, 3, stride * page)
    need2 = b2.beam_select_workspace(0, 2, 3, vocab, 3)
    room = torch.empty(max(need, need2), dtype=torch.uint8, device="cuda")
    b2.block_map(0, n, p["past"], p["fresh"], p["table"], stride, page, p["free"], len(free), p["cursor"], p["cursor"], p["kv"], p["qs"], p["slots"], p["pos"],
                 rows + 2)
    b2.kv4_store(0, h, p["k"], p["v"], p["slots"], rows + 2)
    b2.kv4_attn(0, h, p["q"], p["y"], rows + 2, nh, p["table"], stride, p["qs"], p["kv"], n, 3, stride * page, 0.1, room.data_ptr(), need)
    b2.beam_select(0, p["logits"], vocab, p["scores"], 2, 3, 3, p["out"], p["par"], p["tok"], room.data_ptr(), need2)
    b2.beam_reorder(0, dst.data_ptr(), dst.data_ptr(), p["par"], 2, 3, 4 * 512, 2)
    torch.cuda.synchronize()
    assert np.array_equal(dev.cpu().numpy().view(np.uint32), first.view(np.uint32))
    assert np.array_equal(dst.cpu().numpy().reshape(-1), np.asarray(state1).reshape(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 48])
def test_hybrid_decoder_with_the_4bit_cache(orc, page):
    """Three tokens, each token its captured lists: every command but the new ones by the oracle, those by the restatement. The
    same greedy tokens; logits within 1e-4 of the largest (as with the F16 cache)."""
    m = D.HybridDecoder(SMALL, seed=9, kv4_page=page)
    ws = {}
    s, L = SMALL, m.L
    with b2.Context(device=0, **m.context_config()) as ctx:
        m.load(ctx, keep=ws)
        graphs = [ctx.graph(cl) for cl in m.token_lists()]
        toks = []
        for t in range(3):
            ctx.write(L.REC, m.record(s.prefill + t))
            ctx.launch_many(graphs, len(graphs))
            toks.append(int(ctx.read(L.TOK, 1).view(np.uint32)[0]))
        got = ctx.read(0, L.size)
        for g in graphs:
            g.close()
    act, state = m.initial_act(), m.initial_state()
    words = act.view(np.uint32)
    pools = []
    raw = m.initial_kv()
    for j in range(s.n_attn):
        at, n_pages = m.kv4_pool(j)
        p = ref.Pool(n_pages, page, s.n_kv_head, s.head_dim)
        p.bytes.reshape(-1)[:] = raw[at:at + p.bytes.size]
        pools.append(p)

    def step(cl):
        """Runs of old commands through the oracle, new ones here."""
        i, start, layer = 0, 0, [0]
        cmds = cl.reshape(-1, 8)

        def flush(end):
            if end > start:
                assert orc.run_list(act, cmds[start:end].reshape(-1).copy(), ws, state=state, kv=np.zeros(2, np.uint16), kv_ctx=s.kv_ctx) == 0

        while i < len(cmds):
            op = int(cmds[i, 0])
            if op == b2.OP_GDN:
                i += 3
                continue
            if op < 18:
                i += 1
                continue
            flush(i)
            if op == b2.OP_BLOCK_MAP:
                out = ref.block_map([int(words[L.POS])], [1], words[L.TABLE:L.TABLE + L.stride][None], page,
                                    list(words[L.FREE:L.FREE + L.stride].astype(int)), int(words[L.CURSOR]), 1)
                words[L.TABLE:L.TABLE + L.stride] = out[0][0]
                words[L.KVLEN], words[L.QSTART], words[L.QSTART + 1], words[L.SLOT], words[L.CURSOR] = out[1][0], 0, 1, out[3][0], out[5]
                i += 2
            elif op == b2.OP_KV4_STORE:
                w = s.n_kv_head * s.head_dim
                pools[layer[0]].store([int(words[L.SLOT])], act[L.KR:L.KR + w][None], act[L.V:L.V + w][None])
                i += 2
            else:
                assert op == b2.OP_KV4_ATTN
                y, _, _ = ref.attention(pools[layer[0]], act[L.QR:L.QR + s.n_head * s.head_dim].reshape(1, s.n_head, s.head_dim),
                                        words[L.TABLE:L.TABLE + L.stride][None].astype(np.int64), [0, 1], [int(words[L.KVLEN])], s.head_dim ** -0.5)
                act[L.YA:L.YA + y.size] = y.reshape(-1)
                layer[0] += 1
                i += 3
            start = i
        flush(len(cmds))

    want = []
    for t in range(3):
        act[L.REC:L.REC + D.RECORD] = m.record(s.prefill + t)
        assert len(m.token_lists()) == 1
        step(m.token_lists()[0])
        want.append(int(words[L.TOK]))
    assert toks == want
    lg, rl = got[L.LOGITS:L.LOGITS + s.vocab], act[L.LOGITS:L.LOGITS + s.vocab]
    assert np.abs(lg - rl).max() <= 1e-4 * np.abs(rl).max()
    assert int(got.view(np.uint32)[L.KVLEN]) == s.prefill + 3
