"""Cases, plain forms and exact forms of the operators that serve several sequences from a paged 4-bit KV cache.

Operators, each with the call of the b200q package that computes it:

  block_map   block tables, slot maps, row starts and positions of a step, from the requests' lengths
  kv4_store   K and V rows quantized to Q4_0 blocks in the cache pages (read back with kv4_load as the values they stand for)
  kv4_attn    attention of each request's new tokens over its pages of the 4-bit cache, causal, ragged
  beam_select the best continuations over a request's beams and the vocabulary
  reorder     states moved to their beams' parents: dense state rows (beam_reorder), block tables and tail pages (kv4_reorder)

`own` False: elementary torch operations in 32 bits (64 where scores of neighbouring candidates are compared).
`own` True: the package's calls on the same tensors.

The cache. A page holds `page` tokens (a multiple of 16) of every KV head; page p, head h, 16-token tile t is the run of
16 * D / 2 * 2 + 16 * D / 32 * 2 * 2 bytes number (p * n_kv + h) * (page / 16) + t of the pool:
  K codes   planes of 128 dims (the last one narrower), in a plane [token 16][word 4][block], word w of a 32-dim block
            holding in byte i element 4 w + i (low nibble) and 16 + 4 w + i (high nibble); a code c stands for d (c - 8)
  V codes   as K, in a plane [token / 8][token % 2][word 4][token / 2 % 4][block]
  K scales, V scales   FP16 d, [token 16][block]
"""
import math

import numpy as np
import torch

own = False

SKIP = -1  # a slot that names no token


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of a small server: one new token for each of 64 requests
        {"name": "map 64 decode", "op": "block_map", "req": 64, "new": 1, "past": 4096, "page": 16},
        # prompts admitted together: 512 requests of up to 512 new tokens, some with a cached prefix
        {"name": "map 512 prompts", "op": "block_map", "req": 512, "new": 512, "past": 1000, "page": 64},
        # the decoder's attention layer (4 KV heads of 256) writing one token for 8 sequences
        {"name": "store 8 tokens", "op": "kv4_store", "rows": 8, "n_kv": 4, "dim": 256, "page": 16, "gap": 0},
        # a prompt's K and V, read out of wider q|k|v rows
        {"name": "store 8192 tokens", "op": "kv4_store", "rows": 8192, "n_kv": 8, "dim": 128, "page": 64, "gap": 4096},
        # one token of the decoder behind its 512-token prompt: latency
        {"name": "attn 1 x 513", "op": "kv4_attn", "req": 1, "new": 1, "kv": 513, "kv_low": 513, "n_head": 16, "n_kv": 4,
         "dim": 256, "page": 16, "window": 0},
        # a serving batch with lengths from a few tokens to 8192, one to three new tokens each (drafts being checked)
        {"name": "attn 64 ragged", "op": "kv4_attn", "req": 64, "new": 3, "kv": 8192, "kv_low": 5, "n_head": 32, "n_kv": 8,
         "dim": 128, "page": 64, "window": 0},
        # one long sequence: the cache is all there is to read
        {"name": "attn 1 x 131000", "op": "kv4_attn", "req": 1, "new": 1, "kv": 131000, "kv_low": 131000, "n_head": 16,
         "n_kv": 4, "dim": 256, "page": 64, "window": 0},
        # prompts of 200 to 2048 tokens through the decoder's attention layer
        {"name": "attn prompts", "op": "kv4_attn", "req": 4, "new": 2048, "kv": 2560, "kv_low": 200, "n_head": 16, "n_kv": 4,
         "dim": 256, "page": 32, "window": 0},
        # four beams over a 32000-word vocabulary
        {"name": "select 4 x 32000", "op": "beam_select", "req": 1, "beams": 4, "vocab": 32000, "n_out": 8, "masked": 0},
        # sixteen requests of eight beams over the decoder's vocabulary, part of it masked by a grammar
        {"name": "select 128 x 151936", "op": "beam_select", "req": 16, "beams": 8, "vocab": 151936, "n_out": 16, "masked": 1},
        # block tables and tail pages of eight attention layers, two requests of four beams
        {"name": "reorder pages", "op": "kv4_reorder", "req": 2, "beams": 4, "live": 2, "kv": 1003, "layers": 8, "n_kv": 4,
         "dim": 256, "page": 16},
        # DeltaNet states (16 heads of 128 x 128) of six layers, four requests of eight beams
        {"name": "reorder states", "op": "beam_reorder", "req": 4, "beams": 8, "live": 3, "row": 16 * 128 * 128, "layers": 6},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["block_map", "kv4_store", "kv4_attn", "kv4_attn", "kv4_attn", "beam_select", "kv4_reorder", "beam_reorder"])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "block_map":
        return {"op": op, "req": _log(rng, 1, 512), "new": _log(rng, 1, 512), "past": _log(rng, 1, 4096), "page": page}
    n_kv, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 96, 128, 160, 192, 224, 256])
    if op == "kv4_store":
        return {"op": op, "rows": _log(rng, 1, 8192), "n_kv": n_kv, "dim": dim, "page": page, "gap": rng.choice([0, 1, 7, 64, 500])}
    if op == "kv4_attn":
        group = rng.choice([1, 2, 3, 4, 6, 8, 16])
        if rng.random() < 0.3:  # prompts
            new, req = _log(rng, 17, 1024), rng.randint(1, 4)
            kv = new + _log(rng, 1, 2048)
        else:                   # single tokens and drafts
            new, req = rng.choice([1, 1, 1, 2, 4, 7]), _log(rng, 1, 64)
            kv = new + _log(rng, 1, 100000 // req)
        group = min(group, 32 // n_kv)
        low = _log(rng, new, kv)
        return {"op": op, "req": req, "new": new, "kv": kv, "kv_low": low, "n_head": n_kv * group, "n_kv": n_kv, "dim": dim, "page": page,
                "window": rng.choice([0, 0, 0, _log(rng, 1, kv)])}
    if op == "beam_select":
        beams = rng.randint(1, 16)
        return {"op": op, "req": _log(rng, 1, 128 // beams), "beams": beams, "vocab": _log(rng, 100, 151936),
                "n_out": rng.choice([1, beams, 2 * beams]), "masked": rng.randint(0, 1)}
    beams = rng.randint(2, 12)
    if op == "kv4_reorder":
        return {"op": op, "req": rng.randint(1, 6), "beams": beams, "live": rng.randint(1, beams), "kv": _log(rng, 1, 4000),
                "layers": rng.randint(1, 8), "n_kv": n_kv, "dim": dim, "page": page}
    return {"op": op, "req": rng.randint(1, 4), "beams": beams, "live": rng.randint(1, beams), "row": 4 * _log(rng, 4, 60000),
            "layers": rng.randint(1, 6)}


# ---- shapes that follow from a case alone -------------------------------------------------------------------------

def _spaced(n, low, high):
    """n lengths from low to high, evenly spaced by their logarithm."""
    if n == 1:
        return [high]
    return [int(round(math.exp(math.log(low) + (math.log(high) - math.log(low)) * i / (n - 1)))) for i in range(n)]


def _map_lengths(case):
    past = [p - 1 for p in _spaced(case["req"], 1, case["past"] + 1)]
    new = [1 + (i * 37) % case["new"] for i in range(case["req"])]
    return past, new


def _attn_lengths(case):
    """(new tokens, cached tokens with the new ones) of each request."""
    kv = _spaced(case["req"], case["kv_low"], case["kv"])
    if case["new"] > 16:
        return [min(k, case["new"]) for k in kv], kv
    return [min(k, 1 + i % case["new"]) if case["req"] > 1 else min(k, case["new"]) for i, k in enumerate(kv)], kv


def _seen(case):
    """Keys that each request's rows see in all, and the keys of each request that any row sees."""
    pairs, keys = 0, 0
    new, kv = _attn_lengths(case)
    w = case["window"] or 1 << 40
    for t, n in zip(new, kv):
        pairs += sum(min(w, n - t + i + 1) for i in range(t))
        keys += min(n, t - 1 + w)
    return pairs, keys


def _tile_bytes(dim):
    return 16 * dim + 16 * (dim // 32) * 4


def work(case):
    op = case["op"]
    if op == "block_map":
        past, new = _map_lengths(case)
        fresh = sum(-(-(p + n) // case["page"]) - -(-p // case["page"]) for p, n in zip(past, new))
        return {"bytes": 8 * case["req"] + 8 * fresh + 8 * case["req"] + 8 * sum(new), "flops": 0}
    if op == "kv4_store":
        values = 2 * case["rows"] * case["n_kv"] * case["dim"]
        return {"bytes": values * 4 + values * 9 // 16 + 4 * case["rows"] + values * 4, "flops": 4 * values}
    if op == "kv4_attn":
        pairs, keys = _seen(case)
        rows = sum(_attn_lengths(case)[0])
        return {"bytes": keys * case["n_kv"] * case["dim"] * 9 // 8 + 8 * rows * case["n_head"] * case["dim"],
                "flops": 4 * pairs * case["n_head"] * case["dim"]}
    if op == "beam_select":
        n = case["req"] * case["beams"]
        return {"bytes": 4 * n * case["vocab"] + 4 * n + 12 * case["req"] * case["n_out"], "flops": 3 * n * case["vocab"]}
    n = case["req"] * (case["live"] + case["beams"])
    if op == "beam_reorder":
        return {"bytes": 4 * n * case["layers"] * case["row"], "flops": 0}
    full, tail = divmod(case["kv"], case["page"])
    return {"bytes": n * (4 * full + case["layers"] * case["n_kv"] * -(-tail // 16) * _tile_bytes(case["dim"])) or 4 * n, "flops": 0}


# ---- the cache layout ---------------------------------------------------------------------------------------------

def _planes(dim):
    return [(p, min(4, dim // 32 - 4 * p)) for p in range(-(-dim // 128))]


def _codes_to_tiles(x):
    """Codes [..., 16 tokens, dim] (uint8, 0..15) as a tile's K codes and V codes, each [..., 8 dim] bytes."""
    lead, dim = x.shape[:-2], x.shape[-1]
    b = x.reshape(*lead, 16, dim // 32, 2, 4, 4)            # token, block, nibble, word, byte
    b = b[..., 0, :, :] | (b[..., 1, :, :] << 4)            # token, block, word, byte
    k, v = [], []
    for p, nb in _planes(dim):
        w = b[..., 4 * p:4 * p + nb, :, :].transpose(-3, -2)  # token, word, block, byte
        k.append(w.reshape(*lead, -1))
        w = w.reshape(*lead, 2, 4, 2, 4, nb * 4)            # token / 8, token / 2 % 4, token % 2, word, block bytes
        v.append(w.permute(*range(len(lead)), -5, -3, -2, -4, -1).reshape(*lead, -1))
    return torch.cat(k, -1), torch.cat(v, -1)


def _tiles_to_codes(k, v, dim):
    """The inverse: codes [..., 16, dim] of the K codes and of the V codes."""
    lead, kk, vv, at = k.shape[:-1], [], [], 0
    for p, nb in _planes(dim):
        n = 16 * 16 * nb
        kk.append(k[..., at:at + n].reshape(*lead, 16, 4, nb, 4))
        w = v[..., at:at + n].reshape(*lead, 2, 2, 4, 4, nb * 4)
        vv.append(w.permute(*range(len(lead)), -5, -2, -4, -3, -1).reshape(*lead, 16, 4, nb, 4))
        at += n
    both = []
    for planes in (kk, vv):
        b = torch.cat([x.transpose(-3, -2) for x in planes], -3)       # token, block, word, byte
        both.append(torch.stack([b & 15, b >> 4], -3).reshape(*lead, 16, dim))
    return both


def _quantize(x):
    """Q4_0 of [..., dim] FP32: (codes uint8 [..., dim], scales FP16 [..., dim / 32]), in the format's own FP32 steps."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = b.abs()
    amax = a.amax(-1, keepdim=True)
    first = torch.where(a == amax, torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = b.gather(-1, first.clamp(max=31)) / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    codes = (b * inv + 8.5).clamp(0, 15).to(torch.uint8)
    return codes.reshape(x.shape), d[..., 0].half()


def _dequantize(codes, scales):
    b = codes.reshape(*codes.shape[:-1], -1, 32).to(torch.float32) - 8.0
    return (b * scales.float()[..., None]).reshape(codes.shape)


def _make_tiles(gen, tiles, dim, k_std):
    """[tiles, tile bytes] of quantized normal K and V."""
    out = torch.empty(tiles, _tile_bytes(dim), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (16 * dim))
    for a in range(0, tiles, step):
        n = min(step, tiles - a)
        kc, ks = _quantize(torch.randn(n, 16, dim, generator=gen, device="cuda") * k_std)
        vc, vs = _quantize(torch.randn(n, 16, dim, generator=gen, device="cuda"))
        out[a:a + n, :8 * dim] = _codes_to_tiles(kc)[0]
        out[a:a + n, 8 * dim:16 * dim] = _codes_to_tiles(vc)[1]
        out[a:a + n, 16 * dim:] = torch.stack([ks, vs], 1).reshape(n, -1).view(torch.uint8)
    return out


def _read_tiles(tiles, dim):
    """K and V values [..., 16, dim] of tiles [..., tile bytes]."""
    kc, vc = _tiles_to_codes(tiles[..., :8 * dim], tiles[..., 8 * dim:16 * dim], dim)
    s = tiles[..., 16 * dim:].contiguous().view(torch.float16).reshape(*tiles.shape[:-1], 2, 16, dim // 32)
    return _dequantize(kc, s[..., 0, :, :]), _dequantize(vc, s[..., 1, :, :])


# ---- inputs -------------------------------------------------------------------------------------------------------

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    order = np.random.RandomState(seed % (1 << 31))
    if op == "block_map":
        past, new = _map_lengths(case)
        pick = order.permutation(case["req"])
        past, new = [past[i] for i in pick], [new[i] for i in pick]
        page = case["page"]
        stride = max(-(-(p + n) // page) for p, n in zip(past, new))
        held = [-(-p // page) for p in past]
        free = sum(-(-(p + n) // page) for p, n in zip(past, new)) - sum(held)
        pages = torch.randperm(sum(held) + free + 5, generator=gen, device="cuda").to(torch.int32)
        table = torch.zeros(case["req"], stride, dtype=torch.int32, device="cuda")
        mask = torch.arange(stride, device="cuda")[None] < _ints(held)[:, None]
        table[mask] = pages[:sum(held)]
        rows = -(-sum(new) // 64) * 64  # the step's buffers are padded
        s.update(past=_ints(past), new=_ints(new), table=table, stride=stride, free=pages[sum(held):].contiguous(), rows=rows,
                 n_pages=pages.numel(), at=_ints([2]), at_out=_ints([0]), kv_len=_ints([0] * case["req"]), q_start=_ints([0] * (case["req"] + 1)),
                 slots=_ints([0] * rows), positions=_ints([0] * rows))
        return s
    if op == "beam_select":
        n = case["req"] * case["beams"]
        x = torch.randn(n, case["vocab"], generator=gen, device="cuda") * 2.5
        if case["masked"]:
            x[torch.rand(n, case["vocab"], generator=gen, device="cuda") < 0.4] = -math.inf
        scores = -20.0 * torch.rand(n, generator=gen, device="cuda")
        k = case["req"] * case["n_out"]
        s.update(logits=x, scores=scores, out=torch.empty(k, device="cuda"), parent=_ints([0] * k), token=_ints([0] * k))
        return s
    if op in ("beam_reorder", "kv4_reorder"):
        parent = []
        for _ in range(case["req"]):
            live = sorted(order.choice(case["beams"], case["live"], replace=False))
            parent += sorted(live + [live[i] for i in order.randint(0, case["live"], case["beams"] - case["live"])])
        s["parent"] = _ints([int(p) for p in parent])
    if op == "beam_reorder":
        s["src"] = torch.randn(case["layers"], case["req"] * case["beams"], case["row"], generator=gen, device="cuda")
        s["dst"] = torch.zeros_like(s["src"])
        return s
    page, n_kv, dim = case["page"], case["n_kv"], case["dim"]
    if op == "kv4_reorder":
        n, full = case["req"] * case["beams"], case["kv"] // page
        n_pages = n * (full + 1)
        s["table"] = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32).reshape(n, full + 1)
        s["kv_len"] = _ints([case["kv"]] * n)
        s["pool"] = _make_tiles(gen, case["layers"] * n_pages * n_kv * (page // 16), dim, 1.0)
        s["n_pages"] = n_pages
        return s
    if op == "kv4_store":
        n_pages = -(-case["rows"] // page) + 3
        width = n_kv * dim
        both = torch.randn(case["rows"], 2 * width + case["gap"], generator=gen, device="cuda")
        s["k"], s["v"] = both[:, case["gap"]:case["gap"] + width], both[:, case["gap"] + width:]
        s["slots"] = torch.randperm(n_pages * page, generator=gen, device="cuda")[:case["rows"]].to(torch.int32)
        s["pool"] = _make_tiles(gen, n_pages * n_kv * (page // 16), dim, 1.0)
        s["k_back"], s["v_back"] = (torch.empty(case["rows"], width, device="cuda") for _ in range(2))
        s["n_pages"] = n_pages
        return s
    new, kv = _attn_lengths(case)
    pick = order.permutation(case["req"])
    new, kv = [new[i] for i in pick], [kv[i] for i in pick]
    held = [-(-n // page) for n in kv]
    stride, n_pages = max(held), sum(held) + 2
    pages = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(case["req"], stride, dtype=torch.int32, device="cuda")
    table[torch.arange(stride, device="cuda")[None] < _ints(held)[:, None]] = pages[:sum(held)]
    rows = sum(new)
    # keys of which a row's scores spread by about two
    s.update(q=torch.randn(rows, case["n_head"], dim, generator=gen, device="cuda") * 2.0, table=table, stride=stride, rows=rows, max_q=max(new),
             max_kv=max(kv), q_start=_ints([0] + list(np.cumsum(new))), kv_len=_ints(kv), n_pages=n_pages, scale=1.0 / math.sqrt(dim),
             pool=_make_tiles(gen, n_pages * n_kv * (page // 16), dim, 1.0), y=torch.empty(rows, case["n_head"], dim, device="cuda"))
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------

def _plain_map(s):
    page = s["page"]
    past, new = s["past"].long(), s["new"].long()
    kv_len = past + new
    q_start = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    first, last = (past + page - 1) // page, (kv_len + page - 1) // page
    need = last - first
    at = s["at"].long()
    base = at + need.cumsum(0) - need
    b = torch.arange(s["stride"], device="cuda")[None]
    fresh = (b >= first[:, None]) & (b < last[:, None])
    table = torch.where(fresh, s["free"][(base[:, None] + b - first[:, None]).clamp(0, s["free"].numel() - 1)], s["table"])
    j = torch.arange(s["rows"], device="cuda")
    r = (torch.searchsorted(q_start, j, right=True) - 1).clamp(max=s["req"] - 1)
    real = j < q_start[-1]
    pos = torch.where(real, past[r] + j - q_start[r], 0)
    slots = torch.where(real, table[r, pos // page].long() * page + pos % page, SKIP)
    return [x.to(torch.int32) for x in (table, kv_len, q_start, slots, pos, at + need.sum())]


def _tile_view(s):
    return s["pool"].view(-1, s["n_kv"], s["page"] // 16, _tile_bytes(s["dim"]))


def _plain_store(s):
    page, dim, n_kv = s["page"], s["dim"], s["n_kv"]
    slot = s["slots"].long()
    tiles = _tile_view(s)
    p, t, i = slot // page, slot % page // 16, slot % 16
    # where the bytes of token i lie in its tile: those of a tile whose codes are their tokens' numbers
    owner = torch.arange(16, device="cuda", dtype=torch.uint8)[:, None].expand(16, dim)
    k_at, v_at = ((x & 15).argsort(stable=True).reshape(16, dim // 2) for x in _codes_to_tiles(owner))
    v_at = v_at + 8 * dim
    s_at = 16 * dim + torch.arange(16 * (dim // 32) * 2, device="cuda").reshape(16, -1)
    back = []
    for x, at, scale_at, which in ((s["k"], k_at, s_at, 0), (s["v"], v_at, s_at + 32 * (dim // 32), 1)):
        codes, d = _quantize(x.reshape(-1, n_kv, dim))
        one = codes[:, :, None].expand(-1, -1, 16, -1)  # the token's bytes, as any of a tile's tokens holds them
        laid = _codes_to_tiles(one)[which].gather(-1, (at[i] - 8 * dim * which)[:, None].expand(-1, n_kv, -1))
        place = (p[:, None], torch.arange(n_kv, device="cuda")[None], t[:, None])
        tiles[(*(q[..., None] for q in place), at[i][:, None])] = laid
        tiles[(*(q[..., None] for q in place), scale_at[i][:, None])] = d.view(torch.uint8).reshape(len(slot), n_kv, -1)
    for x in _read_tiles(tiles[p, :, t], dim):
        back.append(x[torch.arange(len(slot), device="cuda"), :, i].reshape(len(slot), -1))
    return back


def _plain_attn(s):
    page, dim, n_kv, n_head = s["page"], s["dim"], s["n_kv"], s["n_head"]
    group, req = n_head // n_kv, s["req"]
    tiles = _tile_view(s)[s["table"].long()]                                   # req, block, head, tile, bytes
    k, v = (x.transpose(1, 2).reshape(req, n_kv, -1, dim) for x in _read_tiles(tiles, dim))
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    new = start[1:] - start[:-1]
    at = (start[:-1, None] + torch.arange(s["max_q"], device="cuda")).clamp(max=s["rows"] - 1)
    q = s["q"][at].reshape(req, -1, n_kv, group, dim).permute(0, 2, 1, 3, 4).reshape(req, n_kv, -1, dim)
    x = q @ k.transpose(-1, -2) * s["scale"]
    pos = kv_len[:, None] - new[:, None] + torch.arange(s["max_q"], device="cuda")   # req, new token
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= pos[..., None]
    if s["window"]:
        seen &= key > pos[..., None] - s["window"]
    seen = seen[:, None, :, None].expand(req, 1, -1, group, -1).reshape(req, 1, -1, k.shape[2])
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top.isinf(), 0.0, top))
    total = x.sum(-1, keepdim=True)
    y = (x @ v) / torch.where(total == 0, 1.0, total)
    y = y.reshape(req, n_kv, -1, group, dim).permute(0, 2, 1, 3, 4).reshape(req, -1, n_head, dim)
    j = torch.arange(s["rows"], device="cuda")
    r = torch.searchsorted(start, j, right=True) - 1
    return y[r, j - start[r]]


def _plain_select(s):
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    x = (x - lse + s["scores"].double()[:, None]).reshape(s["req"], -1)
    best, at = torch.sort(x, dim=-1, descending=True, stable=True)
    best, at = best[:, :s["n_out"]], at[:, :s["n_out"]]
    return best.float().reshape(-1), (at // s["vocab"]).to(torch.int32).reshape(-1), (at % s["vocab"]).to(torch.int32).reshape(-1)


def _rows_of(s):
    n = s["req"] * s["beams"]
    return torch.arange(n, device="cuda") // s["beams"] * s["beams"] + s["parent"].long()


def _plain_reorder(s):
    s["dst"].copy_(s["src"][:, _rows_of(s)])
    return s["dst"]


def _plain_pages(s):
    at = _rows_of(s)
    full, tail = divmod(s["kv"], s["page"])
    own_tail, from_tail = s["table"][:, -1].long(), s["table"][at, -1].long()
    s["table"][:, :full] = s["table"][at, :full]
    if tail:
        tiles = s["pool"].view(s["layers"], s["n_pages"], s["n_kv"], s["page"] // 16, -1)
        n = -(-tail // 16)
        tiles[:, own_tail, :, :n] = tiles[:, from_tail, :, :n]
    return s["table"], s["pool"]


# ---- the package's calls ------------------------------------------------------------------------------------------

_b200q = None


def _package():
    """The package, whose folder has dashes in its name."""
    global _b200q
    if _b200q is None:
        import importlib.util
        import os
        import sys
        name = "fpga_llama_gguf_b200"
        if name not in sys.modules:
            folder = os.path.join(os.getcwd(), "fpga-llama-gguf_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _b200q = sys.modules[name]
    return _b200q


def _pool(b2, s, layers=1):
    pool = s["pool"]
    return b2.Kv4Pool(pool.data_ptr(), s["n_pages"], s["page"], s["n_kv"], s["dim"], layers, pool.numel() // layers)


def _own(s):
    b2, op = _package(), s["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "block_map":
        b2.block_map(0, s["req"], s["past"].data_ptr(), s["new"].data_ptr(), s["table"].data_ptr(), s["stride"], s["page"],
                     s["free"].data_ptr(), s["free"].numel(), s["at"].data_ptr(), s["at_out"].data_ptr(), s["kv_len"].data_ptr(),
                     s["q_start"].data_ptr(), s["slots"].data_ptr(), s["positions"].data_ptr(), s["rows"], stream=stream)
        return s["table"], s["kv_len"], s["q_start"], s["slots"], s["positions"], s["at_out"]
    if op == "kv4_store":
        pool, k, v = _pool(b2, s), s["k"], s["v"]
        b2.kv4_store(0, pool, k.data_ptr(), v.data_ptr(), s["slots"].data_ptr(), s["rows"], k.stride(0), v.stride(0), stream=stream)
        b2.kv4_load(0, pool, s["slots"].data_ptr(), s["rows"], s["k_back"].data_ptr(), s["v_back"].data_ptr(), stream=stream)
        return s["k_back"], s["v_back"]
    if op == "kv4_attn":
        pool = _pool(b2, s)
        need = b2.kv4_attn_workspace(0, pool, s["rows"], s["n_head"], s["req"], s["max_q"], s["max_kv"])
        room = torch.empty(need, dtype=torch.uint8, device="cuda")
        b2.kv4_attn(0, pool, s["q"].data_ptr(), s["y"].data_ptr(), s["rows"], s["n_head"], s["table"].data_ptr(), s["stride"],
                    s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["req"], s["max_q"], s["max_kv"], s["scale"], room.data_ptr(), need,
                    window=s["window"], stream=stream)
        return s["y"]
    if op == "beam_select":
        need = b2.beam_select_workspace(0, s["req"], s["beams"], s["vocab"], s["n_out"])
        room = torch.empty(need, dtype=torch.uint8, device="cuda")
        b2.beam_select(0, s["logits"].data_ptr(), s["vocab"], s["scores"].data_ptr(), s["req"], s["beams"], s["n_out"], s["out"].data_ptr(),
                       s["parent"].data_ptr(), s["token"].data_ptr(), room.data_ptr(), need, stream=stream)
        return s["out"], s["parent"], s["token"]
    if op == "beam_reorder":
        b2.beam_reorder(0, s["src"].data_ptr(), s["dst"].data_ptr(), s["parent"].data_ptr(), s["req"], s["beams"], 4 * s["row"], s["layers"],
                        stream=stream)
        return s["dst"]
    b2.kv4_reorder(0, _pool(b2, s, s["layers"]), s["table"].data_ptr(), s["table"].shape[1], s["kv_len"].data_ptr(), s["parent"].data_ptr(),
                   s["req"], s["beams"], stream=stream)
    return s["table"], s["pool"]


def run(state):
    if own:
        return _own(state)
    return {"block_map": _plain_map, "kv4_store": _plain_store, "kv4_attn": _plain_attn, "beam_select": _plain_select,
            "beam_reorder": _plain_reorder, "kv4_reorder": _plain_pages}[state["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _value_at(pool, which, first, token, dim):
    """Values [tokens, dim] in 64 bits of K (which 0) or V (1): each element found by its own address. first: the tile's first
    byte, token: the token's number in the tile (both [tokens])."""
    e = torch.arange(dim, device="cuda")
    block, j = e // 32, e % 32
    plane, nb = block // 4, torch.clamp(dim // 32 - block // 4 * 4, max=4)
    word, byte = j % 16 // 4, j % 4
    t = token[:, None]
    row = t * 4 + word if which == 0 else ((t // 8 * 2 + t % 2) * 4 + word) * 4 + t // 2 % 4
    at = first[:, None] + which * 8 * dim + plane * 1024 + (row * nb + block % 4) * 4 + byte
    code = (pool[at] >> (j // 16 * 4).to(torch.uint8)) & 15
    d_at = first[:, None] + 16 * dim + which * 32 * (dim // 32) + (t * (dim // 32) + torch.arange(dim // 32, device="cuda")) * 2
    d = (pool[d_at].int() | (pool[d_at + 1].int() << 8)).to(torch.int16).view(torch.float16).double()
    return (code.double() - 8) * d[:, block]


def _exact_attn(s):
    page, dim, n_kv = s["page"], s["dim"], s["n_kv"]
    group, pool, size = s["n_head"] // n_kv, s["pool"].reshape(-1), _tile_bytes(s["dim"])
    start, kv_len = s["q_start"].tolist(), s["kv_len"].tolist()
    y = torch.zeros(s["rows"], s["n_head"], dim, dtype=torch.float64, device="cuda")
    for r in range(s["req"]):
        a, b, n = start[r], start[r + 1], kv_len[r]
        key = torch.arange(n, device="cuda")
        pages = s["table"][r].long()[key // page]
        for h in range(n_kv):
            first = ((pages * n_kv + h) * (page // 16) + key % page // 16) * size
            k, v = (_value_at(pool, i, first, key % 16, dim) for i in (0, 1))
            for c in range(a, b, 256):
                e = min(b, c + 256)
                q = s["q"][c:e, h * group:(h + 1) * group].double()
                x = torch.einsum("tgd,kd->tgk", q, k) * s["scale"]
                pos = n - (b - a) + torch.arange(c - a, e - a, device="cuda")
                hide = key[None] > pos[:, None]
                if s["window"]:
                    hide |= key[None] <= pos[:, None] - s["window"]
                p = torch.softmax(x.masked_fill(hide[:, None], -math.inf), -1)
                y[c:e, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", p, v)
    return y


def exact(case, seed):
    op = case["op"]
    if op in ("block_map", "kv4_reorder"):
        return None  # whole numbers and moved bytes
    s = prepare(case, seed)
    if op == "beam_reorder":
        return torch.stack([s["src"][:, i // case["beams"] * case["beams"] + p].double() for i, p in enumerate(s["parent"].tolist())], 1)
    if op == "kv4_attn":
        return _exact_attn(s)
    if op == "kv4_store":
        # the format states its own FP32 steps: the signed extreme over -8, its reciprocal, a product, + 8.5, cut off
        back = []
        for x in (s["k"], s["v"]):
            b = np.ascontiguousarray(x.cpu().numpy()).reshape(-1, 32)
            d = (b[np.arange(len(b)), np.abs(b).argmax(1)] / np.float32(-8)).astype(np.float32)[:, None]
            code = np.minimum((b * (np.float32(1) / d) + np.float32(8.5)).astype(np.int32), 15)
            back.append(((code - 8).astype(np.float64) * d.astype(np.float16).astype(np.float64)).reshape(x.shape))
        return back
    x = s["logits"].reshape(case["req"], case["beams"], -1)
    best = []
    for r in range(case["req"]):
        z = torch.log_softmax(x[r].double(), -1) + s["scores"].reshape(case["req"], -1)[r].double()[:, None]
        best.append(torch.topk(z.reshape(-1), case["n_out"]).values)
    return torch.cat(best), None, None
