"""The operators of the 4-bit paged KV cache, as a serving step meets them: block tables and slot maps made from request
lengths, rows quantised into the pool, rows read back, decode attention over the pool, and blocks given back.

Pool format, for each group of 32 head dims of one token's K or V row of one kv head (G = head_dim / 32 groups):
    s = f16((max - min) / 15),  m = f16(min + 8 s),  c = clamp(rne((x - m) / s) + 8, 0, 15)  (c = 8 where s = 0)
and the element reads back as s (c - 8) + m.  A (block, layer, kv head) chunk of 20 * head_dim bytes holds 16 tokens:
    K codes  [16 tokens][4 lanes][G] words, word (i, g): dims 32 g + 8 i + j, j = 0..7 from its low nibble up
    K params [16 tokens][G] words, m in the low half and s in the high half
    V codes  [head_dim / 64 planes][16 tokens][16 / G][G] 16-bit units; unit r = plane * 16 / G + r', group g: dims
             32 g + 4 r + j, j = 0..3 from its low nibble up
    V params as K's.
"""
import importlib
import math
import random

import torch

own = False

F = {"f16": torch.float16, "bf16": torch.bfloat16}


# ----------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of the 64-sequence microbenchmark batch: every sequence gets one row
        {"name": "map decode 64", "op": "map", "n": 64, "lo": 128, "hi": 1023, "new": 1, "room": 1.0, "pad": 0, "lens": 1},
        # admission of 512 ragged prompts over cached prefixes, with padded rows behind the last one and a pool
        # that runs out for the last sequences
        {"name": "map prefill 512", "op": "map", "n": 512, "lo": 1, "hi": 1024, "new": 2047, "room": 0.97, "pad": 1000, "lens": 2},
        # a few of 128 sequences end in this step
        {"name": "release decode 128", "op": "release", "n": 128, "lo": 256, "hi": 1011, "share": 0.1, "lens": 3},
        # a batch job ends: half of 4096 sequences go
        {"name": "release batch 4096", "op": "release", "n": 4096, "lo": 1, "hi": 2048, "share": 0.5, "lens": 4},
        # the decode step's 64 new rows (12 heads of 64), written and read back as later steps see them
        {"name": "append decode f16", "op": "append", "rows": 64, "heads": 12, "dim": 64, "dtype": "f16", "pad": 0},
        # a prefill chunk of 8 kv heads of 128 with padded rows, written and read back
        {"name": "append prefill bf16", "op": "append", "rows": 16384, "heads": 8, "dim": 128, "dtype": "bf16", "pad": 77},
        # a short cached prefix of a 25-head model read back to 16 bits for a prefill over it
        {"name": "gather prefix f16", "op": "gather", "rows": 1011, "heads": 25, "dim": 64, "dtype": "f16", "pad": 0},
        # long cached prefixes of several requests read back
        {"name": "gather prefixes bf16", "op": "gather", "rows": 65531, "heads": 8, "dim": 128, "dtype": "bf16", "pad": 5},
        # one user, a short context, 16 heads with a distance bias: latency
        {"name": "attn one alibi f16", "op": "attn", "batch": 1, "heads": 16, "kv": 16, "dim": 64, "dtype": "f16", "lo": 100, "hi": 130, "window": 0, "cap": 0.0, "alibi": True, "lens": 5},
        # the microbenchmark batch: 64 sequences, 12 heads of 64, contexts 128 to 1024
        {"name": "attn microbench f16", "op": "attn", "batch": 64, "heads": 12, "kv": 12, "dim": 64, "dtype": "f16", "lo": 128, "hi": 1024, "window": 0, "cap": 0.0, "alibi": False, "lens": 6},
        # grouped queries with a sliding window and capped scores over mixed contexts
        {"name": "attn window cap bf16", "op": "attn", "batch": 61, "heads": 32, "kv": 8, "dim": 128, "dtype": "bf16", "lo": 512, "hi": 16384, "window": 4096, "cap": 30.0, "alibi": False, "lens": 7},
        # grouped queries over long mixed contexts
        {"name": "attn long gqa bf16", "op": "attn", "batch": 32, "heads": 32, "kv": 8, "dim": 128, "dtype": "bf16", "lo": 512, "hi": 32768, "window": 0, "cap": 0.0, "alibi": False, "lens": 8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["map", "release", "append", "gather", "attn", "attn", "attn"])
    if op == "map":
        return {"op": op, "n": _log_int(rng, 1, 512), "lo": 1, "hi": _log_int(rng, 2, 1024), "new": _log_int(rng, 1, 2047),
                "room": rng.choice([1.0, 1.0, 0.9]), "pad": rng.choice([0, 0, 13]), "lens": rng.randrange(1 << 30)}
    if op == "release":
        return {"op": op, "n": _log_int(rng, 1, 4096), "lo": 1, "hi": _log_int(rng, 2, 2048), "share": rng.choice([0.05, 0.5, 1.0]), "lens": rng.randrange(1 << 30)}
    if op in ("append", "gather"):
        heads, dim = rng.choice([(12, 64), (25, 64), (16, 64), (8, 128), (1, 64), (3, 128), (7, 64)])
        most = 16384 if op == "append" else 65531
        return {"op": op, "rows": _log_int(rng, 1, most * 1024 // (max(heads * dim, 1024))), "heads": heads, "dim": dim,
                "dtype": rng.choice(["f16", "bf16"]), "pad": rng.choice([0, 0, 3])}
    dim, kv, group = rng.choice([64, 128]), rng.choice([1, 2, 4, 8, 12, 25]), rng.choice([1, 1, 2, 3, 4, 8])
    hi = _log_int(rng, 2, 32768)
    batch = _log_int(rng, 1, max(1, min(256, 8 * 32 * 32768 // (hi * max(kv * dim // 128, 1) * 2))))
    return {"op": op, "batch": batch, "heads": kv * group, "kv": kv, "dim": dim, "dtype": rng.choice(["f16", "bf16"]), "lo": max(1, hi // 64), "hi": hi,
            "window": rng.choice([0, 0, _log_int(rng, 1, 4096)]), "cap": rng.choice([0.0, 0.0, 30.0]), "alibi": rng.choice([False, False, True]), "lens": rng.randrange(1 << 30)}


def _lens(case, key, n, lo, hi):
    """n lengths, log-uniform over [lo, hi]: part of the case, the same for every seed."""
    r = random.Random("%s %d" % (key, case["lens"]))
    return [min(hi, max(lo, _log_int(r, lo, hi))) for _ in range(n)]


def _blocks(tokens):
    return (tokens + 15) // 16


def _map_lens(case):
    pre = _lens(case, "pre", case["n"], case["lo"], case["hi"])
    r = random.Random("cold %d" % case["lens"])
    pre = [0 if case["new"] > 1 and r.random() < 0.25 else p for p in pre]  # prompts with nothing cached
    new = _lens(case, "new", case["n"], 1, case["new"]) if case["new"] > 1 else [1] * case["n"]
    return pre, new


def _released(case):
    r = random.Random("gone %d" % case["lens"])
    return [int(r.random() < case["share"]) for _ in range(case["n"])]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------- the format, in elementary operations

def _quantise(x):
    """x [..., dim] in 16 bits -> codes [..., G, 32] uint8, s and m [..., G] f16."""
    v = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32))
    low, high = v.amin(-1), v.amax(-1)
    s = ((high - low) / 15.0).half()
    m = (low + 8.0 * s.float()).half()
    step = s.float().unsqueeze(-1)
    c = torch.round((v - m.float().unsqueeze(-1)) / torch.where(step == 0, torch.ones_like(step), step)) + 8.0
    c = torch.where(step == 0, torch.full_like(c, 8.0), c.clamp(0.0, 15.0))
    return c.to(torch.uint8), s, m


def _regions(pool, dim):
    """K codes [.., 16, dim/2], K params [.., 16, 4 G], V codes [.., planes, 16, 32], V params: views of the pool's chunks."""
    a, b = 8 * dim, 2 * dim
    return (pool[..., :a].unflatten(-1, (16, dim // 2)), pool[..., a:a + b].unflatten(-1, (16, dim // 8)),
            pool[..., a + b:2 * a + b].unflatten(-1, (dim // 64, 16, 32)), pool[..., 2 * a + b:].unflatten(-1, (16, dim // 8)))


def _params(s, m):
    return torch.stack([m, s], -1).contiguous().view(torch.uint8).flatten(-2)  # [..., 4 G] bytes


def _k_bytes(c):
    """codes [..., G, 32] -> [..., dim / 2] bytes in the pool's K order."""
    c = c.unflatten(-1, (4, 4, 2)).movedim(-4, -3)  # [..., i, G, byte, nibble]
    return (c[..., 0] | (c[..., 1] << 4)).flatten(-3)


def _v_bytes(c):
    """codes [..., G, 32] -> [..., planes, 32] bytes in the pool's V order."""
    g = c.shape[-2]
    c = c.unflatten(-1, (8, 2, 2)).movedim(-4, -3)  # [..., r, G, byte, nibble]
    return (c[..., 0] | (c[..., 1] << 4)).unflatten(-3, (g // 2, 16 // g)).flatten(-3)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1)


def _values(codes, params):
    """codes [..., G, 32] uint8, params [..., 4 G] bytes -> [..., dim] in 32 bits."""
    p = params.contiguous().view(torch.float16).unflatten(-1, (-1, 2)).float()
    return ((codes.float() - 8.0) * p[..., 1:] + p[..., :1]).flatten(-2)


def _k_values(b, params):
    g = b.shape[-1] // 16
    return _values(_nibbles(b.unflatten(-1, (4, g, 4))).flatten(-2).movedim(-3, -2).flatten(-2), params)


def _v_values(b, params):
    g = b.shape[-2] * 2
    c = _nibbles(b.unflatten(-1, (16 // g, g, 2))).flatten(-2)  # [..., plane, r', G, 4]
    return _values(c.flatten(-4, -3).movedim(-3, -2).flatten(-2), params)


def _fill(pool, gen, dim, k_spread):
    """Every block of the pool holds rows that were quantised from normal values, K's channels of different sizes."""
    kc, kp, vc, vp = _regions(pool, dim)
    shape = (*pool.shape[:3], 16, dim)
    c, s, m = _quantise((torch.randn(shape, device="cuda", generator=gen) * k_spread).half())
    kc.copy_(_k_bytes(c))
    kp.copy_(_params(s, m))
    c, s, m = _quantise(torch.randn(shape, device="cuda", generator=gen).half())
    vc.copy_(_v_bytes(c).movedim(-3, -2))
    vp.copy_(_params(s, m))


# ----------------------------------------------------------------- what a program has in hand

def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "map":
        pre, new = _map_lens(case)
        have = [_blocks(p) for p in pre]
        need = sum(_blocks(p + q) - h for p, q, h in zip(pre, new, have))
        width = max(_blocks(p + q) for p, q in zip(pre, new)) + 1
        blocks = sum(have) + need + 8
        ids = torch.randperm(blocks, generator=g, device="cuda").int()
        tables = torch.full((case["n"], width), -1, dtype=torch.int32, device="cuda")
        at = torch.arange(width, device="cuda")[None, :] < _ints(have)[:, None]
        tables[at] = ids[:sum(have)]
        free = ids[sum(have):].contiguous()
        rows = sum(new) + case["pad"]
        room = int(need * case["room"]) if case["room"] < 1 else need
        return {"op": op, "pre": _ints(pre), "new": None if case["new"] == 1 else _ints(new), "tables": tables, "free": free, "count": _ints([room]), "blocks": blocks,
                "count_out": _ints([0]), "start": _ints([0] * case["n"]), "post": _ints([0] * case["n"]), "slots": torch.zeros(rows, dtype=torch.int32, device="cuda")}
    if op == "release":
        lens = _lens(case, "pre", case["n"], case["lo"], case["hi"])
        have = [_blocks(p) for p in lens]
        width, blocks = max(have) + 1, sum(have) + 8
        ids = torch.randperm(blocks, generator=g, device="cuda").int()
        tables = torch.full((case["n"], width), -1, dtype=torch.int32, device="cuda")
        tables[torch.arange(width, device="cuda")[None, :] < _ints(have)[:, None]] = ids[:sum(have)]
        free = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
        free[:8] = ids[sum(have):]
        return {"op": op, "lens": _ints(lens), "gone": _ints(_released(case)), "tables": tables, "free": free, "count": _ints([8]), "blocks": blocks,
                "count_out": _ints([0]), "lens_out": _ints([0] * case["n"])}
    heads, dim, t = case["kv"] if op == "attn" else case["heads"], case["dim"], F[case["dtype"]]
    spread = torch.exp(0.5 * torch.randn(heads, 1, dim, device="cuda", generator=g))
    if op == "attn":
        lens = _lens(case, "ctx", case["batch"], case["lo"], case["hi"])
        width, blocks = max(_blocks(p) for p in lens), sum(_blocks(p) for p in lens) + 3
        ids = torch.randperm(blocks, generator=g, device="cuda").int()
        tables = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
        tables[torch.arange(width, device="cuda")[None, :] < _ints([_blocks(p) for p in lens])[:, None]] = ids[:blocks - 3]
        pool = torch.zeros(blocks, 1, heads, 20 * dim, dtype=torch.uint8, device="cuda")
        _fill(pool, g, dim, spread)
        q = torch.randn(case["batch"], case["heads"] * dim, device="cuda", generator=g).to(t)
        slopes = torch.exp2(-8.0 / case["heads"] * torch.arange(1, case["heads"] + 1, device="cuda").float()) if case["alibi"] else None
        return {"op": op, "q": q, "pool": pool, "tables": tables, "lens": _ints(lens), "out": torch.zeros(case["batch"], case["heads"], dim, dtype=t, device="cuda"),
                "slopes": slopes, "window": case["window"], "cap": case["cap"], "heads": case["heads"], "kv": heads, "dim": dim, "blocks": blocks}
    rows = case["rows"]
    blocks = _blocks(rows) + 3
    order = torch.randperm(blocks, generator=g, device="cuda")
    at = torch.arange(rows, device="cuda") + 5  # the first row follows five cached ones
    slots = (order[at // 16] * 16 + at % 16).int()
    slots = torch.cat([slots, torch.full((case["pad"],), -1, dtype=torch.int32, device="cuda")])  # rows behind the last sequence
    pool = torch.zeros(blocks, 1, heads, 20 * dim, dtype=torch.uint8, device="cuda")
    n = rows + case["pad"]
    state = {"op": op, "pool": pool, "slots": slots, "heads": heads, "dim": dim, "blocks": blocks,
             "k_out": torch.zeros(n, heads, dim, dtype=t, device="cuda"), "v_out": torch.zeros(n, heads, dim, dtype=t, device="cuda")}
    if op == "append":
        kv = torch.randn(n, 2, heads, dim, device="cuda", generator=g)
        kv[:, 0] *= spread[:, 0]
        state["kv_rows"] = kv.to(t)
    else:
        _fill(pool, g, dim, spread)
    return state


# ----------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    return {"map": _plain_map, "release": _plain_release, "append": _plain_append, "gather": _plain_gather, "attn": _plain_attn}[state["op"]](state)


def _plain_map(s):
    pre = s["pre"].long()
    new = torch.ones_like(pre) if s["new"] is None else s["new"].long()
    have = (pre + 15) // 16
    need = (pre + new + 15) // 16 - have
    upto = need.cumsum(0)
    ok = (need == 0) | (upto <= s["count"])
    first = s["count"].long() - 1 - (upto - need) + have  # list place of table column c: first - c
    tables, width = s["tables"], s["tables"].shape[1]
    col = torch.arange(width, device="cuda")[None, :]
    fresh = ok[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    tables = torch.where(fresh, s["free"][(first[:, None] - col).clamp(0, s["free"].numel() - 1)], tables)
    end = new.cumsum(0)
    row = torch.arange(s["slots"].numel(), device="cuda")
    b = torch.searchsorted(end, row, right=True).clamp(max=pre.numel() - 1)
    p = row - (end - new)[b] + pre[b]
    slots = tables[b, (p // 16).clamp(0, width - 1)] * 16 + p % 16
    slots = torch.where(ok[b] & (row < end[-1]), slots, torch.full_like(slots, -1))
    used = torch.where(ok & (need > 0), upto, torch.zeros_like(upto)).amax()
    return {"start": (end - new).int(), "post": torch.where(ok, pre + new, pre).int(), "slots": slots.int(), "tables": tables, "count": (s["count"] - used).int()}


def _plain_release(s):
    have = torch.where(s["gone"] != 0, (s["lens"].long() + 15) // 16, torch.zeros_like(s["lens"].long()))
    upto = have.cumsum(0)
    col = torch.arange(s["tables"].shape[1], device="cuda")[None, :]
    fresh = col < have[:, None]
    place = torch.where(fresh, s["count"].long() + (upto - have)[:, None] + col, torch.full_like(fresh, s["blocks"], dtype=torch.long))
    free = torch.cat([s["free"], s["free"][:1]])  # one place more takes the entries that stay
    free = free.scatter(0, place.flatten(), s["tables"].flatten())[:-1]
    return {"free": free, "count": (s["count"] + upto[-1]).int(), "lens": torch.where(s["gone"] != 0, torch.zeros_like(s["lens"]), s["lens"])}


def _plain_gather(s):
    kc, kp, vc, vp = _regions(s["pool"], s["dim"])
    slot = s["slots"].long().clamp(min=0)
    b, t = slot // 16, slot % 16
    keep = (s["slots"] >= 0)[:, None, None]
    k = _k_values(kc[b, 0, :, t], kp[b, 0, :, t])
    v = _v_values(vc[b, 0, :, :, t], vp[b, 0, :, t])
    return {"k": torch.where(keep, k, torch.zeros_like(k)).to(s["k_out"].dtype), "v": torch.where(keep, v, torch.zeros_like(v)).to(s["v_out"].dtype)}


def _plain_append(s):
    pool, rows = s["pool"], s["kv_rows"]
    spare = torch.cat([pool, pool[:1]])  # one block more takes the padded rows
    kc, kp, vc, vp = _regions(spare, s["dim"])
    slot = torch.where(s["slots"] >= 0, s["slots"].long(), torch.full_like(s["slots"], s["blocks"] * 16, dtype=torch.long))
    b, t = slot // 16, slot % 16
    c, sc, m = _quantise(rows[:, 0])
    kc[b, 0, :, t] = _k_bytes(c)
    kp[b, 0, :, t] = _params(sc, m)
    c, sc, m = _quantise(rows[:, 1])
    vc[b, 0, :, :, t] = _v_bytes(c)
    vp[b, 0, :, t] = _params(sc, m)
    pool.copy_(spare[:-1])
    return _plain_gather(s)


def _plain_attn(s):
    chunks = s["pool"][s["tables"].long().clamp(min=0), 0]  # [batch, blocks, kv heads, bytes]
    kc, kp, vc, vp = _regions(chunks, s["dim"])
    k = _k_values(kc, kp).movedim(2, 1).flatten(2, 3)  # [batch, kv heads, tokens, dim]
    v = _v_values(vc.movedim(-2, -3), vp).movedim(2, 1).flatten(2, 3)
    group = s["heads"] // s["kv"]
    q = s["q"].float().unflatten(1, (s["kv"], group, s["dim"]))
    x = q @ k.mT / math.sqrt(s["dim"])
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    at = torch.arange(k.shape[2], device="cuda")
    last = s["lens"][:, None] - 1
    seen = at <= last
    if s["window"]:
        seen = seen & (at > last - s["window"])
    if s["slopes"] is not None:
        x = x + s["slopes"].view(s["kv"], group, 1) * (at - last).float()[:, None, None, :]
    x = x.masked_fill(~seen[:, None, None, :], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    out = e @ v.masked_fill(~seen[:, None, :, None], 0.0) / e.sum(-1, keepdim=True)
    return out.flatten(1, 2).to(s["out"].dtype)


def _run_own(s):
    b2 = importlib.import_module("llm-inference-server_b200")
    op = s["op"]
    plan = s.get("plan")
    if plan is None:  # argument structs and workspaces, which a program keeps
        if op == "map":
            free = s["free"].new_zeros(s["blocks"])  # a pool's list has room for every block's id
            free[:s["free"].numel()] = s["free"]
            plan = b2.block_map_args(s["tables"], s["pre"], free, s["count"], s["slots"], new_lens=s["new"], q_start=s["start"],
                                     seq_lens_post=s["post"], free_count_out=s["count_out"], num_blocks=s["blocks"])
        elif op == "release":
            plan = b2.block_release_args(s["tables"], s["lens"], s["gone"], s["free"], s["count"], seq_lens_out=s["lens_out"],
                                         free_count_out=s["count_out"], num_blocks=s["blocks"])
        elif op == "attn":
            args = b2.attn_q4_args(s["q"], s["pool"], s["tables"], s["lens"], s["out"], n_head=s["heads"], n_kv_head=s["kv"], head_dim=s["dim"],
                                   layer_idx=0, n_layer=1, num_blocks=s["blocks"], softcap=s["cap"], window=s["window"], alibi_slopes=s["slopes"])
            plan = (args, b2.attention_q4_workspace(args))
        else:
            shape = dict(n_kv_head=s["heads"], head_dim=s["dim"], layer_idx=0, n_layer=1, num_blocks=s["blocks"])
            put = b2.kv_q4_args(s["pool"], s["kv_rows"][:, 0], s["kv_rows"][:, 1], s["slots"], **shape) if op == "append" else None
            plan = (put, b2.kv_q4_args(s["pool"], s["k_out"], s["v_out"], s["slots"], **shape))
        s["plan"] = plan
    if op == "map":
        b2.block_map(plan)
        return {"start": s["start"], "post": s["post"], "slots": s["slots"], "tables": s["tables"], "count": s["count_out"]}
    if op == "release":
        b2.block_release(plan)
        return {"free": s["free"], "count": s["count_out"], "lens": s["lens_out"]}
    if op == "attn":
        b2.paged_attention_q4(*plan)
        return s["out"]
    if op == "append":
        b2.kv_append_q4(plan[0])
    b2.kv_gather_q4(plan[1])
    return {"k": s["k_out"], "v": s["v_out"]}


# ----------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "map":
        pre, new = _map_lens(case)
        need = sum(_blocks(p + q) - _blocks(p) for p, q in zip(pre, new))
        return {"bytes": 4 * (4 * case["n"] + sum(new) + case["pad"] + 2 * need + sum(p % 16 > 0 for p in pre)), "flops": 0}
    if op == "release":
        lens = _lens(case, "pre", case["n"], case["lo"], case["hi"])
        return {"bytes": 4 * (3 * case["n"] + 2 * sum(_blocks(p) for p, x in zip(lens, _released(case)) if x)), "flops": 0}
    if op == "attn":
        lens = _lens(case, "ctx", case["batch"], case["lo"], case["hi"])
        seen = [min(p, case["window"] or p) for p in lens]
        rows = sum(seen)
        return {"bytes": rows * case["kv"] * case["dim"] * 5 // 4 + 4 * case["batch"] * case["heads"] * case["dim"] + 4 * sum(_blocks(p) for p in seen) + 4 * case["batch"],
                "flops": 4 * rows * case["heads"] * case["dim"]}
    n = case["rows"] * case["heads"] * case["dim"]
    thin, wide = n * 5 // 4, 4 * n
    return {"bytes": (2 * (thin + wide) if op == "append" else thin + wide) + 4 * (case["rows"] + case["pad"]), "flops": 8 * n}


# ----------------------------------------------------------------- from the definition, in 64 bits

def _element(pool, head, block, token, dim, d, value):
    """Element d (a tensor of dims) of K (value = 0) or V (1) rows at (block, token): by its address in the pool's bytes."""
    g = dim // 32
    group, e = d // 32, d % 32
    if value:
        unit = e // 4
        per = 16 // g
        code = 10 * dim + ((unit // per) * 16 + token) * 32 + (unit % per * g + group) * 2 + e % 4 // 2
    else:
        code = token * (dim // 2) + (e // 8 * g + group) * 4 + e % 8 // 2
    word = (18 if value else 8) * dim + (token * g + group) * 4
    flat = pool.flatten()
    base = (block * pool.shape[2] + head) * 20 * dim
    c = (flat[base + code].long() >> (e % 2 * 4)) & 15
    half = lambda at: (flat[at].to(torch.int16) | (flat[at + 1].to(torch.int16) << 8)).view(torch.float16).double()  # noqa: E731
    return (c - 8).double() * half(base + word + 2) + half(base + word)


def _exact_rows(x):
    """What rows x [n, heads, dim] read back as."""
    v = x.double().clamp(-65504, 65504).reshape(*x.shape[:2], -1, 32)
    low, high = v.min(-1, keepdim=True).values, v.max(-1, keepdim=True).values
    s = ((high - low) / 15).half().double()
    m = (low + 8 * s).half().double()
    c = torch.where(s > 0, torch.round((v - m) / s).clamp(-8, 7), torch.zeros_like(v))
    return (m + c.nan_to_num(0.0) * s).reshape(x.shape)


def exact(case, seed):
    op = case["op"]
    if op in ("map", "release"):
        return None
    s = prepare(case, seed)
    dim = case["dim"]
    d = torch.arange(dim, device="cuda")
    if op == "append":
        keep = (s["slots"] >= 0).double()[:, None, None]
        return {"k": _exact_rows(s["kv_rows"][:, 0]) * keep, "v": _exact_rows(s["kv_rows"][:, 1]) * keep}
    if op == "gather":
        slot = s["slots"].long()
        keep = (slot >= 0).double()[:, None, None]
        slot = slot.clamp(min=0)[:, None, None]
        head = torch.arange(s["heads"], device="cuda")[None, :, None]
        return {"k": _element(s["pool"], head, slot // 16, slot % 16, dim, d, 0) * keep, "v": _element(s["pool"], head, slot // 16, slot % 16, dim, d, 1) * keep}
    group = s["heads"] // s["kv"]
    out = torch.zeros(case["batch"], s["heads"], dim, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        j = torch.arange(first, n, device="cuda")
        block = s["tables"][b].long()[j // 16]
        head = torch.arange(s["kv"], device="cuda")[:, None, None]
        k = _element(s["pool"], head, block[:, None], (j % 16)[:, None], dim, d, 0)
        v = _element(s["pool"], head, block[:, None], (j % 16)[:, None], dim, d, 1)
        q = s["q"][b].double().view(s["kv"], group, dim)
        x = torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(dim)
        if case["cap"]:
            x = case["cap"] * torch.tanh(x / case["cap"])
        if s["slopes"] is not None:
            x = x + s["slopes"].double().view(s["kv"], group, 1) * (j - (n - 1)).double()
        out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(x, -1), v).reshape(s["heads"], dim)
    return out
