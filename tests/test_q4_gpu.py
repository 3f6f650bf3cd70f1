"""Block maps and the 4-bit paged KV pool on the GPU, through the C-ABI, against 64-bit and integer restatements.

Tolerances (set from arithmetic before the first run):
  * block maps, releases, the bytes an append writes: equal;
  * gather: the value the codes stand for, rounded to fp32 and then to the dtype: half an fp32 step plus half a step of
    the dtype (f16 below its normal range: 2^-25);
  * attention: q4_ref.attention's bound plus half a step of the output's dtype.
"""
from __future__ import annotations

import numpy as np
import pytest

import q4_ref as R
from test_kernels_gpu import ints_dev, to_dev

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def _rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


def _tdt(dt):
    torch = _torch()
    return torch.float16 if dt == R.F16 else torch.bfloat16


def rows16(rng, dt, shape, spread=1.0):
    """Random rows in 16 bits: (bit patterns, their float64 values)."""
    bits = R.O.round_to(dt, (rng.standard_normal(int(np.prod(shape))) * spread).astype(np.float32)).reshape(shape)
    return bits, R.widen(dt, bits)


def tables_for(rng, lens, extra=0, slack=3):
    """Block tables of randomly placed blocks for lens tokens each (-1 behind), and the pool's block count."""
    nb = [-(-max(0, int(n)) // 16) for n in lens]
    width, blocks = max(1, max(nb, default=0) + extra), sum(nb) + slack
    perm = rng.permutation(blocks).astype(np.int32)
    bt = np.full((len(lens), width), -1, np.int32)
    o = 0
    for b, n in enumerate(nb):
        bt[b, :n] = perm[o:o + n]
        o += n
    return bt, blocks


# ------------------------------------------------------------------ block maps

MAP_CASES = {
    "decode": dict(n=64, lo=0, hi=300, new=None),
    "one": dict(n=1, lo=0, hi=1, new=(1, 2)),
    "prefill-ragged": dict(n=37, lo=0, hi=80, new=(0, 200), pad=7),
    "odd-pad": dict(n=5, lo=3, hi=50, new=(1, 30), pad=1),
    "no-rows": dict(n=9, lo=0, hi=50, new=(0, 1)),
    "runs-out": dict(n=50, lo=0, hi=60, new=(0, 90), room=0.5),
    "runs-out-at-once": dict(n=50, lo=0, hi=60, new=(1, 90), room=0.0),
    "rows-run-out": dict(n=20, lo=0, hi=60, new=(1, 40), pad=-90),
    "many": dict(n=5000, lo=0, hi=40, new=(0, 30)),
    "most": dict(n=16384, lo=0, hi=20, new=(0, 3)),
    "long": dict(n=3, lo=0, hi=9, new=(20000, 70000)),
}


@pytest.mark.parametrize("name", list(MAP_CASES))
@pytest.mark.parametrize("in_place", [False, True])
def test_block_map(b2, cuda, name, in_place):
    torch = _torch()
    c = MAP_CASES[name]
    rng = _rng(len(name) * 7 + 1)
    n = c["n"]
    pre = rng.integers(c["lo"], c["hi"], size=n).astype(np.int32)
    new = np.ones(n, np.int32) if c["new"] is None else rng.integers(*c["new"], size=n).astype(np.int32)
    have, total = -(-pre // 16), -(-(pre + new) // 16)
    width = int(total.max()) + 2
    need = int((total - have).sum())
    num_blocks = int(have.sum()) + need + 5
    perm = rng.permutation(num_blocks).astype(np.int32)
    tables = np.full((n, width), -7, np.int32)
    o = 0
    for b in range(n):
        tables[b, :have[b]] = perm[o:o + have[b]]
        o += have[b]
    free = np.full(num_blocks, -9, np.int32)
    free[:num_blocks - o] = perm[o:]
    count = int(need * c.get("room", 1.0)) if "room" in c else num_blocks - o
    max_rows = max(0, int(new.sum()) + c.get("pad", 0))
    want = R.block_map(tables, pre, new, free, count, num_blocks, max_rows)
    t = ints_dev(tables)
    p, f, cnt = ints_dev(pre), ints_dev(free), ints_dev([count])
    slots = torch.full((max_rows,), -5, dtype=torch.int32, device="cuda")
    start = torch.full((n,), -5, dtype=torch.int32, device="cuda")
    post = p if in_place else torch.full((n,), -5, dtype=torch.int32, device="cuda")
    out = cnt if in_place else torch.full((1,), -5, dtype=torch.int32, device="cuda")
    args = b2.block_map_args(t, p, f, cnt, slots, num_blocks=num_blocks, new_lens=None if c["new"] is None else ints_dev(new),
                             q_start=start, seq_lens_post=post, free_count_out=None if in_place else out)
    b2.block_map(args)
    got = [x.cpu().numpy() for x in (t, slots, start, post)]
    for g, w in zip(got, want[:4]):
        assert np.array_equal(g, w)
    assert int(out.item()) == want[4]
    assert b2.device_errors() == want[5]
    assert np.array_equal(f.cpu().numpy(), free)


def test_block_map_refuses_bad_lengths_and_ids(b2, cuda):
    torch = _torch()
    pre = np.array([5, -3, 20, 127, 0, 8, 2 ** 31 - 1], np.int32)
    new = np.array([20, 4, -2, 5, 2 ** 31 - 1, 3, 2 ** 31 - 1], np.int32)
    tables = np.full((7, 8), -1, np.int32)
    tables[0, 0], tables[2, :2], tables[3, :8], tables[5, 0] = 99, [1, 2], np.arange(3, 11), 11  # 99: outside the pool
    free = np.array([12, 50, 13] + [0] * 17, np.int32)  # 50: outside
    want = R.block_map(tables, pre, new, free, 3, 20, 64)
    t, slots = ints_dev(tables), torch.zeros(64, dtype=torch.int32, device="cuda")
    start, post = torch.zeros(7, dtype=torch.int32, device="cuda"), torch.zeros(7, dtype=torch.int32, device="cuda")
    cnt = ints_dev([3])
    b2.block_map(b2.block_map_args(t, ints_dev(pre), ints_dev(free), cnt, slots, num_blocks=20, new_lens=ints_dev(new),
                                   q_start=start, seq_lens_post=post))
    for g, w in zip((t, slots, start, post), want[:4]):
        assert np.array_equal(g.cpu().numpy(), w)
    assert int(cnt.item()) == want[4] and b2.device_errors() == want[5]
    for bad, cut in ((-4, 0), (21, 20)):
        cnt = ints_dev([bad])
        b2.block_map(b2.block_map_args(ints_dev(np.full((1, 8), -1)), ints_dev([0]), ints_dev(np.arange(20)), cnt, slots,
                                       num_blocks=20, new_lens=ints_dev([1])))
        assert int(cnt.item()) == (0 if cut == 0 else 19)
        assert b2.device_errors() == (b2.DEVERR_BLOCK_ID | (b2.DEVERR_NO_BLOCKS if cut == 0 else 0))


def test_block_map_without_sequences_fills_the_slots(b2, cuda):
    torch = _torch()
    slots = torch.zeros(9, dtype=torch.int32, device="cuda")
    cnt = ints_dev([3])
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    b2.block_map(b2.block_map_args(torch.empty(0, 4, dtype=torch.int32, device="cuda"), e, ints_dev([1, 2, 3]), cnt, slots, num_blocks=3))
    assert slots.tolist() == [-1] * 9 and cnt.item() == 3


@pytest.mark.parametrize("n,hi,share", [(1, 5, 1.0), (128, 1011, 0.1), (700, 300, 0.5), (5000, 60, 1.0), (16384, 30, 0.3), (40, 9, 0.0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_block_release(b2, cuda, n, hi, share, in_place):
    torch = _torch()
    rng = _rng(n + hi)
    lens = rng.integers(0, hi + 1, size=n).astype(np.int32)
    gone = (rng.random(n) < share).astype(np.int32) * rng.integers(1, 9, size=n).astype(np.int32)
    tables, blocks = tables_for(rng, lens, extra=1, slack=4)
    free = np.full(blocks, -1, np.int32)
    want = R.block_release(tables, lens, gone, free, 4, blocks)
    f, ln, cnt = ints_dev(free), ints_dev(lens), ints_dev([4])
    lo = ln if in_place else torch.full((n,), -5, dtype=torch.int32, device="cuda")
    out = cnt if in_place else ints_dev([-5])
    b2.block_release(b2.block_release_args(ints_dev(tables), ln, ints_dev(gone), f, cnt, num_blocks=blocks, seq_lens_out=lo,
                                           free_count_out=None if in_place else out))
    assert np.array_equal(f.cpu().numpy(), want[0]) and np.array_equal(lo.cpu().numpy(), want[1])
    assert int(out.item()) == want[2] and b2.device_errors() == want[3] == 0


def test_block_release_leaves_out_bad_ids_and_what_does_not_fit(b2, cuda):
    rng = _rng(3)
    lens = np.array([40, 1000, -3, 33, 16, 100] * 50, np.int32)
    tables = rng.integers(0, 4000, size=(300, 8)).astype(np.int32)
    tables[::7, 1], tables[5, 0] = -1, 4000
    gone = np.ones(300, np.int32)
    for count, blocks in ((0, 4000), (3000, 4000), (-2, 4000), (4001, 4000)):
        free = np.arange(blocks, dtype=np.int32)
        want = R.block_release(tables, lens, gone, free, count, blocks)
        f, cnt, lo = ints_dev(free), ints_dev([count]), ints_dev(np.zeros(300))
        b2.block_release(b2.block_release_args(ints_dev(tables), ints_dev(lens), ints_dev(gone), f, cnt, num_blocks=blocks, seq_lens_out=lo))
        assert np.array_equal(f.cpu().numpy(), want[0]) and np.array_equal(lo.cpu().numpy(), want[1])
        assert int(cnt.item()) == want[2] and b2.device_errors() == want[3]


def test_map_then_release_gives_every_block_back(b2, cuda):
    torch = _torch()
    rng = _rng(8)
    n, blocks = 33, 200
    free, cnt = ints_dev(rng.permutation(blocks)), ints_dev([blocks])
    t = torch.full((n, 16), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(n, dtype=torch.int32, device="cuda")
    new = ints_dev(rng.integers(0, 60, size=n))
    slots = torch.empty(int(new.sum()), dtype=torch.int32, device="cuda")
    b2.block_map(b2.block_map_args(t, lens, free, cnt, slots, num_blocks=blocks, new_lens=new, seq_lens_post=lens))
    assert torch.equal(lens, new) and slots.unique().numel() == slots.numel() and int(slots.min()) >= 0
    b2.block_release(b2.block_release_args(t, lens, torch.ones_like(lens), free, cnt, num_blocks=blocks, seq_lens_out=lens))
    assert cnt.item() == blocks and sorted(free.tolist()) == list(range(blocks)) and not lens.any()
    assert b2.device_errors() == 0


# ------------------------------------------------------------------ append and gather

KV_CASES = [  # dtype, heads, dim, rows, layers, layer
    (R.F16, 12, 64, 64, 1, 0), (R.BF16, 8, 128, 200, 1, 0), (R.F16, 1, 64, 1, 1, 0), (R.BF16, 25, 64, 77, 3, 2),
    (R.F16, 3, 128, 130, 2, 1), (R.BF16, 1, 128, 17, 1, 0), (R.F16, 7, 64, 1011, 1, 0),
]


def _special_rows(bits, dt):
    """Rows with constant groups, tiny and huge values, NaN and infinities."""
    one, huge, inf, nan = (0x3C00, 0x7BFF, 0x7C00, 0x7E00) if dt == R.F16 else (0x3F80, 0x7F7F, 0x7F80, 0x7FC0)
    flat = bits.reshape(bits.shape[0], -1)
    flat[0, :32] = one
    flat[-1, :32] = 0
    flat[0, 32:64] = np.arange(32)  # subnormal
    if bits.shape[0] > 4:
        flat[1, 3], flat[1, 5] = huge, huge | 0x8000
        flat[2, 40] = nan
        flat[3, 7] = inf
        flat[4, 33] = inf | 0x8000
    return flat.reshape(bits.shape)


@pytest.mark.parametrize("case", KV_CASES)
def test_append_writes_the_formats_bytes_and_no_others(b2, cuda, case):
    torch = _torch()
    dt, heads, dim, rows, layers, layer = case
    rng = _rng(rows + heads)
    blocks = -(-rows // 16) + 4
    bits, x = rows16(rng, dt, (rows, 2, heads, dim), np.exp(rng.standard_normal(rows * 2 * heads * dim)))
    bits[:, 0] = _special_rows(bits[:, 0].copy(), dt)
    bits[:, 1] = _special_rows(bits[:, 1].copy(), dt)
    x = R.widen(dt, bits)
    slots = rng.permutation(blocks * 16)[:rows].astype(np.int32)
    if rows > 10:
        slots[5], slots[9] = -1, -12345
    fill = rng.integers(0, 256, size=blocks * layers * heads * 20 * dim)
    pool = R.Pool(blocks, layers, heads, dim, fill)
    dev = torch.from_numpy(pool.b.copy()).cuda()
    kv = to_dev(dt, bits)
    b2.kv_append_q4(b2.kv_q4_args(dev, kv[:, 0], kv[:, 1], ints_dev(slots), n_kv_head=heads, head_dim=dim, layer_idx=layer,
                                  n_layer=layers, num_blocks=blocks))
    for r in range(rows):
        if slots[r] >= 0:
            pool.put(int(slots[r]), layer, x[r, 0], x[r, 1])
    got = dev.cpu().numpy()
    # a group that reads back as NaN may hold any codes
    bad = ~np.isfinite(x).reshape(rows, 2, heads, dim // 32, 32).all(-1)
    ko, vo, _ = R.chunk_offsets(dim)
    for r, kv_i, h, g in zip(*np.nonzero(bad)):
        if slots[r] >= 0:
            at = (vo if kv_i else ko)[g * 32:(g + 1) * 32] + slots[r] % 16 * (32 if kv_i else dim // 2)
            pool.b[slots[r] // 16, layer, h, at] = got[slots[r] // 16, layer, h, at]
    assert np.array_equal(got, pool.b)
    assert b2.device_errors() == 0


@pytest.mark.parametrize("case", KV_CASES)
def test_gather_reads_what_the_codes_stand_for(b2, cuda, case):
    torch = _torch()
    dt, heads, dim, rows, layers, layer = case
    rng = _rng(rows * 3 + heads)
    blocks = -(-rows // 16) + 4
    pool = R.Pool(blocks, layers, heads, dim, rng.integers(0, 256, size=blocks * layers * heads * 20 * dim))
    g = dim // 32
    for base in (8 * dim, 18 * dim):  # params of ordinary size
        w = pool.b[..., base:base + 64 * g].reshape(blocks, layers, heads, 16, g, 4)
        w[..., 0:2] = (rng.standard_normal(w.shape[:-1]) * 3).astype(np.float16).view(np.uint8).reshape(*w.shape[:-1], 2)
        w[..., 2:4] = np.abs(rng.standard_normal(w.shape[:-1]) * 10.0 ** rng.integers(-6, 2, size=w.shape[:-1])).astype(np.float16).view(np.uint8).reshape(*w.shape[:-1], 2)
    slots = rng.integers(0, blocks * 16, size=rows).astype(np.int32)  # repeats allowed
    if rows > 10:
        slots[3] = -1
    width = heads * dim + 24  # strided rows
    buf = torch.full((rows, 2 * width), 7.0, dtype=_tdt(dt), device="cuda")
    k, v = buf[:, :heads * dim], buf[:, width:width + heads * dim]
    b2.kv_gather_q4(b2.kv_q4_args(torch.from_numpy(pool.b).cuda(), k, v, ints_dev(slots), n_kv_head=heads, head_dim=dim,
                                  layer_idx=layer, n_layer=layers, num_blocks=blocks))
    got = buf.float().cpu().numpy().astype(np.float64)
    keep = slots >= 0
    want = pool.rows(np.maximum(slots, 0), layer)
    for at, w in ((0, want[0]), (width, want[1])):
        gk = got[:, at:at + heads * dim].reshape(rows, heads, dim)
        tol = np.abs(w) * (R.EPS[dt] / 2 + 2.0 ** -23) + 2.0 ** -25
        assert np.all(np.abs(gk - w)[keep] <= tol[keep])
        assert np.all(gk[~keep] == 7.0)
    assert np.all(got[:, heads * dim:width] == 7.0) and np.all(got[:, width + heads * dim:] == 7.0)
    assert b2.device_errors() == 0


def test_slots_behind_the_pool_are_skipped_and_flagged(b2, cuda):
    torch = _torch()
    pool = torch.zeros(4, 1, 2, 1280, dtype=torch.uint8, device="cuda")
    k = torch.randn(3, 2, 64, device="cuda").half()
    shape = dict(n_kv_head=2, head_dim=64, layer_idx=0, n_layer=1, num_blocks=3)  # the fourth block is not the pool's
    b2.kv_append_q4(b2.kv_q4_args(pool, k, k, ints_dev([48, 63, 2 ** 31 - 1]), **shape))
    assert b2.device_errors() == b2.DEVERR_BLOCK_ID and not pool.any()
    out = torch.full_like(k, 3.0)
    b2.kv_gather_q4(b2.kv_q4_args(pool, out, out, ints_dev([48, 63, 2 ** 31 - 1]), **shape))
    assert b2.device_errors() == b2.DEVERR_BLOCK_ID and bool((out == 3.0).all())


def test_pool_offsets_past_32_bits(b2, cuda):
    torch = _torch()
    heads, dim, layers = 8, 128, 4
    blocks = (1 << 32) // (layers * heads * 20 * dim) + 5000  # 4.7 GB
    pool = b2.kv_q4_pool(blocks, n_layer=layers, n_kv_head=heads, head_dim=dim)
    last = blocks - 1
    pool[last].zero_()
    rng = _rng(2)
    bits, x = rows16(rng, R.BF16, (16, 2, heads, dim))
    kv = to_dev(R.BF16, bits)
    slots = ints_dev(last * 16 + np.arange(16))
    shape = dict(n_kv_head=heads, head_dim=dim, layer_idx=3, n_layer=layers, num_blocks=blocks)
    b2.kv_append_q4(b2.kv_q4_args(pool, kv[:, 0], kv[:, 1], slots, **shape))
    ref = R.Pool(1, layers, heads, dim, np.zeros(layers * heads * 20 * dim))
    for t in range(16):
        ref.put(t, 3, x[t, 0], x[t, 1])
    assert np.array_equal(pool[last].cpu().numpy(), ref.b[0])
    out = torch.empty(16, 2, heads, dim, dtype=torch.bfloat16, device="cuda")
    b2.kv_gather_q4(b2.kv_q4_args(pool, out[:, 0], out[:, 1], slots, **shape))
    w = ref.rows(np.arange(16), 3)
    got = out.float().cpu().numpy()
    assert np.all(np.abs(got[:, 0] - w[0]) <= np.abs(w[0]) * (2.0 ** -8 + 2.0 ** -23) + 2.0 ** -25)
    q = torch.randn(1, heads, dim, device="cuda").to(torch.bfloat16)
    o = torch.empty(1, heads, dim, dtype=torch.float32, device="cuda")
    a = b2.attn_q4_args(q, pool, ints_dev([[last]]), ints_dev([16]), o, n_head=heads, n_kv_head=heads, head_dim=dim, layer_idx=3,
                        n_layer=layers, num_blocks=blocks)
    b2.paged_attention_q4(a, b2.attention_q4_workspace(a))
    want, bound = R.attention(ref, q.double().cpu().numpy(), np.array([[0]]), [16], group=1, layer=3)
    assert np.all(np.abs(o.double().cpu().numpy() - want) <= bound + np.abs(want) * 2.0 ** -24)
    assert b2.device_errors() == 0


# ------------------------------------------------------------------ attention

def _filled(rng, blocks, layers, heads, dim, k_spread=1.0, v_spread=1.0, v_shift=0.0):
    """A pool whose every slot holds quantised normal rows, all at once."""
    pool = R.Pool(blocks, layers, heads, dim, np.zeros(blocks * layers * heads * 20 * dim))
    g = dim // 32
    ko, vo, odd = R.chunk_offsets(dim)
    flat = pool.b.reshape(-1, 20 * dim)
    for off, stride, par, spread, shift in ((ko, dim // 2, 8 * dim, k_spread, 0.0), (vo, 32, 18 * dim, v_spread, v_shift)):
        c, s, m = R.quantise((rng.standard_normal((flat.shape[0], 16, dim)) * spread + shift).astype(np.float16).astype(np.float64))
        c = c.reshape(flat.shape[0], 16, dim) << (4 * odd).astype(np.uint8)
        for t in range(16):
            flat[:, off[odd == 0] + t * stride] = c[:, t, odd == 0]
            flat[:, off[odd == 1] + t * stride] |= c[:, t, odd == 1]
        w = (s.view(np.uint16).astype(np.uint32) << 16 | m.view(np.uint16)).astype("<u4")
        flat[:, par:par + 64 * g] = w.view(np.uint8).reshape(flat.shape[0], -1)
    return pool


def _attend(b2, dt, pool, q_bits, tables, lens, *, group, out_dtype=None, layer=0, ws=None, max_ctas=0, times=1, poison=True, **kw):
    torch = _torch()
    batch, heads, dim = q_bits.shape
    blocks, layers, kv = pool.b.shape[:3]
    dev = torch.from_numpy(pool.b).cuda()
    out = torch.full((batch, heads, dim), float("nan"), dtype=out_dtype or _tdt(dt), device="cuda")
    q = to_dev(dt, q_bits)
    ints = {k: ints_dev(v) for k, v in (("key_starts", kw.pop("starts", None)),) if v is not None}
    slopes = kw.pop("slopes", None)
    if slopes is not None:
        ints["alibi_slopes"] = torch.tensor(np.asarray(slopes), dtype=torch.float32, device="cuda")
    a = b2.attn_q4_args(q, dev, ints_dev(tables), ints_dev(lens), out, n_head=heads, n_kv_head=kv, head_dim=dim,
                        layer_idx=layer, n_layer=layers, num_blocks=blocks, max_ctas=max_ctas, **ints, **kw)
    ws = b2.attention_q4_workspace(a) if ws is None else ws
    got = []
    for _ in range(times):
        b2.paged_attention_q4(a, ws)
        got.append(out.double().cpu().numpy())
    return got


def _poison(pool, tables, lens, firsts=None):
    """NaN params and all-ones codes in every slot that no query may see."""
    seen = np.zeros(pool.b.shape[0] * 16, bool)
    for b, n in enumerate(lens):
        j = np.arange(0 if firsts is None else firsts[b], max(0, int(n)))
        seen[tables[b][j // 16].astype(np.int64) * 16 + j % 16] = True
    dim, g = pool.dim, pool.dim // 32
    for s in np.nonzero(~seen)[0]:
        t = s % 16
        pool.b[s // 16, :, :, 8 * dim + t * g * 4: 8 * dim + (t + 1) * g * 4] = 0xFF
        pool.b[s // 16, :, :, 18 * dim + t * g * 4: 18 * dim + (t + 1) * g * 4] = 0xFF


def _check(got, want, bound, dt, out32=False):
    eps = 2.0 ** -23 if out32 else R.EPS[dt]
    tol = bound + (np.abs(want) + bound) * eps / 2 + (0 if out32 else 2.0 ** -25)
    err = np.abs(got - want)
    assert np.all(np.isfinite(got)) and np.all(err <= tol), f"error {err.max():.3g}, {np.max(err / tol):.3g} of its bound"


ATTN_CASES = {
    "boundaries": dict(dt=R.F16, dim=64, kv=12, group=1, lens=[1, 15, 16, 17, 31, 32, 33, 200]),
    "microbench": dict(dt=R.F16, dim=64, kv=12, group=1, lens=(64, 128, 1024)),
    "xl-heads": dict(dt=R.BF16, dim=64, kv=25, group=1, lens=(9, 1, 300), layers=3, layer=2),
    "gqa4": dict(dt=R.BF16, dim=128, kv=8, group=4, lens=[512, 700, 33, 1000, 1]),
    "gqa2": dict(dt=R.F16, dim=128, kv=8, group=2, lens=(6, 1, 400), layers=2, layer=1),
    "gqa8": dict(dt=R.F16, dim=64, kv=2, group=8, lens=(4, 1, 100)),
    "odd-groups-3": dict(dt=R.BF16, dim=128, kv=3, group=3, lens=(5, 1, 300)),
    "odd-groups-5": dict(dt=R.F16, dim=64, kv=1, group=5, lens=(5, 1, 300)),
    "odd-groups-7": dict(dt=R.F16, dim=128, kv=2, group=7, lens=(3, 1, 200)),
    "one-token": dict(dt=R.F16, dim=64, kv=1, group=1, lens=[1]),
    "one-token-each": dict(dt=R.BF16, dim=128, kv=2, group=4, lens=[1] * 40),
    "one-long": dict(dt=R.F16, dim=64, kv=12, group=1, lens=[5000]),
    "one-longer": dict(dt=R.BF16, dim=128, kv=1, group=8, lens=[40001]),
    "skew": dict(dt=R.BF16, dim=64, kv=4, group=1, lens=[6000] + list(range(1, 41))),
    "empty": dict(dt=R.F16, dim=64, kv=4, group=1, lens=[0, 7, 0, 100, 0]),
    "all-empty": dict(dt=R.F16, dim=128, kv=2, group=2, lens=[0, 0, 0]),
    "many": dict(dt=R.F16, dim=64, kv=1, group=2, lens=(3000, 0, 40)),
    "window": dict(dt=R.BF16, dim=128, kv=2, group=4, lens=(9, 1, 900), window=100),
    "window-1": dict(dt=R.F16, dim=64, kv=3, group=1, lens=(9, 1, 90), window=1),
    "window-17": dict(dt=R.F16, dim=64, kv=3, group=2, lens=[16, 17, 18, 33, 200], window=17),
    "softcap": dict(dt=R.F16, dim=128, kv=2, group=2, lens=(7, 1, 400), softcap=5.0),
    "alibi": dict(dt=R.F16, dim=64, kv=16, group=1, lens=(5, 1, 500), alibi=True),
    "alibi-up": dict(dt=R.BF16, dim=128, kv=2, group=3, lens=(5, 1, 500), alibi=-0.3),
    "all-options": dict(dt=R.BF16, dim=128, kv=2, group=4, lens=(6, 1, 700), window=333, softcap=20.0, alibi=True, starts=True, scale=0.2),
    "documents": dict(dt=R.F16, dim=64, kv=2, group=1, lens=[50, 64, 7, 300, 33, 5], starts=[10, 64, -5, 255, 32, 100]),
    "peaked": dict(dt=R.F16, dim=64, kv=2, group=2, lens=(6, 1, 600), q_spread=30.0),
    "tiny-values": dict(dt=R.BF16, dim=64, kv=2, group=1, lens=(6, 1, 600), v_spread=1e-3),
    "huge-values": dict(dt=R.BF16, dim=128, kv=2, group=2, lens=(6, 1, 600), v_spread=1e4),
    "shifted-values": dict(dt=R.F16, dim=64, kv=2, group=2, lens=(6, 1, 600), v_shift=50.0),
    "tiny-queries": dict(dt=R.BF16, dim=64, kv=2, group=2, lens=(6, 1, 300), q_spread=1e-20),
    "huge-queries": dict(dt=R.BF16, dim=64, kv=2, group=2, lens=(6, 1, 300), q_spread=1e30),
    "few-ctas": dict(dt=R.F16, dim=128, kv=4, group=4, lens=(11, 1, 700), max_ctas=3),
    "one-cta": dict(dt=R.F16, dim=64, kv=4, group=1, lens=(11, 1, 300), max_ctas=1),
}


def _setup(name):
    c = ATTN_CASES[name]
    rng = _rng(sum(map(ord, name)))
    lens = c["lens"]
    if isinstance(lens, tuple):
        n, lo, hi = lens
        lens = rng.integers(lo, hi + 1, size=n)
    lens = np.asarray(lens, np.int32)
    tables, blocks = tables_for(rng, lens, extra=1)
    pool = _filled(rng, blocks, c.get("layers", 1), c["kv"], c["dim"], v_spread=c.get("v_spread", 1.0), v_shift=c.get("v_shift", 0.0))
    heads = c["kv"] * c["group"]
    q_bits, q = rows16(rng, c["dt"], (len(lens), heads, c["dim"]), c.get("q_spread", 1.0))
    opt = {k: c[k] for k in ("window", "softcap", "scale") if k in c}
    starts = c.get("starts")
    if starts is True:
        starts = rng.integers(0, 200, size=len(lens))
    if starts is not None:
        opt["starts"] = np.asarray(starts, np.int32)
    if "alibi" in c:
        opt["slopes"] = (2.0 ** (-8.0 / heads * np.arange(1, heads + 1))).astype(np.float32) if c["alibi"] is True else np.full(heads, c["alibi"], np.float32)
    firsts = np.zeros(len(lens), np.int64)
    if "window" in opt:
        firsts = np.maximum(firsts, lens.astype(np.int64) - opt["window"])
    if starts is not None:
        firsts = np.maximum(firsts, opt["starts"])
    _poison(pool, tables, lens, firsts)
    return c, pool, q_bits, q, tables, lens, opt


@pytest.mark.parametrize("name", list(ATTN_CASES))
def test_attention(b2, cuda, name):
    c, pool, q_bits, q, tables, lens, opt = _setup(name)
    want, bound = R.attention(pool, q, tables, lens, group=c["group"], layer=c.get("layer", 0), **opt)
    if name == "huge-queries":  # scores of 1e30: a rounding of one may choose another key
        x = _attend(b2, c["dt"], pool, q_bits, tables, lens, group=c["group"], **dict(opt))[0]
        assert np.all(np.isfinite(x))
        assert b2.device_errors() == 0
        return
    torch = _torch()
    for out_dtype in (None, torch.float32):
        a, b = _attend(b2, c["dt"], pool, q_bits, tables, lens, group=c["group"], out_dtype=out_dtype, layer=c.get("layer", 0),
                       max_ctas=c.get("max_ctas", 0), times=2, **dict(opt))
        _check(a, want, bound, c["dt"], out_dtype is not None)
        assert np.array_equal(a, b)  # the same bits again, with the workspace as the first launch left it
    assert b2.device_errors() == 0


def test_attention_q_rows_inside_a_fused_buffer(b2, cuda):
    torch = _torch()
    rng = _rng(12)
    lens = np.array([5, 77, 300], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 4, 64)
    bits, x = rows16(rng, R.F16, (3, 3 * 4 * 64))
    buf = to_dev(R.F16, bits)
    out = torch.empty(3, 4, 64, dtype=torch.float16, device="cuda")
    a = b2.attn_q4_args(buf[:, 256:512], torch.from_numpy(pool.b).cuda(), ints_dev(tables), ints_dev(lens), out, n_head=4,
                        n_kv_head=4, head_dim=64, layer_idx=0, n_layer=1, num_blocks=blocks)
    b2.paged_attention_q4(a, b2.attention_q4_workspace(a))
    want, bound = R.attention(pool, x[:, 256:512].reshape(3, 4, 64), tables, lens, group=1)
    _check(out.double().cpu().numpy(), want, bound, R.F16)


def test_attention_nan_stays_in_its_sequence_head_and_group(b2, cuda):
    rng = _rng(13)
    lens = np.array([50, 60], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, 64)
    q_bits, q = rows16(rng, R.F16, (2, 4, 64))
    clean, bound = R.attention(pool, q, tables, lens, group=2)
    word = 18 * 64 + 3 * 8 + 4  # V params of token 3, group 1
    pool.b[tables[0, 1], 0, 1, word:word + 4] = 0xFF
    got = _attend(b2, R.F16, pool, q_bits, tables, lens, group=2)[0]
    bad = np.zeros(got.shape, bool)
    bad[0, 2:4, 32:] = True
    assert np.all(np.isnan(got[bad]))
    assert np.all(np.abs(got - clean)[~bad] <= (bound + (np.abs(clean) + bound) * 2.0 ** -11 + 2.0 ** -25)[~bad])
    q_bits[1, 3, 5] = 0x7C00  # an infinite query: only its own row is lost
    got2 = _attend(b2, R.F16, pool, q_bits, tables, lens, group=2)[0]
    assert np.all(np.isnan(got2[1, 3])) and np.array_equal(got2[1, :3], got[1, :3])


def test_attention_clamps_bad_pages_and_lengths(b2, cuda):
    rng = _rng(14)
    lens = np.array([40, 64], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, 64)
    q_bits, q = rows16(rng, R.F16, (2, 2, 64))
    bad = tables.copy()
    bad[0, 1], bad[1, 0] = blocks, -3
    cut = bad.copy()
    cut[0, 1], cut[1, 0] = blocks - 1, 0
    want, bound = R.attention(pool, q, cut, lens, group=1)
    got = _attend(b2, R.F16, pool, q_bits, bad, lens, group=1)[0]
    assert b2.device_errors() == b2.DEVERR_BLOCK_ID
    _check(got, want, bound, R.F16)
    want, bound = R.attention(pool, q, tables, np.array([0, 64]), group=1)
    got = _attend(b2, R.F16, pool, q_bits, tables, np.array([-5, 2 ** 31 - 1], np.int32), group=1)[0]
    assert b2.device_errors() == b2.DEVERR_SEQ_LEN
    _check(got, want, bound, R.F16)


def test_workspace_is_checked(b2, cuda):
    torch = _torch()
    rng = _rng(15)
    lens = np.array([40], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = torch.from_numpy(_filled(rng, blocks, 1, 1, 64).b).cuda()
    q = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda")
    a = b2.attn_q4_args(q, pool, ints_dev(tables), ints_dev(lens), torch.empty_like(q), n_head=1, n_kv_head=1, head_dim=64,
                        layer_idx=0, n_layer=1, num_blocks=blocks)
    ws = b2.attention_q4_workspace(a)
    with pytest.raises(b2.B2Error) as e:
        b2.paged_attention_q4(a, ws[:ws.numel() - 1])
    assert e.value.code == -5
    with pytest.raises(b2.B2Error) as e:
        b2.paged_attention_q4(a, ws[4:])
    assert e.value.code == -5


def test_calls_of_different_shapes_share_a_workspace(b2, cuda):
    torch = _torch()
    names = ["gqa4", "microbench", "few-ctas", "one-long", "odd-groups-7", "one-cta", "gqa8"]
    ws = torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")
    for name in names * 2:
        c, pool, q_bits, q, tables, lens, opt = _setup(name)
        want, bound = R.attention(pool, q, tables, lens, group=c["group"], layer=c.get("layer", 0), **opt)
        got = _attend(b2, c["dt"], pool, q_bits, tables, lens, group=c["group"], layer=c.get("layer", 0), max_ctas=c.get("max_ctas", 0),
                      ws=ws, **dict(opt))[0]
        _check(got, want, bound, c["dt"])
    assert not ws[:4096].any()  # the counters
    assert b2.device_errors() == 0


@pytest.mark.parametrize("dt,dim,group", [(R.F16, 64, 3), (R.BF16, 128, 4)])
def test_attention_on_any_number_of_ctas(b2, cuda, dt, dim, group):
    rng = _rng(77)
    lens = np.array([700, 3, 64], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, dim)
    q_bits, q = rows16(rng, dt, (3, 2 * group, dim))
    want, bound = R.attention(pool, q, tables, lens, group=group)
    for n in (1, 2, 5, 17, 100, 0):
        _check(_attend(b2, dt, pool, q_bits, tables, lens, group=group, max_ctas=n)[0], want, bound, dt)


def test_tiny_softcap_and_zero_scores(b2, cuda):
    # x / cap overflows for every nonzero score: tanh is 1 or -1, and 0 for the zero query of head 1.
    rng = _rng(78)
    lens = np.array([40], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, 64)
    q_bits, q = rows16(rng, R.F16, (1, 2, 64))
    q_bits[0, 1], q[0, 1] = 0, 0.0
    want, bound = R.attention(pool, q, tables, lens, group=1, softcap=1e-37)
    _check(_attend(b2, R.F16, pool, q_bits, tables, lens, group=1, softcap=1e-37)[0], want, bound, R.F16)
    assert b2.device_errors() == 0


# ------------------------------------------------------------------ together

def _step(b2, s, stream=None):
    b2.block_map(s["map"], stream)
    b2.kv_append_q4(s["put"], stream)
    b2.paged_attention_q4(s["attn"], s["ws"], stream)


def _serving_state(b2, rng, dt, n, kv, group, dim, blocks, mbps, lens0):
    """A decode loop's buffers, the sequences' first lens0 tokens appended as a prefill."""
    torch = _torch()
    s = {"free": ints_dev(rng.permutation(blocks)), "count": ints_dev([blocks]), "lens": torch.zeros(n, dtype=torch.int32, device="cuda"),
         "tables": torch.full((n, mbps), -1, dtype=torch.int32, device="cuda"),
         "pool": b2.kv_q4_pool(blocks, n_layer=1, n_kv_head=kv, head_dim=dim)}
    s["pool"].fill_(0xFF)  # what nobody wrote reads as NaN
    shape = dict(n_kv_head=kv, head_dim=dim, layer_idx=0, n_layer=1, num_blocks=blocks)
    total = int(lens0.sum())
    bits, x = rows16(rng, dt, (total, 2, kv, dim))
    slots = torch.empty(total + 5, dtype=torch.int32, device="cuda")  # five padded rows
    pad = torch.cat([to_dev(dt, bits), torch.zeros(5, 2, kv, dim, dtype=_tdt(dt), device="cuda")])
    b2.block_map(b2.block_map_args(s["tables"], s["lens"], s["free"], s["count"], slots, num_blocks=blocks, new_lens=ints_dev(lens0),
                                   seq_lens_post=s["lens"]))
    b2.kv_append_q4(b2.kv_q4_args(s["pool"], pad[:, 0], pad[:, 1], slots, **shape))
    at = np.concatenate([[0], np.cumsum(lens0)])
    s["rows"] = [[x[at[b] + i] for i in range(lens0[b])] for b in range(n)]
    s["kv"] = torch.empty(n, 2, kv, dim, dtype=_tdt(dt), device="cuda")
    s["q"] = torch.empty(n, kv * group, dim, dtype=_tdt(dt), device="cuda")
    s["out"] = torch.empty_like(s["q"])
    s["slots"] = torch.empty(n, dtype=torch.int32, device="cuda")
    s["map"] = b2.block_map_args(s["tables"], s["lens"], s["free"], s["count"], s["slots"], num_blocks=blocks, seq_lens_post=s["lens"])
    s["put"] = b2.kv_q4_args(s["pool"], s["kv"][:, 0], s["kv"][:, 1], s["slots"], **shape)
    s["attn"] = b2.attn_q4_args(s["q"], s["pool"], s["tables"], s["lens"], s["out"], n_head=kv * group, window=0, **shape)
    s["ws"] = b2.attention_q4_workspace(s["attn"])
    return s


def _dense(rows, dim):
    """A pool that holds one sequence's rows in order."""
    p = R.Pool(-(-len(rows) // 16), 1, rows[0].shape[1], dim, np.zeros(-(-len(rows) // 16) * rows[0].shape[1] * 20 * dim))
    for i, r in enumerate(rows):
        p.put(i, 0, r[0], r[1])
    return p


@pytest.mark.parametrize("graph", [False, True])
def test_serving_loop(b2, cuda, graph):
    """Prefill, then decode steps of map -> append -> attention on the device alone, once as a captured graph on a side stream."""
    torch = _torch()
    rng = _rng(21)
    dt, n, kv, group, dim, blocks, mbps = R.BF16, 6, 2, 4, 128, 40, 8
    lens0 = np.array([1, 15, 16, 17, 40, 3], np.int32)
    s = _serving_state(b2, rng, dt, n, kv, group, dim, blocks, mbps, lens0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = None
    for step in range(20):
        bits, x = rows16(rng, dt, (n, 2, kv, dim))
        q_bits, q = rows16(rng, dt, (n, kv * group, dim))
        with torch.cuda.stream(side):
            s["kv"].copy_(to_dev(dt, bits))
            s["q"].copy_(to_dev(dt, q_bits))
            if graph:
                if g is None:
                    torch.cuda.synchronize()
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=side):
                        _step(b2, s)
                g.replay()
            else:
                _step(b2, s)
        side.synchronize()
        for b in range(n):
            s["rows"][b].append(x[b])
        got = s["out"].double().cpu().numpy()
        for b in (step % n, n - 1):
            p = _dense(s["rows"][b], dim)
            want, bound = R.attention(p, q[b:b + 1], np.arange(p.b.shape[0])[None], [len(s["rows"][b])], group=group)
            _check(got[b:b + 1], want, bound, dt)
    assert s["lens"].tolist() == [len(r) for r in s["rows"]]
    need = sum(-(-len(r) // 16) for r in s["rows"])
    assert s["count"].item() == blocks - need and b2.device_errors() == 0
    # sequences 1 and 4 end; their blocks serve a new prompt
    gone = ints_dev([0, 1, 0, 0, 1, 0])
    b2.block_release(b2.block_release_args(s["tables"], s["lens"], gone, s["free"], s["count"], num_blocks=blocks, seq_lens_out=s["lens"]))
    assert s["count"].item() == blocks - need + sum(-(-len(s["rows"][b]) // 16) for b in (1, 4))
    assert s["lens"].tolist() == [0 if b in (1, 4) else len(r) for b, r in enumerate(s["rows"])]
    assert b2.device_errors() == 0


def test_two_streams_with_their_own_workspaces(b2, cuda):
    torch = _torch()
    c, pool, q_bits, q, tables, lens, opt = _setup("gqa4")
    want, bound = R.attention(pool, q, tables, lens, group=c["group"])
    dev, qd, t, ln = torch.from_numpy(pool.b).cuda(), to_dev(c["dt"], q_bits), ints_dev(tables), ints_dev(lens)
    sides = []
    for _ in range(2):
        out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
        a = b2.attn_q4_args(qd, dev, t, ln, out, n_head=32, n_kv_head=8, head_dim=128, layer_idx=0, n_layer=1, num_blocks=pool.b.shape[0])
        sides.append((torch.cuda.Stream(), a, b2.attention_q4_workspace(a), out))
    torch.cuda.synchronize()
    for _ in range(50):
        for st, a, ws, _ in sides:
            b2.paged_attention_q4(a, ws, stream=st)
    torch.cuda.synchronize()
    for _, _, _, out in sides:
        _check(out.double().cpu().numpy(), want, bound, c["dt"])
    assert b2.device_errors() == 0


def test_prefill_over_a_gathered_prefix_matches_decode(b2, cuda):
    """Rows read back into a 16-bit pool and attended by b2_paged_attention: the same result as over the 4-bit pool."""
    torch = _torch()
    rng = _rng(31)
    heads, dim, n = 4, 64, 100
    tables, blocks = tables_for(rng, [n])
    pool = _filled(rng, blocks, 1, heads, dim)
    dev = torch.from_numpy(pool.b).cuda()
    q_bits, q = rows16(rng, R.F16, (1, heads, dim))
    want, bound = R.attention(pool, q, tables, [n], group=1)
    j = np.arange(n)
    slots = ints_dev(tables[0][j // 16] * 16 + j % 16)
    k = torch.empty(n, heads, dim, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    b2.kv_gather_q4(b2.kv_q4_args(dev, k, v, slots, n_kv_head=heads, head_dim=dim, layer_idx=0, n_layer=1, num_blocks=blocks))
    wide = torch.zeros(blocks * 2 * 16 * heads * dim, dtype=torch.float16, device="cuda")
    b2.kv_append(wide, k, v, heads * dim, ints_dev(np.repeat(tables, n, 0)), ints_dev(j), n_kv_head=heads, head_dim=dim,
                 max_blocks_per_seq=tables.shape[1], layer_idx=0, n_layer=1, num_blocks=blocks)
    out = torch.empty(1, heads, dim, dtype=torch.float32, device="cuda")
    a = b2.attn_args(to_dev(R.F16, q_bits), heads * dim, wide, ints_dev(tables), ints_dev([n]), out, n_head=heads, n_kv_head=heads,
                     head_dim=dim, max_blocks_per_seq=tables.shape[1], layer_idx=0, n_layer=1, num_blocks=blocks)
    b2.paged_attention(a, b2.attention_workspace(a))
    # K and V rounded once more to f16 on the way: 2^-11 of every product of a score and of every value
    mag = float(np.abs(q).max() * np.abs(k.double().cpu().numpy()).max() * dim / np.sqrt(dim))
    extra = (2 * 2.0 ** -11 * mag + 2.0 ** -11) * np.abs(v.double().cpu().numpy()).max()
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound + extra + 2e-3)
