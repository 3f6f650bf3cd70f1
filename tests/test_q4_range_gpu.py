"""The 4-bit paged KV pool where its numbers reach far: steps below f16's normal range, score caps of any size, long
contexts with one dominant key, values of very different sizes, scores near the end of fp32's precision.

Tolerances (set from arithmetic before the first run):
  * the bytes an append writes: equal;
  * attention: with w the exact weights, S and M the largest step and |middle| a group of 32 dims meets and n keys,
      (2^-11 + 2 e) sum w (8 s + |m|)  +  n (2^-30 S + 2^-36 M)  +  2^-20 max w max (8 s + |m|)
    where 2^-11 covers the rounding of weight times step and of weight to f16, n 2^-30 S and n 2^-36 M what weights far
    below the largest lose to f16's smallest number, and e the error of a score: 2^-18 (sum of the magnitudes of its
    products, + 1) and, under a cap, 2^-19 of the capped score; plus half a step of the output's type.
"""
from __future__ import annotations

import numpy as np
import pytest

import q4_ref as R
from test_kernels_gpu import ints_dev, to_dev
from test_q4_gpu import _attend, _check, _filled, _rng, _torch, rows16, tables_for

pytestmark = pytest.mark.gpu


def _want(pool, q, tables, lens, *, group, softcap=0.0, scale=0.0):
    """(out, bound) in float64.  Slots that a table names repeatedly are computed once."""
    batch, heads, dim = q.shape
    scale = scale or 1.0 / np.sqrt(dim)
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for b in range(batch):
        n = int(lens[b])
        j = np.arange(n)
        slots, times = np.unique(tables[b][j // 16].astype(np.int64) * 16 + j % 16, return_counts=True)
        k, v, ks, km, vs, vm = pool.rows(slots, 0)
        for h in range(heads):
            hk = h // group
            x = scale * (k[:, hk] @ q[b, h])
            mag = scale * ((8 * ks[:, hk] + np.abs(km[:, hk])).repeat(32, -1) @ np.abs(q[b, h]))
            err = 2.0 ** -18 * (mag.max() + 1.0)
            if softcap:
                x = softcap * np.tanh(x / softcap)
                err += 2.0 ** -19 * np.abs(x).max()
            w = np.exp(x - x.max()) * times
            top = 1.0 / w.sum()
            w *= top
            out[b, h] = w @ v[:, hk]
            each = (8 * vs[:, hk] + np.abs(vm[:, hk])).repeat(32, -1)
            lost = n * (2.0 ** -30 * vs[:, hk].max(0) + 2.0 ** -36 * np.abs(vm[:, hk]).max(0)).repeat(32)
            bound[b, h] = (2.0 ** -11 + 2 * err) * (w @ each) + lost + 2.0 ** -20 * top * each.max(0)
    return out, bound


# ------------------------------------------------------------------ append

def _small_groups(rng, dt):
    """Groups of 32 whose steps lie around and below f16's smallest normal number, as multiples of 2^-30 (so that no quotient lies next to a rounding border)."""
    tiny, out = 2.0 ** -24, []
    for span in list(range(1, 301)) + [15360 + i for i in (-40, -9, -1, 0, 1, 8, 40)]:  # 15 steps of 2^-14 = 15360 2^-24
        for low in (0, -(span // 2), -span, 7):
            g = rng.integers(0, span + 1, size=32)
            g[rng.permutation(32)[:2]] = 0, span
            out.append((g + low) * tiny)
    for at in range(32):
        g = np.zeros(32)
        g[at] = 22 * tiny
        out += [g, -g]
    out.append(np.where(np.arange(32) % 2, 22 * tiny, 0.0))
    for std in 10.0 ** rng.uniform(-7, -4, size=1500):
        out.append(np.rint(rng.standard_normal(32) * std * 2.0 ** 30) * 2.0 ** -30)
    bits = R.O.round_to(dt, np.asarray(out, np.float32).ravel())
    return bits.reshape(-1, 32)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dt", [R.F16, R.BF16])
def test_append_of_groups_with_subnormal_steps(b2, cuda, dt, dim):
    torch = _torch()
    rng = _rng(dim + dt)
    heads, g = 2, dim // 32
    bits = _small_groups(rng, dt)
    rows = -(-bits.shape[0] // (2 * heads * g))
    bits = np.concatenate([bits, bits[:rows * 2 * heads * g - bits.shape[0]]]).reshape(rows, 2, heads, dim)
    x = R.widen(dt, bits)
    blocks = -(-rows // 16)
    pool = R.Pool(blocks, 1, heads, dim, np.zeros(blocks * heads * 20 * dim))
    dev = torch.from_numpy(pool.b.copy()).cuda()
    kv = to_dev(dt, bits)
    b2.kv_append_q4(b2.kv_q4_args(dev, kv[:, 0], kv[:, 1], ints_dev(np.arange(rows)), n_kv_head=heads, head_dim=dim, layer_idx=0,
                                  n_layer=1, num_blocks=blocks))
    for r in range(rows):
        pool.put(r, 0, x[r, 0], x[r, 1])
    assert np.array_equal(dev.cpu().numpy(), pool.b)
    assert b2.device_errors() == 0


@pytest.mark.parametrize("dt", [R.F16, R.BF16])
def test_append_of_any_finite_bits_follows_the_format_in_fp32(b2, cuda, dt):
    """Random bit patterns: elements up to 2^40 apart in one group, saturated ones, ties that fp32 decides.  The format restated in numpy's fp32."""
    torch = _torch()
    rng = _rng(7 + dt)
    rows, heads, dim = 2000, 2, 64
    bits = rng.integers(0, 65536, size=(rows, 2, heads, dim)).astype(np.uint16)
    top = 0x7C00 if dt == R.F16 else 0x7F80
    bits = np.where((bits & top) == top, bits & 0x83FF, bits).astype(np.uint16)  # finite
    x = np.clip(R.widen(dt, bits), -65504.0, 65504.0).astype(np.float32).reshape(rows, 2, heads, 2, 32)
    lo, hi = x.min(-1), x.max(-1)
    s = ((hi - lo) / np.float32(15)).astype(np.float16)
    m = (np.float32(8) * s.astype(np.float32) + lo).astype(np.float16)
    s32, m32 = s.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
    c = np.where(s32 > 0, np.rint(np.clip((x - m32) / np.where(s32 > 0, s32, np.float32(1)), -8, 7)), 0)
    want = (c.astype(np.float64) * s32 + m32).reshape(rows, 2, heads, dim)
    pool = R.Pool(-(-rows // 16), 1, heads, dim, np.zeros(-(-rows // 16) * heads * 20 * dim))
    dev = torch.from_numpy(pool.b).cuda()
    kv = to_dev(dt, bits)
    b2.kv_append_q4(b2.kv_q4_args(dev, kv[:, 0], kv[:, 1], ints_dev(np.arange(rows)), n_kv_head=heads, head_dim=dim, layer_idx=0,
                                  n_layer=1, num_blocks=pool.b.shape[0]))
    pool.b[:] = dev.cpu().numpy()
    k, v, ks, km, vs, vm = pool.rows(np.arange(rows), 0)
    for i, (got, steps, middles) in enumerate(((k, ks, km), (v, vs, vm))):
        assert np.array_equal(steps, s[:, i].astype(np.float64)) and np.array_equal(middles, m[:, i].astype(np.float64))
        assert np.array_equal(got, want[:, i])
    assert b2.device_errors() == 0


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("cap", [0.25, 3.0, 30.0, 1e2, 1e3, 1e5, 1e7, 1e30, 3e38])
@pytest.mark.parametrize("dt,dim,group", [(R.F16, 64, 1), (R.BF16, 128, 4)])
def test_a_cap_of_any_size_keeps_the_scores(b2, cuda, dt, dim, group, cap):
    torch = _torch()
    rng = _rng(int(np.log2(cap)) + 50)
    lens = np.array([300, 1, 77, 32], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, dim)
    q_bits, q = rows16(rng, dt, (4, 2 * group, dim), 5.0)
    want, bound = _want(pool, q, tables, lens, group=group, softcap=cap)
    got = _attend(b2, dt, pool, q_bits, tables, lens, group=group, softcap=cap, out_dtype=torch.float32)[0]
    _check(got, want, bound, dt, True)
    assert b2.device_errors() == 0


@pytest.mark.parametrize("n", [131072, 1 << 20])
@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_far_below_a_peak_keep_their_mass(b2, cuda, dim, spread, n):
    # The warps of one CTA take a quarter of the keys each; each quarter has one key 25.4 binary orders above the others.
    torch = _torch()
    pool = R.Pool(2, 1, 1, dim, np.zeros(2 * 20 * dim))
    d = np.arange(dim)
    plain, peak = np.zeros((1, dim)), np.zeros((1, dim))
    peak[0, 0] = 17.6
    some = (1.0 + spread * np.sin(d))[None].astype(np.float16).astype(np.float64)
    for s in range(32):
        pool.put(s, 0, peak if s == 3 else plain, np.zeros((1, dim)) if s == 3 else some)
    q = np.zeros((1, 1, dim))
    q[0, 0, 0] = np.sqrt(128.0) if dim == 128 else 8.0
    q_bits = R.O.round_to(R.F16, q.astype(np.float32).ravel()).reshape(q.shape)
    q = R.widen(R.F16, q_bits)
    tables = np.ones((1, n // 16), np.int32)
    tables[0, ::n // 64] = 0
    want, bound = _want(pool, q, tables, [n], group=1)
    got = _attend(b2, R.F16, pool, q_bits, tables, np.array([n], np.int32), group=1, out_dtype=torch.float32, max_ctas=1)[0]
    _check(got, want, bound, R.F16, True)


@pytest.mark.parametrize("ratio", [10, 14, 18, 22])
@pytest.mark.parametrize("dt,dim,group", [(R.F16, 64, 2), (R.BF16, 128, 4)])
def test_groups_of_dims_of_different_sizes(b2, cuda, dt, dim, group, ratio):
    torch = _torch()
    rng = _rng(ratio + dim)
    lens = np.array([500, 40, 1], np.int32)
    tables, blocks = tables_for(rng, lens)
    spread = np.where(np.arange(dim) // 32 == 1, 2.0 ** (ratio - 10), 2.0 ** -10)
    pool = _filled(rng, blocks, 1, 2, dim, v_spread=spread)
    q_bits, q = rows16(rng, dt, (3, 2 * group, dim), 3.0)
    want, bound = _want(pool, q, tables, lens, group=group)
    got = _attend(b2, dt, pool, q_bits, tables, lens, group=group, out_dtype=torch.float32)[0]
    _check(got, want, bound, dt, True)


@pytest.mark.parametrize("ratio", [8, 12, 16])
@pytest.mark.parametrize("at", [0, 150, 299])
def test_one_key_with_huge_values_and_no_weight(b2, cuda, ratio, at):
    torch = _torch()
    rng = _rng(ratio + at)
    dim, n = 64, 300
    tables, blocks = tables_for(rng, [n])
    pool = _filled(rng, blocks, 1, 1, dim, v_spread=2.0 ** -3)
    q_bits, q = rows16(rng, R.F16, (1, 2, dim))
    q_bits[0, 1], q[0, 1] = q_bits[0, 0], q[0, 0]
    k = -5.0 * np.sign(q[0, :1])
    v = rng.standard_normal((1, dim)) * 2.0 ** (ratio - 3)
    pool.put(int(tables[0, at // 16]) * 16 + at % 16, 0, k, v.astype(np.float16).astype(np.float64))
    want, bound = _want(pool, q, tables, [n], group=2)
    got = _attend(b2, R.F16, pool, q_bits, tables, np.array([n], np.int32), group=2, out_dtype=torch.float32)[0]
    _check(got, want, bound, R.F16, True)


def test_scores_of_any_size_choose_the_largest(b2, cuda):
    """Queries up to 2^110: where the largest score leads by more than its rounding, the output is that key's value."""
    rng = _rng(91)
    lens = np.array([300, 33, 5], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, 64)
    clear = 0
    for top in (20, 24, 26, 27, 28, 30, 60, 100, 108):
        q_bits, q = rows16(rng, R.BF16, (3, 4, 64), 2.0 ** (top - 2))
        got = _attend(b2, R.BF16, pool, q_bits, tables, lens, group=2)[0]
        assert np.all(np.isfinite(got))
        for b in range(3):
            j = np.arange(lens[b])
            k, v, ks, km, vs, vm = pool.rows(tables[b][j // 16].astype(np.int64) * 16 + j % 16, 0)
            for h in range(4):
                x = k[:, h // 2] @ q[b, h] / 8.0
                mag = ((8 * ks[:, h // 2] + np.abs(km[:, h // 2])).repeat(32, -1) @ np.abs(q[b, h])).max() / 8.0
                first, second = np.sort(x)[::-1][:2]
                if first - second <= 2.0 ** -17 * mag + 60.0:  # a lead of 60 leaves the others e^-60
                    continue
                clear += 1
                i = int(np.argmax(x))
                want = v[i, h // 2]
                each = (8 * vs[i, h // 2] + np.abs(vm[i, h // 2])).repeat(32)
                assert np.all(np.abs(got[b, h] - want) <= 2.0 ** -11 * each + np.abs(want) * 2.0 ** -7)
    assert clear > 60


def test_scores_a_rounding_step_apart(b2, cuda):
    """Scores of 2^26 to 2^27 (in log2 units), where fp32 holds multiples of 8: in each warp the second step's are about one step above
    the first's, and the steps of its values 2^6 times the first's."""
    torch = _torch()
    dim, heads, batch = 64, 1, 128  # (one head: a head whose reference moves takes the others along)
    rng = _rng(92)
    pool = R.Pool(4, 1, 1, dim, np.zeros(4 * 20 * dim))
    small = (rng.standard_normal((1, dim))).astype(np.float16).astype(np.float64)
    for s in range(64):
        k = np.ones((1, dim))  # a step of 0: exact
        k[0, 32:] = 1.0 if s < 32 else 2.0
        pool.put(s, 0, k, small if s < 32 else small * 64.0)
    q = np.zeros((batch, heads, dim))
    q[..., 0] = 2.0 ** 28 * rng.uniform(1.4, 2.7, size=(batch, heads))  # x = (q0 + q1 or 2 q1) / 8 log2 e
    q[..., 32] = 8.0 * 8.0 / np.log2(np.e) * rng.uniform(0.8, 1.5, size=(batch, heads))
    q_bits = R.O.round_to(R.BF16, q.astype(np.float32).ravel()).reshape(q.shape)
    tables = np.tile(np.tile(np.arange(4, dtype=np.int32), 4), (batch, 1))
    got = _attend(b2, R.BF16, pool, q_bits, tables, np.full(batch, 256, np.int32), group=1, out_dtype=torch.float32, max_ctas=128)[0]
    v = pool.rows(np.arange(64), 0)[1][:, 0]
    lo, hi = v.min(0), v.max(0)
    slack = 2.0 ** -10 * (hi - lo + np.abs(hi) + np.abs(lo))
    assert np.all(np.isfinite(got)) and np.all(got >= lo - slack) and np.all(got <= hi + slack)


@pytest.mark.parametrize("power", [-110, -60, 60, 112])
def test_scale_and_queries_of_opposite_size(b2, cuda, power):
    """scale 2^power and queries of 2^-power: the same scores, and the same bits, as with neither (powers of two are exact)."""
    rng = _rng(5)
    lens = np.array([100, 33], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, 64)
    q_bits, q = rows16(rng, R.BF16, (2, 4, 64))
    want, bound = _want(pool, q, tables, lens, group=2, scale=0.25)
    plain = _attend(b2, R.BF16, pool, q_bits, tables, lens, group=2, scale=0.25)[0]
    _check(plain, want, bound, R.BF16)
    far = R.O.round_to(R.BF16, (q * 2.0 ** -power).astype(np.float32).ravel()).reshape(q.shape)
    assert np.array_equal(_attend(b2, R.BF16, pool, far, tables, lens, group=2, scale=0.25 * 2.0 ** power)[0], plain)


@pytest.mark.parametrize("size", [65504.0, 30000.0, 1e-3, 1e-5, 3e-7])
@pytest.mark.parametrize("dt,dim,group", [(R.F16, 64, 2), (R.BF16, 128, 3)])
def test_values_at_the_ends_of_f16s_range(b2, cuda, dt, dim, group, size):
    """Steps of up to 8736 and down to 2^-24 (below 2^-14, f16's products of a weight and a step end at 2^-45 instead of 2^-30 of the largest)."""
    torch = _torch()
    rng = _rng(int(-np.log(size)) + 60)
    lens = np.array([100, 37], np.int32)
    tables, blocks = tables_for(rng, lens)
    pool = _filled(rng, blocks, 1, 2, dim)
    v = (rng.uniform(-size, size, size=(blocks * 16, 2, dim))).astype(np.float16).astype(np.float64)
    for s in range(blocks * 16):
        k_half = pool.b[s // 16, 0, :, :10 * dim].copy()
        pool.put(s, 0, v[s], v[s])
        pool.b[s // 16, 0, :, :10 * dim] = k_half  # V alone
    q_bits, q = rows16(rng, dt, (2, 2 * group, dim), 4.0)
    want, bound = _want(pool, q, tables, lens, group=group)
    got = _attend(b2, dt, pool, q_bits, tables, lens, group=group, out_dtype=torch.float32)[0]
    _check(got, want, bound + 100 * 2.0 ** -45, dt, True)
    assert b2.device_errors() == 0


@pytest.mark.parametrize("ratio", [8, 14, 20])
@pytest.mark.parametrize("dt", [R.F16, R.BF16])
def test_queries_with_one_huge_element(b2, cuda, dt, ratio):
    """One element of q 2^ratio times the others, at a dim whose keys are 0 (their group's step is 0 too): the others, kept to 2^-29 of it,
    make the scores."""
    torch = _torch()
    rng = _rng(ratio)
    dim, n = 64, 200
    tables, blocks = tables_for(rng, [n])
    pool = _filled(rng, blocks, 1, 1, dim, k_spread=np.where(np.arange(dim) < 32, 0.0, 1.0))
    q_bits, q = rows16(rng, dt, (1, 4, dim), 2.0 ** -6)
    q[:, :, 5] = 2.0 ** (ratio - 6)
    q_bits = R.O.round_to(dt, q.astype(np.float32).ravel()).reshape(q.shape)
    q = R.widen(dt, q_bits)
    want, bound = _want(pool, q, tables, [n], group=4, scale=8.0)
    k, v, ks, km, vs, vm = pool.rows(tables[0][np.arange(n) // 16].astype(np.int64) * 16 + np.arange(n) % 16, 0)
    err = 8.0 * 2.0 ** (ratio - 6 - 29) * (32 * (8 * ks[:, 0] + np.abs(km[:, 0]))).sum(-1).max()  # of a score
    bound += 2 * err * np.abs(v).max()
    got = _attend(b2, dt, pool, q_bits, tables, np.array([n], np.int32), group=4, scale=8.0, out_dtype=torch.float32)[0]
    _check(got, want, bound, dt, True)
    # The bound is not idle: at 2^20 a score may be off by 8 2^-15 32 (8 s + |m|) = 0.029 with s up to 0.4 and |m| up to 0.5 in
    # one group, an output by twice that times the largest value, 3.9: 0.23.  It falls with the ratio.
    assert bound.max() < 0.1 * np.abs(v).max()
