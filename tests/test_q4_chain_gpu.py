"""The 4-bit cache's calls after one another, on a B200: blocks given back and handed out again, rows read back for
attention over a 16-bit pool, launches on the stream that is current.

Tolerances (set from arithmetic before the first run): attention as in the tests of the operator; over rows read back to f16,
each K and V element is off by 2^-11 of itself, so a score by e = scale sum |q| |k| 2^-11, a weight by 2 e of itself,
an output by (2 e + 2^-11) sum w |v|, and fp32 sums of n terms by 2^-24 n of their magnitudes.
"""
from __future__ import annotations

import numpy as np
import pytest

import q4_ref as R
from test_kernels_gpu import ints_dev, to_dev
from test_q4_gpu import _check, _dense, _filled, _rng, _serving_state, _step, _tdt, _torch, rows16, tables_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,dim,kv,group", [(R.BF16, 128, 2, 4), (R.F16, 64, 3, 1)])
def test_released_blocks_serve_new_prompts(b2, cuda, dt, dim, kv, group):
    """Sequences end, prompts take their places in the batch and their blocks: old table entries lie behind the new ones, old rows
    in the blocks' tails.  Three generations, so that blocks pass from hand to hand."""
    torch = _torch()
    rng = _rng(dim + kv)
    n, blocks, mbps = 5, 17, 6
    s = _serving_state(b2, rng, dt, n, kv, group, dim, blocks, mbps, np.array([70, 33, 16, 47, 1], np.int32))
    shape = dict(n_kv_head=kv, head_dim=dim, layer_idx=0, n_layer=1, num_blocks=blocks)

    def decode(steps):
        for _ in range(steps):
            bits, x = rows16(rng, dt, (n, 2, kv, dim))
            q_bits, q = rows16(rng, dt, (n, kv * group, dim))
            s["kv"].copy_(to_dev(dt, bits))
            s["q"].copy_(to_dev(dt, q_bits))
            _step(b2, s)
            for b in range(n):
                s["rows"][b].append(x[b])
        got = s["out"].double().cpu().numpy()
        for b in range(n):
            p = _dense(s["rows"][b], dim)
            want, bound = R.attention(p, q[b:b + 1], np.arange(p.b.shape[0])[None], [len(s["rows"][b])], group=group)
            _check(got[b:b + 1], want, bound, dt)

    decode(3)
    for gone, fresh in (([0, 1], [20, 60]), ([1, 2, 4], [5, 48, 31]), ([0, 1, 2, 3, 4], [15, 16, 17, 1, 80])):
        flags = np.zeros(n, np.int32)
        flags[gone] = 1
        b2.block_release(b2.block_release_args(s["tables"], s["lens"], ints_dev(flags), s["free"], s["count"], num_blocks=blocks, seq_lens_out=s["lens"]))
        new = np.zeros(n, np.int32)
        new[gone] = fresh
        total = int(new.sum())
        bits, x = rows16(rng, dt, (total, 2, kv, dim))
        slots = torch.empty(total, dtype=torch.int32, device="cuda")
        start = torch.empty(n, dtype=torch.int32, device="cuda")
        b2.block_map(b2.block_map_args(s["tables"], s["lens"], s["free"], s["count"], slots, num_blocks=blocks, new_lens=ints_dev(new),
                                       q_start=start, seq_lens_post=s["lens"]))
        rows = to_dev(dt, bits)
        b2.kv_append_q4(b2.kv_q4_args(s["pool"], rows[:, 0], rows[:, 1], slots, **shape))
        for b, at in zip(gone, start.cpu().numpy()[gone]):
            s["rows"][b] = [x[at + i] for i in range(new[b])]
        decode(2)
        used = sum(-(-len(r) // 16) for r in s["rows"])
        assert s["count"].item() == blocks - used and b2.device_errors() == 0
        held = torch.cat([s["tables"][b, :-(-len(r) // 16)] for b, r in enumerate(s["rows"])] + [s["free"][:blocks - used]])
        assert sorted(held.tolist()) == list(range(blocks))  # every block in one place


def test_launches_go_to_the_current_stream(b2, cuda):
    torch = _torch()
    assert b2._stream(None) == torch.cuda.current_stream().cuda_stream
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert b2._stream(None) == side.cuda_stream == torch.cuda.current_stream().cuda_stream
        with torch.cuda.stream(other):
            assert b2._stream(None) == other.cuda_stream
        assert b2._stream(None) == side.cuda_stream
    assert b2._stream(other) == other.cuda_stream and b2._stream(7) == 7
    # a launch behind work of the side stream sees its result
    t = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens, free, count = ints_dev([17, 40]), ints_dev(np.arange(20)), ints_dev([0])
    slots = torch.full((2,), -5, dtype=torch.int32, device="cuda")
    args = b2.block_map_args(t, lens, free, count, slots, num_blocks=20, seq_lens_post=lens)
    torch.cuda.synchronize()
    big = torch.randn(4096, 4096, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(10):
            big = torch.tanh(big @ big)
        lens.fill_(18)
        b2.block_map(args)
    side.synchronize()
    assert slots.tolist() == [1 * 16 + 2, 5 * 16 + 2] and lens.tolist() == [19, 19] and b2.device_errors() == 0


def test_attention_over_rows_read_back(b2, cuda):
    """Rows read back into a 16-bit pool and attended by b2_paged_attention: off by the rounding of K and V to f16."""
    torch = _torch()
    rng = _rng(33)
    heads, dim, n = 4, 64, 100
    tables, blocks = tables_for(rng, [n])
    pool = _filled(rng, blocks, 1, heads, dim)
    q_bits, q = rows16(rng, R.F16, (1, heads, dim))
    want, _ = R.attention(pool, q, tables, [n], group=1)
    j = np.arange(n)
    at = tables[0][j // 16].astype(np.int64) * 16 + j % 16
    k = torch.empty(n, heads, dim, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    b2.kv_gather_q4(b2.kv_q4_args(torch.from_numpy(pool.b).cuda(), k, v, ints_dev(at), n_kv_head=heads, head_dim=dim, layer_idx=0,
                                  n_layer=1, num_blocks=blocks))
    wide = torch.zeros(blocks * 2 * 16 * heads * dim, dtype=torch.float16, device="cuda")
    b2.kv_append(wide, k, v, heads * dim, ints_dev(np.repeat(tables, n, 0)), ints_dev(j), n_kv_head=heads, head_dim=dim,
                 max_blocks_per_seq=tables.shape[1], layer_idx=0, n_layer=1, num_blocks=blocks)
    out = torch.empty(1, heads, dim, dtype=torch.float32, device="cuda")
    a = b2.attn_args(to_dev(R.F16, q_bits), heads * dim, wide, ints_dev(tables), ints_dev([n]), out, n_head=heads, n_kv_head=heads,
                     head_dim=dim, max_blocks_per_seq=tables.shape[1], layer_idx=0, n_layer=1, num_blocks=blocks)
    b2.paged_attention(a, b2.attention_workspace(a))
    kx, vx = pool.rows(at, 0)[:2]
    got = out.double().cpu().numpy()
    for h in range(heads):
        x = kx[:, h] @ q[0, h] / 8.0
        w = np.exp(x - x.max())
        w /= w.sum()
        e = (np.abs(kx[:, h]) @ np.abs(q[0, h])).max() / 8.0 * (2.0 ** -11 + 2.0 ** -24 * dim)
        bound = (2 * e + 2.0 ** -11 + 2.0 ** -24 * (n + 16)) * (w @ np.abs(vx[:, h]))
        assert np.all(np.abs(got[0, h] - want[0, h]) <= bound)
    assert bound.max() < 0.02  # outputs are of size 0.1


def test_the_widest_f16_group_reads_back_past_its_range(b2, cuda):
    """-65504 .. 65504: the step rounds up to 8736 and the top code stands for 65536, an infinity in f16; attention reads 65536."""
    torch = _torch()
    x = torch.zeros(1, 1, 64, device="cuda")
    x[0, 0, 3], x[0, 0, 9] = 65504.0, -65504.0
    pool = b2.kv_q4_pool(1, n_layer=1, n_kv_head=1, head_dim=64)
    pool.zero_()
    shape = dict(n_kv_head=1, head_dim=64, layer_idx=0, n_layer=1, num_blocks=1)
    back = {}
    for t in (torch.float16, torch.bfloat16):
        rows = x.to(t)
        b2.kv_append_q4(b2.kv_q4_args(pool, rows, rows, ints_dev([0]), **shape))
        k, v = torch.empty_like(rows), torch.empty_like(rows)
        b2.kv_gather_q4(b2.kv_q4_args(pool, k, v, ints_dev([0]), **shape))
        assert torch.equal(k, v)
        back[t] = k[0, 0, 3].item()
    assert back == {torch.float16: float("inf"), torch.bfloat16: 65536.0}
    out = torch.empty(1, 1, 64, dtype=torch.float32, device="cuda")
    a = b2.attn_q4_args(torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda"), pool, ints_dev([[0]]), ints_dev([1]), out, n_head=1, **shape)
    b2.paged_attention_q4(a, b2.attention_q4_workspace(a))
    assert abs(out[0, 0, 3].item() - 65536.0) <= 2.0 ** -11 * (8 * 8736 + 4384)
