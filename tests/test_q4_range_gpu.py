"""The 4-bit paged KV pool where its numbers reach far: steps below f16's normal range.

Tolerances (set from arithmetic before the first run):
  * the bytes an append writes: equal.
"""
from __future__ import annotations

import numpy as np
import pytest

import q4_ref as R
from test_kernels_gpu import ints_dev, to_dev
from test_q4_gpu import _rng, _torch

pytestmark = pytest.mark.gpu


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
