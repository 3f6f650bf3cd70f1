"""Block maps and the 4-bit KV pool: argument checks on the host and the format's arithmetic (CPU only)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import q4_ref as R


def test_argument_structs_match_the_header(b2, tmp_path):
    import shutil
    import subprocess
    from conftest import ROOT
    names = {"B2BlockMapArgs": b2.BlockMapArgs, "B2BlockReleaseArgs": b2.BlockReleaseArgs, "B2KvQ4Args": b2.KvQ4Args,
             "B2PagedAttnQ4Args": b2.PagedAttnQ4Args}
    lines = [f'printf("%zu\\n", sizeof({c}));' for c in names]
    for c, s in names.items():
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in s._fields_]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "b2_decode.h"\nint main(void) { ' + "\n".join(lines) + " return 0; }\n")
    subprocess.run([shutil.which("gcc"), "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    want = [ctypes.sizeof(s) for s in names.values()]
    for s in names.values():
        want += [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


def _map(b2, **kw):
    base = dict(n_seqs=4, max_blocks_per_seq=8, num_blocks=100, max_rows=16, seq_lens_pre=16, new_lens=32, free_list=48,
                free_count=64, block_tables=80, slots=96, q_start=112, seq_lens_post=128, free_count_out=64)
    base.update(kw)
    return b2.BlockMapArgs(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(n_seqs=-1), -3), (dict(n_seqs=16385), -3), (dict(max_rows=-1), -3), (dict(max_rows=(1 << 30) + 1), -3),
    (dict(max_blocks_per_seq=0), -3), (dict(num_blocks=0), -3), (dict(num_blocks=1 << 27), -3),
    (dict(seq_lens_pre=None), -1), (dict(free_list=None), -1), (dict(free_count=None), -1), (dict(free_count_out=None), -1),
    (dict(block_tables=None), -1), (dict(slots=None), -1), (dict(slots=100), -4), (dict(seq_lens_post=32), -3),
])
def test_block_map_host_checks(b2, kw, code):
    assert b2.load().b2_block_map(ctypes.byref(_map(b2, **kw)), None) == code
    assert b2.load().b2_last_error_string().decode() != ""
    assert b2.load().b2_block_map(None, None) == -1


def _release(b2, **kw):
    base = dict(n_seqs=4, max_blocks_per_seq=8, num_blocks=100, block_tables=16, seq_lens=32, release=48, free_list=64,
                free_count=80, free_count_out=80, seq_lens_out=32)
    base.update(kw)
    return b2.BlockReleaseArgs(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(n_seqs=-1), -3), (dict(n_seqs=16385), -3), (dict(max_blocks_per_seq=0), -3), (dict(num_blocks=-5), -3),
    (dict(block_tables=None), -1), (dict(seq_lens=None), -1), (dict(release=None), -1), (dict(free_list=None), -1),
    (dict(free_count=None), -1), (dict(free_count_out=None), -1),
])
def test_block_release_host_checks(b2, kw, code):
    assert b2.load().b2_block_release(ctypes.byref(_release(b2, **kw)), None) == code
    assert b2.load().b2_last_error_string().decode() != ""


def _kv(b2, **kw):
    base = dict(dtype=b2.F16, kv_pool=16, k=32, v=48, row_stride=768, slots=64, rows=3, n_kv_head=12, head_dim=64,
                layer_idx=0, n_layer=1, num_blocks=10)
    base.update(kw)
    return b2.KvQ4Args(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), -2), (dict(dtype=9), -2), (dict(rows=-1), -3), (dict(head_dim=96), -6), (dict(n_kv_head=0), -3),
    (dict(layer_idx=1), -3), (dict(layer_idx=-1), -3), (dict(num_blocks=0), -3), (dict(num_blocks=1 << 27), -3),
    (dict(num_blocks=1 << 26, n_layer=48), -3), (dict(kv_pool=None), -1), (dict(k=None), -1), (dict(v=None), -1),
    (dict(slots=None), -1), (dict(row_stride=767), -3), (dict(row_stride=772), -4), (dict(k=40), -4), (dict(v=56), -4),
    (dict(kv_pool=24), -4),
])
def test_kv_q4_host_checks(b2, kw, code):
    lib = b2.load()
    for fn in (lib.b2_kv_append_q4, lib.b2_kv_gather_q4):
        assert fn(ctypes.byref(_kv(b2, **kw)), None) == code
        assert lib.b2_last_error_string().decode() != ""


def test_kv_q4_no_rows_is_a_no_op(b2):
    lib = b2.load()
    for fn in (lib.b2_kv_append_q4, lib.b2_kv_gather_q4):
        assert fn(ctypes.byref(_kv(b2, rows=0, k=None, v=None, slots=None)), None) == 0


def test_kv_q4_pool_bytes(b2):
    f = b2.load().b2_kv_q4_pool_bytes
    assert f(10, 2, 12, 64) == 10 * 2 * 12 * 1280
    assert f(1 << 20, 4, 8, 128) == (1 << 20) * 4 * 8 * 2560  # past 32 bits
    assert f(10, 2, 12, 80) == 0 and f(0, 2, 12, 64) == 0


def _attn(b2, **kw):
    base = dict(dtype=b2.F16, out_dtype=b2.F16, q=16, q_row_stride=768, kv_pool=32, block_tables=48, seq_lens=64,
                key_starts=None, alibi_slopes=None, out=80, batch=4, n_head=12, n_kv_head=12, head_dim=64,
                max_blocks_per_seq=8, layer_idx=0, n_layer=1, num_blocks=100, scale=0.0, softcap=0.0, window=0, max_ctas=0)
    base.update(kw)
    return b2.PagedAttnQ4Args(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), -2), (dict(out_dtype=2), -2), (dict(head_dim=96), -6), (dict(n_kv_head=5), -3), (dict(n_head=108), -6),
    (dict(n_head=0), -3), (dict(layer_idx=1), -3), (dict(num_blocks=0), -3), (dict(batch=-1), -3), (dict(q=None), -1),
    (dict(out=None), -1), (dict(block_tables=None), -1), (dict(seq_lens=None), -1), (dict(kv_pool=None), -1),
    (dict(q=24), -4), (dict(out=88), -4), (dict(q_row_stride=760), -3), (dict(q_row_stride=772), -4),
    (dict(max_blocks_per_seq=0), -3), (dict(max_blocks_per_seq=1 << 23), -3), (dict(batch=1 << 16, max_blocks_per_seq=1 << 15), -3),
    (dict(softcap=-1.0), -3), (dict(softcap=float("nan")), -3), (dict(softcap=float("inf")), -3),
    (dict(scale=float("nan")), -3), (dict(window=-1), -3), (dict(max_ctas=-1), -3),
])
def test_attention_q4_host_checks(b2, kw, code):
    lib = b2.load()
    assert lib.b2_paged_attention_q4(ctypes.byref(_attn(b2, **kw)), None, 0, None) == code
    assert lib.b2_last_error_string().decode() != ""
    assert lib.b2_paged_attention_q4_workspace_bytes(ctypes.byref(_attn(b2, **kw))) == 0


def test_attention_q4_empty_batch_is_a_no_op(b2):
    a = _attn(b2, batch=0, q=None, kv_pool=None, out=None)
    assert b2.load().b2_paged_attention_q4(ctypes.byref(a), None, 0, None) == 0


def test_binding_refuses_tensors_off_the_device(b2):
    import torch
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        b2.block_map_args(i.view(2, 2), i, i, i, i, num_blocks=4)
    with pytest.raises(ValueError):
        b2.block_map_args(i.view(2, 2).long(), i, i, i, i, num_blocks=4)
    with pytest.raises(ValueError):
        b2.block_release_args(i.view(2, 2), i, i, i[:3], i, num_blocks=4)
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):  # the pool is too small
        b2.kv_q4_args(torch.zeros(100, dtype=torch.uint8), x, x, i, n_kv_head=2, head_dim=64, layer_idx=0, n_layer=1, num_blocks=4)


@pytest.mark.parametrize("dt", [R.F16, R.BF16])
def test_format_holds_values_to_half_a_step(dt):
    # |x - x^| <= s / 2 plus what rounding s and m to f16 takes from the range's ends: 8 * 2^-12 s (s is off by half a
    # step of f16, 2^-11 / 2 at most relative, 8 of them to an end) and 2^-11 |m| / 2 <= 2^-12 |m|.
    rng = np.random.Generator(np.random.PCG64(5))
    x = R.widen(dt, R.O.round_to(dt, rng.standard_normal(64 * 128).astype(np.float32))).reshape(64, 128)
    c, s, m = R.quantise(x)
    v = R.values(c, s, m)
    s64, m64 = (a.astype(np.float64).repeat(32, -1) for a in (s, m))
    assert np.all(np.abs(v - x) <= s64 * (0.5 + 8 * 2.0 ** -11) + np.abs(m64) * 2.0 ** -11)
    flat = np.full((1, 64), 0.25)
    c, s, m = R.quantise(flat)
    assert (s == 0).all() and (c == 8).all() and np.array_equal(R.values(c, s, m), flat)
