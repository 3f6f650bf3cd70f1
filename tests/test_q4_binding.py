"""The Python binding's checks of the block maps' and the 4-bit pool's arguments (CPU only)."""
from __future__ import annotations

import pytest
import torch


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_block_map_refuses_a_free_list_shorter_than_the_pool(b2):
    # The device cuts free_count to num_blocks, not to the list's length: it could read past a shorter list.
    for n in (0, 1, 3):
        with pytest.raises(ValueError, match="free_list"):
            b2.block_map_args(_ints(-1, -1).view(1, 2), _ints(0), _ints(*range(n)), _ints(n), _ints(0), num_blocks=4)
    with pytest.raises(ValueError, match="device"):  # long enough: the next check
        b2.block_map_args(_ints(-1, -1).view(1, 2), _ints(0), _ints(0, 1, 2, 3), _ints(3), _ints(0), num_blocks=4)


def test_launches_refuse_arguments_of_another_device(b2, monkeypatch):
    device = 0
    monkeypatch.setattr(b2, "_current", (lambda d: 0, lambda: device))
    calls = [(b2.block_map, b2.BlockMapArgs()), (b2.block_release, b2.BlockReleaseArgs()), (b2.kv_append_q4, b2.KvQ4Args(dtype=b2.F16)),
             (b2.kv_gather_q4, b2.KvQ4Args(dtype=b2.F16)),
             (lambda a, stream=None: b2.paged_attention_q4(a, torch.empty(16, dtype=torch.uint8), stream), b2.PagedAttnQ4Args())]
    for call, args in calls:
        args.device = 1
        for stream in (None, 0):
            with pytest.raises(ValueError, match="cuda:1"):
                call(args, stream)
        device = 1
        with pytest.raises((b2.B2Error, ValueError)) as e:  # the right device: the next check
            call(args)
        assert "cuda:1" not in str(e.value)
        device = 0


def test_attention_refuses_a_workspace_that_the_kernel_cannot_use(b2, monkeypatch):
    monkeypatch.setattr(b2, "_current", (lambda d: 0, lambda: 0))

    class OnGpu:  # what the binding asks of a tensor
        def __init__(self, device=0, contiguous=True):
            self.device_index, self.contiguous = device, contiguous

        def get_device(self):
            return self.device_index

        def is_contiguous(self):
            return self.contiguous

        def data_ptr(self):
            return 16

        nbytes = 0

    args = b2.PagedAttnQ4Args()
    args.device = 0
    # host memory, another device's, an expanded tensor whose bytes it does not have
    for ws in (torch.zeros(1 << 20, dtype=torch.uint8), OnGpu(device=1), OnGpu(contiguous=False)):
        with pytest.raises(ValueError, match="workspace"):
            b2.paged_attention_q4(args, ws)
    with pytest.raises(b2.B2Error):  # the library's own checks come next
        b2.paged_attention_q4(args, OnGpu())


def test_a_single_row_may_have_any_row_stride(b2, monkeypatch):
    # A tensor's stride over one row means nothing: [heads, 1, dim] transposed has one head's.
    monkeypatch.setattr(b2, "_on_device", lambda args, *tensors: args)
    heads, dim = 4, 64
    kv = dict(n_kv_head=heads, head_dim=dim, layer_idx=0, n_layer=1, num_blocks=2)
    pool = torch.zeros(2, 1, heads, 20 * dim, dtype=torch.uint8)
    one = torch.zeros(heads, 1, dim, dtype=torch.float16).transpose(0, 1)
    wide = torch.zeros(1, 3 * heads * dim, dtype=torch.float16)[:, :heads * dim]
    assert one.shape == (1, heads, dim) and one.stride(0) == dim
    for k, v in ((one, one), (one, wide), (wide, one), (wide, wide), (one.expand(1, heads, dim), one)):
        assert b2.kv_q4_args(pool, k, v, _ints(3), **kv).row_stride == heads * dim
    two = torch.zeros(2, 3, heads, dim, dtype=torch.float16)
    assert b2.kv_q4_args(pool, two[:, 0], two[:, 1], _ints(3, 4), **kv).row_stride == 3 * heads * dim
    with pytest.raises(ValueError):  # two rows: the strides count
        b2.kv_q4_args(pool, two[:, 0], two[:, 0].contiguous(), _ints(3, 4), **kv)
    shape = dict(n_head=heads, **kv)
    out = torch.zeros(1, heads, dim, dtype=torch.float16)
    for q in (one, wide):
        assert b2.attn_q4_args(q, pool, _ints(0).view(1, 1), _ints(5), out, **shape).q_row_stride == heads * dim
    assert b2.attn_q4_args(two[:, 0], pool, _ints(0, 1).view(2, 1), _ints(5, 5), torch.zeros(2, heads, dim).half(), **shape).q_row_stride == 3 * heads * dim
