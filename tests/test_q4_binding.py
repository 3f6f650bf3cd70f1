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
