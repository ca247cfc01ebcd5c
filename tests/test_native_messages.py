"""Errors raised by the native module reach Python, numbers included."""

import pytest
import torch

from lmcache_ascend_b200 import ops


@pytest.mark.skipif(not ops.native_available(), reason="native module not built")
def test_message_with_a_number():
    z, t = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="bad block_size -5"):
        ops.native().build_slot_mapping(z, z, t, -5, 2, None, 10, True, None)
