"""Pools without a group: refused as a size, before a rule divides by it."""
from __future__ import annotations

import pytest
import torch

from attention_lab import shared_prefix_attention
from test_shared_host import OnDevice


def test_no_group():
    pool = torch.zeros(8, 0, 16, 128, dtype=torch.bfloat16).as_subclass(OnDevice)
    with pytest.raises(ValueError, match="at least one"):
        shared_prefix_attention(torch.zeros(3, 0, 4, 1, 128, dtype=torch.bfloat16), pool, pool, torch.zeros(3, 4, dtype=torch.int32), 20, 16)
