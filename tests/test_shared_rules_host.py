"""The shared read's sizes that the Python side repeats from the kernel: tiles, workgroups and partials are the same numbers."""
from __future__ import annotations

import os
import re

from attention_lab import shared

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "attention-lab_amd", "csrc", "shared.hip")


def test_constants():
    with open(SOURCE) as f:
        k = {name: int(value) for name, value in re.findall(r"\b(k[A-Z]\w*) = (\d+)\b", f.read())}
    assert (shared.WIDE_ROWS, shared.NARROW_ROWS, shared.MAX_SPLITS) == (k["kWide"], k["kNarrow"], k["kMaxSplits"])
    assert shared.PART_BYTES == 4 * k["kPart"]
    for G in (16, 32):      # one tile of rows a group: the workgroups of the group, and a piece
        assert shared.shared_splits(G, 1, False) == k["kNarrowWorkers"] // G + 2 < k["kMaxSplits"]
        assert shared.shared_splits(G, 1, True) == k["kMixedWorkers"] // G + 2
        assert shared.shared_splits(G, 1, True, True) == k["kWideWorkers"] // G + 2
