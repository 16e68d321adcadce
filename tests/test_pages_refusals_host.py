"""Lengths to truncate to that lie in what a truncation changes: refused before any launch (the pointers are never touched)."""
from __future__ import annotations

import pytest

from attention_lab import _native

# table [16, 48), lengths [4096, 4104), refs [8192, 8224)
TRUNCATE = dict(table=16, lengths=4096, refs=8192, to=12288, length=0, S=2, W=4, pages=8, page=16, stream=None)


@pytest.mark.parametrize("to", [12, 16, 44, 4092, 4100, 8188, 8220])
def test_truncate_refuses_its_own_tensors(native_lib, to):
    with pytest.raises(ValueError, match="own tensors"):
        _native.call("attnlab_page_truncate", *dict(TRUNCATE, to=to).values())
