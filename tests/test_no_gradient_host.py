"""Reads, writes and scores without a gradient: tensors that ask for one, or carry a tangent, are refused before any launch."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from attention_lab import _native, page_append, shared_prefix_attention, token_logprobs
from attention_lab.pages import PagedCache
from test_pages_host import OnDevice, parts


def on(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


def calls():
    cache = PagedCache(**parts())
    table = torch.zeros(3, 4, dtype=torch.int32)
    pool = lambda: on(8, 2, 16, 128)  # noqa: E731
    return {
        "logits": (lambda x: token_logprobs(x), on(3, 10)),
        "q": (lambda x: shared_prefix_attention(x, pool(), pool(), table, 20), on(3, 2, 4, 1, 128)),
        "k_pages": (lambda x: shared_prefix_attention(on(3, 2, 4, 1, 128), x, pool(), table, 20), pool()),
        "v_pages": (lambda x: shared_prefix_attention(on(3, 2, 4, 1, 128), pool(), x, table, 20), pool()),
        "rows k": (lambda x: page_append(cache, 0, x, on(3, 2, 5, 128)), on(3, 2, 5, 128)),
        "rows v": (lambda x: page_append(cache, 0, on(3, 2, 5, 128), x), on(3, 2, 5, 128)),
    }


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(_native, "call_on", lambda device, entry, *args: seen.append(entry))
    monkeypatch.setattr(_native, "stream_of", lambda device: None)
    return seen


@pytest.mark.parametrize("name", list(calls()))
def test_refused(native_lib, launches, name):
    call, x = calls()[name]
    with pytest.raises(ValueError, match="no gradient"):
        call(x.clone().as_subclass(OnDevice).requires_grad_(True))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.as_subclass(torch.Tensor), torch.ones(x.shape, dtype=x.dtype)).as_subclass(OnDevice)
        assert forward_ad.unpack_dual(dual).tangent is not None
        with pytest.raises(ValueError, match="forward-mode"):
            call(dual)
    assert not launches


@pytest.mark.parametrize("name", [n for n in calls() if n != "logits"])   # those take a stream's counters, on a device
def test_taken_without(native_lib, launches, name):
    call, x = calls()[name]
    with torch.no_grad():
        call(x.clone().as_subclass(OnDevice).requires_grad_(True))
    with forward_ad.dual_level():
        call(x)
    assert len(launches) == 2
