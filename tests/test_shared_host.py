"""Attention over shared prompts without a GPU: what the C entry and its Python caller refuse before any launch."""
from __future__ import annotations

import pytest
import torch

import attention_lab
from attention_lab import _native, shared, shared_prefix_attention

ARGS = dict(q=16, k=16, v=16, pages=8, page=16, table=16, stride=4, W=4, lengths=None, length=20, prefixes=None, prefix=16, runs=None,
            R=1, B=3, G=2, h=4, T=1, scale=0.1, wide=0, ns=1, no=1, out=16, part=16, part_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(B=0), "positive"), (dict(G=0), "positive"), (dict(T=-1), "T"), (dict(h=0), "h=0"), (dict(h=17), "h=17"),
    (dict(page=24), "power of two"), (dict(page=0), "power of two"), (dict(page=1 << 17), "power of two"), (dict(pages=0), "positive"),
    (dict(W=0), "positive"), (dict(W=1 << 27, stride=1 << 27), "2\\^31"), (dict(pages=1 << 27), "2\\^31"), (dict(length=-1), "length"),
    (dict(prefix=-1), "prefix"), (dict(R=0), "runs"), (dict(R=2), "runs"), (dict(ns=-1), "splits"), (dict(ns=65), "splits"),
    (dict(no=0), "splits"), (dict(no=65), "splits"), (dict(q=None), "required"), (dict(k=None), "required"), (dict(out=None), "required"),
    (dict(table=None), "required"), (dict(stride=3), "required"), (dict(q=24), "aligned"), (dict(v=8), "aligned"),
    (dict(part=None), "part"), (dict(part=8), "part"), (dict(part_bytes=100), "part"), (dict(B=1 << 20, T=1 << 12, ns=0), "too many"),
])
def test_refused_before_any_launch(native_lib, change, match):
    assert len(ARGS) == len(_native.SIGNATURES["attnlab_shared_prefix_attend"][1])
    with pytest.raises(ValueError, match=match):
        _native.call("attnlab_shared_prefix_attend", *dict(ARGS, **change).values())


def test_nothing_to_do_is_no_launch(native_lib):
    _native.call("attnlab_shared_prefix_attend", *dict(ARGS, T=0, q=None, part=None).values())


def test_part_bytes(native_lib):
    size = native_lib.attnlab_shared_part_bytes
    assert size(3, 2, 4, 5, 2, 1) == 120 * (8 + 3 * 132 * 4) and size(3, 2, 4, 5, 0, 1) == 0
    assert size(1, 1, 1, 3, 2, 2) == 32 + 3 * 4 * 132 * 4   # the counts' room is a multiple of 16 bytes
    assert size(0, 2, 4, 5, 1, 1) == size(1, 2, 4, -1, 1, 1) == size(1, 1, 1, 1, -1, 1) == size(1, 1, 1, 1, 1, 0) == -1


def test_split_rules():
    for rows in (1, 16, 17, 300, 5000):
        for G in (1, 8):
            for wide in (False, True):
                assert 1 <= shared.shared_splits(G, rows, wide) <= shared.MAX_SPLITS
        for keys in (1, 255, 512, 32768):
            assert 1 <= shared.own_splits(8, rows, keys) <= max(1, keys // 256)


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on a HIP device: for the checks, which look no further."""
    is_cuda = True


def test_python_makes_the_part_buffer(native_lib, monkeypatch):
    """The Python side's part buffer is what the C side asks for."""
    seen = []
    monkeypatch.setattr(_native, "call_on", lambda device, entry, *args: seen.append(args))
    monkeypatch.setattr(_native, "stream_of", lambda device: None)
    pool = torch.zeros(8, 2, 16, 128, dtype=torch.bfloat16).as_subclass(OnDevice)
    for B, h, T, prefix, partitions in ((3, 4, 1, 32, None), (3, 4, 5, 32, None), (1, 1, 1, 0, None), (5, 7, 1, 16, (64, 64)),
                                        (1, 1, 3, 16, (0, 2)), (2, 3, 1, 16, (0, 1))):
        q = torch.zeros(B, 2, h, T, 128, dtype=torch.bfloat16).as_subclass(OnDevice)
        shared_prefix_attention(q, pool, pool, torch.zeros(B, 4, dtype=torch.int32), 60, prefix, partitions=partitions)
        args = dict(zip(ARGS, seen.pop()))
        assert args["part_bytes"] == native_lib.attnlab_shared_part_bytes(B, 2, h, T, args["ns"], args["no"])


def test_python_refuses():
    pool = torch.zeros(8, 2, 16, 128, dtype=torch.bfloat16).as_subclass(OnDevice)
    q = torch.zeros(3, 2, 4, 1, 128, dtype=torch.bfloat16)
    ints = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    good = dict(q=q, k_pages=pool, v_pages=pool, block_table=ints(3, 4), lengths=20, prefix_lengths=16, runs=None, partitions=None)
    for change, match in (
        (dict(k_pages=torch.zeros(8, 2, 16, 128, dtype=torch.bfloat16)), "HIP device"), (dict(k_pages=pool.float()), "k_pages"),
        (dict(k_pages=pool[:, :, :, :64]), "k_pages"), (dict(v_pages=pool[:4]), "v_pages"), (dict(q=q[:, :1]), "q must"),
        (dict(q=q[:, :, :, 0]), "q must"), (dict(q=q.float()), "q must"),
        (dict(q=torch.zeros(3, 2, 17, 1, 128, dtype=torch.bfloat16)), "h=17"),
        (dict(q=q[:0], block_table=ints(0, 4)), "at least one"),
        (dict(k_pages=pool[:, :, :12].contiguous().as_subclass(OnDevice), v_pages=pool[:, :, :12].contiguous()), "power of two"),
        (dict(block_table=ints(2, 4)), "block_table"), (dict(block_table=ints(4, 3).t()[:3]), "block_table"),
        (dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), "block_table"), (dict(lengths=-1), "lengths"),
        (dict(lengths=2 ** 31), "lengths"), (dict(lengths=ints(2)), "int32"), (dict(lengths=torch.zeros(3)), "int32"),
        (dict(prefix_lengths=-1), "prefix_lengths"), (dict(prefix_lengths=ints(2)), "int32"), (dict(runs=ints(1)), "runs"),
        (dict(runs=torch.zeros(2, dtype=torch.int64)), "runs"), (dict(partitions=(65, 1)), "partitions"),
        (dict(partitions=(1, 0)), "partitions"),
    ):
        with pytest.raises(ValueError, match=match):
            shared_prefix_attention(**dict(good, **change))
    assert "shared_prefix_attention" in attention_lab.__all__
