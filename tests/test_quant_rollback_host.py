"""The 8-bit cache's rollback without a GPU: the launches replaced by the oracle."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

pytest.importorskip("transformers")

from attention_lab import qwen_wrap  # noqa: E402
from oracle import quant as oq  # noqa: E402
from quant_rollback import B, D, G, L, Expected, append, rows, walk  # noqa: E402


@pytest.fixture
def host(monkeypatch):
    def cache(k, v, k_exp, v_exp, *, block):
        return SimpleNamespace(k=k, v=v, k_exp=k_exp, v_exp=v_exp, block=block)

    def quantize(c, k, v, start):
        for codes, exps, x in ((c.k, c.k_exp, k), (c.v, c.v_exp, v)):
            oq.append(codes.view(torch.uint8).numpy(), exps.numpy(), x.double().numpy(), start, c.block)

    @torch.inference_mode()     # the launches write by address, whatever mode the tensors were made in
    def kept(ring, k, v, start):
        quantize(ring.cache, k, v, start)
        R, T = ring.k.shape[2], k.shape[2]
        for p in range(max(start, start + T - R), start + T):
            ring.k[:, :, p % R], ring.v[:, :, p % R] = k[:, :, p - start], v[:, :, p - start]

    monkeypatch.setattr(qwen_wrap, "QuantCache", cache)
    monkeypatch.setattr(qwen_wrap, "KeptRows", lambda cache, k, v: SimpleNamespace(cache=cache, k=k, v=v))
    monkeypatch.setattr(qwen_wrap, "quantize_append", quantize)
    monkeypatch.setattr(qwen_wrap, "append_kept", kept)


def make(capacity, block):
    return qwen_wrap.LabCache(layers=L, batch=B, groups=G, capacity=capacity, head_dim=D, device="cpu",
                              dtype=torch.bfloat16, kv_format="e4m3", kv_block=block)


@pytest.mark.parametrize("seed,capacity,block", [(0, 40, 16), (1, 150, 16), (2, 150, 32), (3, 300, 16), (4, 61, 64)])
def test_writes_and_rollbacks(host, seed, capacity, block):
    taken, refused = walk(make(capacity, block), seed, 40)
    assert taken > 5 and (refused == 0 or capacity > 4 * block)


def test_a_refused_rollback_names_a_length_that_works(host):
    c, want = make(200, 16), Expected(200, 16)
    append(c, want, rows(1, 190, 0.1), rows(2, 190, 0.1))
    with pytest.raises(ValueError, match="roll back to 32"):
        c.rollback(37)
    c.rollback(32)
    want.rollback(32)
    append(c, want, rows(3, 5, 0.1), rows(4, 5, 0.1))
    want.check(c, "again")
    c.rollback(33)
    want.rollback(33)
    want.check(c, "inside the block written again")


@pytest.mark.parametrize("chunks", [(64, 64, 1), (64, 37), (1,), (64, 36, 1), (50, 50)])
def test_a_prompts_end_can_be_returned_to_from_far_away(host, chunks):
    """Whatever its last chunk's length, one token among them; again and again, and within its block."""
    c, want = make(420, 32), Expected(420, 32)
    for n, T in enumerate(chunks):
        append(c, want, rows(n, T, 0.1), rows(50 + n, T, 0.1))
    end = c.valid_length
    for n in range(2):
        for t in range(40):
            append(c, want, rows(100 + 50 * n + t, 1, 0.3), rows(300 + 50 * n + t, 1, 0.3))
        while c.valid_length < end + 200:
            append(c, want, rows(7, 1, 0.3), rows(8, 1, 0.3))
        c.rollback(end)
        want.rollback(end)
        want.check(c, f"{chunks} {n}")
    if end % 32 > 1:
        c.rollback(end - 1)
        want.rollback(end - 1)
        want.check(c, "inside the prompt's last block")


def test_a_cache_made_in_inference_mode_is_written_and_rolled_back_outside(host):
    with torch.inference_mode():
        c = make(100, 16)
    want = Expected(100, 16)
    for n, T in enumerate((21, 1, 40)):
        append(c, want, rows(n, T, 0.1), rows(50 + n, T, 0.1))
    c.rollback(21)
    want.rollback(21)
    want.check(c, "outside inference mode")


def test_kept_rows_are_no_part_of_the_cache_that_is_counted(host):
    c = make(300, 32)
    b = c.bytes()
    n = L * B * G * c.slots
    assert b["kv_bytes"] == 2 * (n * D + L * B * G * 10) and b["total_bytes"] == b["kv_bytes"] + 2 * L * B * G * 5 * 32 * 256
