"""The 8-bit cache's rollback on the GPU: discarded rows leave no mark on the rows before them."""
from __future__ import annotations

import copy
import random

import pytest
import torch

pytest.importorskip("transformers")

from attention_lab import QuantCache, quantize_append  # noqa: E402
from attention_lab.quant import KeptRows, append_kept  # noqa: E402
from attention_lab.qwen_wrap import LabCache, LabRunner, LabState, make_state, tiny_qwen3, wrap_model  # noqa: E402
from quant_rollback import B, D, G, L, Expected, append, rows, walk  # noqa: E402
from test_gpu_quant import bytes_of, randn, random_cache  # noqa: E402

pytestmark = pytest.mark.gpu


def make(gpu, capacity, block):
    return LabCache(layers=L, batch=B, groups=G, capacity=capacity, head_dim=D, device=gpu, dtype=torch.bfloat16,
                    kv_format="e4m3", kv_block=block)


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("C,R,start,T", [(200, 64, 0, 200), (200, 64, 37, 1), (200, 128, 130, 3), (90, 64, 63, 27),
                                         (300, 192, 5, 290), (64, 64, 0, 64), (17, 16, 16, 1)])
def test_kept_rows_are_the_last_ones(gpu, block, C, R, start, T):
    """The codes and scales are quantize_append's; position p's row lies in slot p % R, and other slots keep theirs."""
    b, g = 2, 3
    got, want = random_cache(gpu, 1, b, g, C, block)[0], random_cache(gpu, 1, b, g, C, block)[0]
    k, v = randn(2, b, g, T, 128), randn(3, b, g, T, 128)
    k[0, 0, 0, 5], v[1, 2, T - 1, 7] = float("inf"), float("nan")
    rings = [randn(4 + i, b, g, R, 128).to(gpu) for i in range(2)]
    expect = [r.clone() for r in rings]
    append_kept(KeptRows(got, *rings), k.to(gpu).transpose(1, 2).contiguous().transpose(1, 2), v.to(gpu), start)
    quantize_append(want, k.to(gpu), v.to(gpu), start)
    for p in range(max(start, start + T - R), start + T):
        for e, x in zip(expect, (k, v)):
            e[:, :, p % R] = x[:, :, p - start].to(gpu)
    for name in ("k", "v", "k_exp", "v_exp"):
        assert (bytes_of(getattr(got, name)) == bytes_of(getattr(want, name))).all(), name
    for r, e in zip(rings, expect):
        assert torch.equal(torch.nan_to_num(r, nan=-99.0), torch.nan_to_num(e, nan=-99.0))


def test_kept_rows_refusals(gpu):
    cache = QuantCache.empty(1, 2, 64, block=16, device=gpu)
    x = randn(1, 1, 2, 3, 128).to(gpu)
    ring = torch.zeros(1, 2, 32, 128, dtype=torch.bfloat16, device=gpu)
    kept = KeptRows(cache, ring, ring.clone())
    for call, match in ((lambda: append_kept(kept, x.float(), x.float(), 0), "bfloat16"),
                        (lambda: append_kept(kept, x, x, 62), "outside"),
                        (lambda: append_kept(kept, x[:, :1], x[:, :1], 0), "must be"),
                        (lambda: KeptRows(cache, ring, ring.float()), "kept rows"),
                        (lambda: KeptRows(cache, ring, ring[:, :, :16]), "kept rows"),
                        (lambda: KeptRows(cache, ring[:, :, :0], ring[:, :, :0]), "R >= 1")):
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("block", [16, 32, 64])
def test_a_discarded_loud_row_leaves_no_mark(gpu, block):
    """A row 2^9 louder, inside a block: it raises the block's scale and rounds the quiet rows before it again. After the
    rollback codes and scale bytes are what they were, and later quiet rows are quantised as if it had never come."""
    c, want = make(gpu, 200, block), Expected(200, block)
    append(c, want, rows(1, block + 5, 0.0), rows(2, block + 5, 0.0))
    before = {n: c._store[n].clone() for n in ("k", "v", "k_exp", "v_exp")}
    loud = rows(3, 1, 0.0) * 512
    append(c, want, loud, loud)
    assert (c._store["k_exp"][..., 1] > before["k_exp"][..., 1]).all()
    n = block + 5
    assert not torch.equal(c._store["v"].view(torch.uint8)[:, :, :, :n], before["v"].view(torch.uint8)[:, :, :, :n])
    c.rollback(n)
    want.rollback(n)
    for x in "kv":
        assert torch.equal(c._store[x].view(torch.uint8)[:, :, :, :n], before[x].view(torch.uint8)[:, :, :, :n])
        assert torch.equal(c._store[x + "_exp"], before[x + "_exp"])
    append(c, want, rows(4, 7, 0.0), rows(5, 7, 0.0))
    want.check(c, "quiet rows behind the rollback")


@pytest.mark.parametrize("seed,capacity,block", [(10, 40, 16), (11, 150, 16), (12, 150, 32), (13, 300, 16), (14, 400, 64),
                                                 (15, 97, 32)])
def test_writes_and_rollbacks(gpu, seed, capacity, block):
    taken, _ = walk(make(gpu, capacity, block), seed, 48)
    assert taken > 5


def test_a_cache_made_in_inference_mode_is_written_and_rolled_back_outside(gpu):
    with torch.inference_mode():
        c = make(gpu, 100, 16)
    want = Expected(100, 16)
    for n, T in enumerate((21, 1, 40)):
        append(c, want, rows(n, T, 0.1), rows(50 + n, T, 0.1))
    for to in (21, 19):
        c.rollback(to)
        want.rollback(to)
        want.check(c, "outside inference mode")


def test_a_clone_takes_its_own_rows_back(gpu):
    c, want = make(gpu, 120, 32), Expected(120, 32)
    append(c, want, rows(1, 37, 0.2), rows(2, 37, 0.2))
    other, other_want = c.clone(), copy.deepcopy(want)
    for i in range(3):
        append(c, want, rows(10 + i, 1, 1.0), rows(20 + i, 1, 1.0))
        append(other, other_want, rows(30 + i, 20, 0.5), rows(40 + i, 20, 0.5))
    for x, w, to in ((c, want, 38), (other, other_want, 50), (c, want, 37)):
        x.rollback(to)
        w.rollback(to)
        w.check(c, "the cache") if x is c else w.check(other, "its clone")
    want.check(c, "the cache, after its clone went back")


@pytest.mark.parametrize("mode,kw", [("full", {}), ("window", dict(window=30, sinks=4)), ("sparse", {}),
                                     ("sparse", dict(selector="recent"))])
@pytest.mark.parametrize("prompt,tokens", [(100, 5), (75, 60)])
def test_the_same_tokens_after_a_rollback_give_the_same_logits(gpu, mode, kw, prompt, tokens):
    """Tokens that were decoded and discarded, other ones first: bit for bit the logits of a run without them."""
    m = tiny_qwen3(seed=0, layers=2, hidden=256, heads=4, groups=2, head_dim=128, intermediate=256, vocab=256,
                   dtype=torch.bfloat16).to(gpu)
    rng = random.Random(prompt)
    ids = torch.tensor([[rng.randrange(256) for _ in range(prompt + 2 * tokens)]], device=gpu)
    with torch.inference_mode():
        holder = wrap_model(m)
        st = make_state(m, 160, mode, kv_format="e4m3", kv_block=32, **kw)
        run = LabRunner(m, holder, st)
        run.prefill(ids[:, :prompt], 50)
        if mode == "sparse":
            st.begin_request(0.25)
        branch = st.cache.clone()
        other = LabState(branch, st.indexers, mode=mode, **kw)
        second = LabRunner(m, holder, other)
        if mode == "sparse":
            other.begin_request(0.25)
        want = [second.step(ids[:, prompt + t:prompt + t + 1]) for t in range(tokens)]
        for t in range(tokens):
            run.step(ids[:, prompt + tokens + t:prompt + tokens + t + 1])
        run.rollback(prompt)
        for t in range(tokens):
            assert torch.equal(run.step(ids[:, prompt + t:prompt + t + 1]), want[t]), t
