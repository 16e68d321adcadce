"""LabRunner.score where parameters ask for gradients, and what it refuses: before the cache holds anything new."""
from __future__ import annotations

import pytest
import torch

transformers = pytest.importorskip("transformers")

from attention_lab.qwen_wrap import LabRunner, make_state, tiny_qwen3, wrap_model  # noqa: E402


def runner(device, capacity=100):
    m = tiny_qwen3(seed=0, layers=2, hidden=256, heads=4, groups=2, head_dim=128, intermediate=256, vocab=256,
                   dtype=torch.bfloat16).to(device)
    for p in m.parameters():
        p.requires_grad_(True)
    return LabRunner(m, wrap_model(m), make_state(m, capacity, "full"))


def ids(n, device):
    return torch.randint(0, 256, (1, n), generator=torch.Generator().manual_seed(3)).to(device)


@pytest.mark.gpu
def test_parameters_that_ask_for_gradients(gpu):
    run = runner(gpu)
    r = run.score(ids(75, gpu), 32, top=3, entropy=True)
    assert run.cache.valid_length == 75 and not any(x.requires_grad for x in r)
    other = runner(gpu)
    with torch.no_grad():
        want = other.score(ids(75, gpu), 32, top=3, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.gpu
@pytest.mark.parametrize("kw,error,match", [(dict(top=65), ValueError, "top"), (dict(top=-1), ValueError, "top"),
                                            (dict(n=98), RuntimeError, "capacity"), (dict(chunk=0), ValueError, "chunk")])
def test_refused_before_the_first_chunk(gpu, kw, error, match):
    run = runner(gpu)
    n, chunk = kw.pop("n", 75), kw.pop("chunk", 32)
    with torch.no_grad():
        run.prefill(ids(3, gpu), 3)
    with pytest.raises(error, match=match):
        run.score(ids(n, gpu), chunk, **kw)
    assert run.cache.valid_length == 3
    assert run.score(ids(75, gpu), 32, top=2).logprobs.shape == (1, 74)


def test_refused_off_the_device():
    run = runner("cpu")
    with pytest.raises(ValueError, match="HIP device"):
        run.score(ids(20, "cpu"), 8)
    assert run.cache.valid_length == 0
