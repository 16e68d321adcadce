"""Token log probabilities on the GPU against a float64 formulation.

Tokens of the order are exact. Values, per row, with R = max x - x_token in nats: the weights' exponents are products rounded
once at a magnitude of at most R log2 e + log2 V (2^-24 of it each, and of the largest one common to all, which cancels), exp2
is within 2^-22, sums over up to 2^20 weights are 64 deep in a thread and pairwise above it (2^-17 of the sum at most: log's
absolute error), and the result is rounded once more at its own size. So a log probability is off by at most
  2^-16 + 2^-22 (R + 20)                     (nats)
and the entropy, a mean of log probabilities under weights that err by the same, by at most (1 + H) times that for R = H + 20.
"""
from __future__ import annotations

import math
import threading

import pytest
import torch

from attention_lab import token_logprobs

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def logits(seed, *shape, dtype="bf16", scale=2.5):
    return (scale * torch.randn(*shape, generator=gen(seed))).to(TYPES[dtype])


def order(x, top):
    """The first `top` tokens of each row of x: larger first, ties to the lower token, NaN last."""
    y = torch.where(torch.isnan(x), torch.tensor(float("-inf"), dtype=torch.float64), x.double())
    nan_last = torch.sort(torch.isnan(x).int(), dim=-1, stable=True).indices
    y = y.gather(-1, nan_last)
    at = torch.sort(y, dim=-1, descending=True, stable=True).indices
    return nan_last.gather(-1, at)[..., :top]


def check(x, tokens=None, top=0, entropy=True, gpu=None, dev=None):
    """x, tokens on the CPU; dev: x on the GPU where it is laid out otherwise."""
    r = token_logprobs(x.to(gpu) if dev is None else dev, None if tokens is None else tokens.to(gpu), top=top, entropy=entropy)
    V = x.shape[-1]
    y = torch.log_softmax(x.double(), dim=-1)
    some = torch.isfinite(x.double().amax(dim=-1)) & ~torch.isnan(x).any(dim=-1)
    largest = x.double().amax(dim=-1)

    def near(got, want, far):
        assert got.dtype == torch.float32 and got.shape == want.shape
        got = got.double().cpu()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
        assert ((got - want).abs() <= 2.0 ** -16 + 2.0 ** -22 * (far + 20) + 2.0 ** -23 * want.abs())[fine].all()

    if tokens is None:
        assert r.logprobs is None
    else:
        t = tokens.long()
        at = t.clamp(0, V - 1).unsqueeze(-1)
        want = torch.where(t < 0, 0.0, torch.where(t < V, y.gather(-1, at).squeeze(-1), float("nan")))
        near(r.logprobs, want, (largest - x.double().gather(-1, at).squeeze(-1)).nan_to_num(0, 0, 0).abs())
    if entropy:
        p = y.exp()
        want = torch.where(some, -(torch.where(p > 0, p * y, 0.0)).sum(dim=-1), float("nan"))
        assert torch.equal(torch.isnan(r.entropy.cpu()), torch.isnan(want))
        err = (r.entropy.double().cpu() - want).abs()[some]
        assert (err <= (1 + want[some]) * (2.0 ** -16 + 2.0 ** -22 * (want[some] + 40))).all()
    else:
        assert r.entropy is None
    best = order(x, top)
    assert r.top_tokens.dtype == torch.int64 and torch.equal(r.top_tokens.cpu(), best)
    z = x.double().gather(-1, best)
    near(r.top_logprobs, y.gather(-1, best), (largest.unsqueeze(-1) - z).nan_to_num(0, 0, 0).abs())
    return r


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 7, 7), (5, 64, 64), (1, 65, 5), (4, 255, 20), (2, 2047, 3),
                                     (2, 2049, 64), (9, 4099, 1), (3, 16384, 8), (2, 16385, 20), (1, 32003, 20), (1, 151936, 20),
                                     (64, 50257, 5), (33, 151936, 32), (700, 5003, 8), (1, 1048560, 64), (1030, 1000, 0)])
def test_sizes(gpu, dtype, N, V, top):
    x = logits(N + V, N, V, dtype=dtype)
    tokens = torch.randint(0, V, (N,), generator=gen(V))
    check(x, tokens, top, gpu=gpu)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_tokens(gpu, dtype):
    """Padding, tokens past the vocabulary, int32, none, several leading dimensions, one row without any."""
    x = logits(3, 2, 5, 331, dtype=dtype)
    tokens = torch.tensor([[0, 330, 331, -1, -100], [7, 2 ** 40, -2 ** 40, 5, 329]])
    check(x, tokens, 4, gpu=gpu)
    check(x, tokens.clamp(-9, 2 ** 31 - 1).to(torch.int32), 0, entropy=False, gpu=gpu)
    check(x, None, 3, gpu=gpu)
    check(x[0, 0], torch.tensor(17), 2, gpu=gpu)
    r = check(x[:, :0], torch.zeros(2, 0, dtype=torch.int64), 4, gpu=gpu)
    assert r.top_tokens.shape == (2, 0, 4)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [100, 4001, 20011])
def test_layouts(gpu, dtype, V):
    """Rows at every address of a 16-byte word, odd strides, repeated rows, a last dimension that is not dense."""
    base = logits(V, 12 * (V + 13) + 8, dtype=dtype)
    tokens = torch.randint(0, V, (6,), generator=gen(1))
    dev = base.to(gpu)
    for off in range(8):
        for step in (V, V + 1, V + 13):
            cut = lambda t: t.as_strided((6, V), (step, 1), off)  # noqa: E731
            check(cut(base), tokens, 9, gpu=gpu, dev=cut(dev))
    one = lambda t: t[:V].expand(6, V)  # noqa: E731
    check(one(base), tokens, 3, gpu=gpu, dev=one(dev))
    turned = lambda t: t[:6 * V].view(V, 6).t()  # noqa: E731
    check(turned(base), tokens, 3, gpu=gpu, dev=turned(dev))
    cube = lambda t: t[:8 * V].view(2, 4, V)[:, 1:]  # noqa: E731
    check(cube(base), tokens.view(2, 3), 3, gpu=gpu, dev=cube(dev))


def test_past_the_row_is_not_read(gpu):
    """What lies before and behind the rows reaches no output: NaN and infinities there."""
    for V, off in ((37, 3), (2051, 5), (16389, 1)):
        x = logits(V, 4, V)
        for bad in (float("nan"), float("inf")):
            dev = torch.full((4 * (V + 9) + off,), bad, dtype=torch.bfloat16, device=gpu).as_strided((4, V), (V + 9, 1), off)
            dev.copy_(x)
            check(x, torch.arange(4), 5, gpu=gpu, dev=dev)


@pytest.mark.parametrize("dtype,N,V", [("bf16", 1, 6138), ("f16", 1, 6142), ("bf16", 64, 57342), ("f16", 64, 6140),
                                       ("f32", 1, 14334), ("f32", 64, 28671)])
def test_row_that_ends_before_the_last_segment(gpu, dtype, N, V):
    """A row of which an aligned word that it only partly fills is the last one before the last segment, which is kept for rows that
    begin inside a word: what is behind the row reaches no output."""
    x = logits(V, N, V, dtype=dtype)
    stride = (V + 31) // 16 * 16
    for bad in (float("nan"), float("inf"), 60000.0):
        dev = torch.full((N, stride), bad, dtype=x.dtype, device=gpu)[:, :V]
        dev.copy_(x)
        check(x, torch.arange(N), 5, gpu=gpu, dev=dev)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [500, 30011, 151936])
def test_masked_and_special(gpu, dtype, V):
    """Masks of -inf and of the type's lowest value, whole rows of them, infinities, NaN, zeros of both signs, huge logits."""
    low = torch.finfo(TYPES[dtype]).min
    high = torch.finfo(TYPES[dtype]).max
    x = logits(V, 14, V, dtype=dtype)
    x[0, 3:] = float("-inf")
    x[1, 1:V // 2] = float("-inf")
    x[2] = float("-inf")
    x[3, 2:] = low
    x[4] = low
    x[5, 7] = float("inf")
    x[6, V // 2:] = float("nan")
    x[7] = float("nan")
    x[8] = 0.0
    x[8, ::2] = -0.0
    x[9] = high
    x[10, V - 1] = high
    x[11] = low
    x[11, V // 3] = float("-inf")
    x[12] = x[12].abs() * (high / 64 if dtype != "f16" else 100)
    x[13, :V - 2] = float("-inf")
    tokens = torch.tensor([1, 0, 5, 1, 2, 7, 0, 1, 3, 4, V - 1, V // 3, 8, V - 1])
    check(x, tokens, 20, gpu=gpu)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("seed,N,V,scale", [(2269, 130, 4826, 1000.0), (4, 200, 30011, 20.0), (5, 90, 151936, 300.0)])
def test_peaks_far_above_the_first_logits(gpu, dtype, seed, N, V, scale):
    """Rows whose few likely logits lie up to 88 above a wave's first ones: entropies near 0 keep their absolute accuracy."""
    check(logits(seed, N, V, dtype=dtype, scale=scale), torch.arange(N), 7, gpu=gpu)
    x = logits(seed + 1, N, V, dtype=dtype)
    x[torch.arange(N), 2048 + 21 * torch.arange(N)] += torch.arange(N).to(x.dtype) % 90
    check(x, torch.arange(N), 3, gpu=gpu)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ties(gpu, dtype):
    """Few different values: the order is by token where logits are equal, within a thread, a wave, a segment and across them."""
    for V in (300, 20000, 151936):
        x = torch.randint(0, 3, (3, V), generator=gen(V)).to(TYPES[dtype])
        check(x, torch.tensor([0, 1, 2]), 64, gpu=gpu)
        x = torch.full((2, V), -1.5, dtype=TYPES[dtype])
        x[1, V - 3] = 2.0
        check(x, torch.tensor([0, V - 3]), 33, gpu=gpu)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_crowded(gpu, dtype):
    """The largest logits all with a few threads, more of them than a workgroup ranks in LDS, rising and falling rows."""
    V, per = 151936, 4 if dtype == "f32" else 8
    t = torch.arange(V)
    thread = t // per % 256
    x = logits(5, 4, V, dtype="f32")
    x[0] += torch.where(thread % 64 < 3, 40.0, 0.0)
    x[1] += torch.where(thread < 12, 40.0, 0.0)
    x[2] = t / 1000.0
    x[3] = -t / 1000.0
    check(x.to(TYPES[dtype]), torch.tensor([0, 5, V - 1, 0]), 64, gpu=gpu)
    check(x[:1].to(TYPES[dtype]), torch.tensor([0]), 64, gpu=gpu)


def test_graph_and_streams(gpu):
    """Captured and replayed with other logits and eager calls between; two graphs, two streams and two host threads at once."""
    V = 20011
    xs = [logits(i, 6, V).to(gpu) for i in range(2)]
    tokens = [torch.randint(0, V, (6,), generator=gen(i)).to(gpu) for i in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for x, t in zip(xs, tokens):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(token_logprobs(x, t, top=7, entropy=True))
        graphs.append(g)
    for step in range(4):
        fresh = [logits(10 + 2 * step + i, 6, V) for i in range(2)]
        want = [token_logprobs(f.to(gpu), t, top=7, entropy=True) for f, t in zip(fresh, tokens)]
        for x, f in zip(xs, fresh):
            x.copy_(f)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(gpu) for _ in graphs]
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))
    results = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(gpu)):
            for _ in range(20):
                results[i] = token_logprobs(xs[i], tokens[i], top=7, entropy=True)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for got, w in zip(results, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_long_rows_past_32_bits(gpu):
    """More logits than 2^31: the last row's are its own."""
    V, N = 151936, 14200
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=gpu)
    row = logits(1, V)
    x[N - 1].copy_(row)
    r = token_logprobs(x, torch.full((N,), 5, device=gpu), top=3, entropy=True)
    one = token_logprobs(row.to(gpu), torch.tensor(5, device=gpu), top=3, entropy=True)
    assert torch.equal(r.top_tokens[N - 1], one.top_tokens) and r.top_tokens[0].tolist() == [0, 1, 2]
    assert abs(float(r.logprobs[N - 1]) - float(one.logprobs)) <= 2.0 ** -14
    assert abs(float(r.logprobs[0]) + math.log(V)) <= 2.0 ** -14 and abs(float(r.entropy[0]) - math.log(V)) <= 2.0 ** -13
