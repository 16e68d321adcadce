"""The sparse step over an 8-bit cache where several run at once: streams, host threads, captured graphs, and a call that
fails between its launches. The score launch adds into a select state that the select launch takes out again, so steps
that shared one would choose each other's rows."""
from __future__ import annotations

import threading

import pytest
import torch

from attention_lab import QuantCache, prepare_request, quant_attention, sparse_decode_step_quant
from attention_lab import _native, decode, hip_range, hip_score, hip_select
from attention_lab.indexer import GroupedIndexer

pytestmark = pytest.mark.gpu
G, D, R = 2, 128, 32


class Step:
    """One step's inputs: its own table, queries and cache, so that another step's scores choose other rows."""

    def __init__(self, gpu, seed, B=2, h=2, C=8192, L=8001, rho=1 / 32):
        gen = torch.Generator().manual_seed(seed)
        t = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(gpu)  # noqa: E731
        self.z, self.q, self.q_pre, self.k_new = t(B, G, R, C), t(B, G, h, 1, D), t(B, G, h, 1, D), t(B, G, 1, D)
        codes = (torch.randint(0, 255, (B, G, C, D), generator=gen).to(torch.uint8) % 0x50).to(gpu)
        exps = torch.full((B, G, -(-C // 64)), 122, dtype=torch.uint8, device=gpu)
        self.cache = QuantCache(codes.view(torch.float8_e4m3fn), codes.view(torch.float8_e4m3fn), exps, exps)
        self.idx = GroupedIndexer(G, h, D, R, device=gpu, dtype=torch.bfloat16, seed=seed)
        self.req = prepare_request(B, G, C, valid_length=L, query_position=L - 1, rho=rho, device=gpu)

    def __call__(self, **kw):
        r, lay = self.req, self.req.layout
        return sparse_decode_step_quant(self.q, self.q_pre, self.cache, self.z, self.idx.wq_t_scaled, self.idx.wk,
                                        r.fixed_rows, r.off_lo, lay.candidate_lo, lay.candidate_hi, r.k,
                                        r.selected_count, k_pre_new=self.k_new, write_col=r.write_col, return_rows=True,
                                        **kw)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_every_stream_has_its_own_state(gpu):
    device = torch.device(gpu)
    held = [decode._step_workspace(device, None)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        with torch.cuda.stream(s):
            held.append(decode._step_workspace(device, None))
    assert len({id(w) for w, _ in held}) == len({id(lock) for _, lock in held}) == 3
    with torch.cuda.stream(streams[0]):
        assert decode._step_workspace(device, None)[0] is held[1][0]
    own = _native.Workspace()
    assert decode._step_workspace(device, own)[0] is own


@pytest.mark.parametrize("own_streams", [True, False])
def test_steps_from_two_threads(gpu, own_streams):
    """Each on a stream of its own, or both on one: the rows and outputs of one after the other."""
    steps = [Step(gpu, 10 + i, L=8001 - 500 * i) for i in range(2)]
    want = [s() for s in steps]
    assert not torch.equal(want[0][1][:200], want[1][1][:200])
    torch.cuda.synchronize()
    shared, failed, start = torch.cuda.Stream(), [], threading.Barrier(2)

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream() if own_streams else shared):
                start.wait(30)
                for _ in range(20):
                    got = [steps[i]() for _ in range(3)]
                torch.cuda.current_stream().synchronize()
            if not all(same(g, want[i]) for g in got):
                failed.append(f"thread {i}: another result")
        except Exception as e:  # noqa: BLE001 - a thread's exception would be lost
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("own", [False, True])
def test_captured_steps_beside_eager_ones(gpu, own):
    """Two graphs replayed on two streams with eager steps of other inputs between: nothing is shared (or, with a
    workspace of the caller's for each graph, what the caller shares)."""
    steps = [Step(gpu, 20 + i) for i in range(2)]
    other = Step(gpu, 30, B=1, L=6000)
    want, want_other = [s() for s in steps], other()
    spaces = [dict(workspace=_native.Workspace()) if own else {} for _ in steps]
    for s, kw in zip(steps, spaces):
        s(**kw)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s, kw in zip(steps, spaces):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s(**kw))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = [other() for _ in range(3)]
        torch.cuda.synchronize()
        assert all(same(o, w) for o, w in zip(outs, want)) and all(same(e, want_other) for e in eager)


def test_a_captured_step_follows_its_inputs(gpu):
    """Replays over a later table, queries and keys equal eager steps over the same."""
    a, b = Step(gpu, 40), Step(gpu, 40)
    a()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = a()
    for n in range(4):
        new = Step(gpu, 50 + n)
        for s in (a, b):
            for name in ("z", "q", "q_pre", "k_new"):
                getattr(s, name).copy_(getattr(new, name))
        g.replay()
        want = b()
        torch.cuda.synchronize()
        assert same(out, want) and torch.equal(a.z, b.z), n


@pytest.mark.parametrize("workspace", [False, True])
def test_a_step_that_fails_between_its_launches_leaves_the_state_clean(gpu, monkeypatch, workspace):
    step = Step(gpu, 60)
    kw = dict(workspace=_native.Workspace()) if workspace else {}
    want = step(**kw)
    with monkeypatch.context() as m:
        def fail(*args, **kwargs):
            raise MemoryError("no room")
        m.setattr(hip_select, "select_rows", fail)
        with pytest.raises(MemoryError):
            step(**kw)
    assert same(step(**kw), want)
    with monkeypatch.context() as m:   # the scratch is there before the table is written
        m.setattr(hip_select, "reserve", fail)
        m.setattr(hip_score, "score_grouped", lambda *a, **k: pytest.fail("scored without a scratch"))
        with pytest.raises(MemoryError):
            step(**kw)
    assert same(step(**kw), want)


def test_every_launch_goes_to_the_caches_device(gpu, monkeypatch):
    """No entry point is called without the device of its tensors made current."""
    step, seen, real = Step(gpu, 70), [], _native.call_on
    want = step()
    monkeypatch.setattr(_native, "call_on", lambda device, name, *a: (seen.append((device, name)), real(device, name, *a)))
    monkeypatch.setattr(_native, "call", lambda name, *a: pytest.fail(f"{name} on whichever device is current"))
    assert same(step(), want)
    assert {d for d, _ in seen} == {torch.device(gpu)}
    assert [n for _, n in seen] == ["attnlab_score_grouped", "attnlab_select_rows", "attnlab_quant_attend"]


def test_a_table_elsewhere_is_refused(gpu):
    step = Step(gpu, 80, C=400, L=300, rho=0.1)
    step.z = step.z.cpu()
    with pytest.raises(ValueError, match="device"):
        step()


# ---------------------------------------------------------------------------------------------------------------------
# the reads' counters and partials of a stream, to their ends
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,G,h,partitions", [
    (16, 4, 8, 16), (hip_range.COUNTERS // 2, 2, 1, 2), (hip_range.COUNTERS // 4, 4, 2, 1), (16, 4, 8, 15),
    (hip_range.COUNTERS // 2 + 1, 2, 1, 2), (43, 3, 4, 16)])
def test_reads_that_fill_the_shared_counters_and_partials(gpu, B, G, h, partitions):
    """At the last counter, at the partials' last row, and past either: the outputs of reads that are not split, and the same
    bits call after call."""
    rows, C = B * G * h * partitions, 300
    shared = partitions > 1 and B * G <= hip_range.COUNTERS and rows <= hip_range.PARTIALS
    device, stream = torch.device(gpu), torch.cuda.current_stream().cuda_stream
    assert (hip_range._split_k(partitions, B * G, h, device, stream, True)[2] is not None) == shared
    g = torch.Generator(device=gpu).manual_seed(B)
    codes = lambda: (torch.randint(0, 255, (B, G, C, D), generator=g, device=gpu) % 0x50).to(torch.uint8)  # noqa: E731
    exps = torch.full((B, G, -(-C // 32)), 122, dtype=torch.uint8, device=gpu)
    cache = QuantCache(codes().view(torch.float8_e4m3fn), codes().view(torch.float8_e4m3fn), exps, exps, block=32)
    q = torch.randn(B, G, h, 1, D, generator=g, device=gpu).to(torch.bfloat16)
    read = lambda P: quant_attention(q, cache, out_dtype=torch.float32, partitions=P)  # noqa: E731
    whole, first = read(1), read(partitions)
    # values of one sign, so an output is its own sum of magnitudes; scores below 2^3 in the log2 domain, so either side's
    # weights are good to 2^-16 + 16 * 2^-20 + 2^-22 and its sums to 2^-17: 2.6 * 2^-16, twice for weights and their sum
    assert bool(((whole - first).abs() <= 2 * 2 * 2.6 * 2.0 ** -16 * whole.abs()).all())
    for _ in range(3):
        assert torch.equal(read(partitions), first)
    buf = hip_range._MERGES.get((device.index, stream))
    assert buf is None or not buf[:hip_range.COUNTERS].any()


def test_eager_reads_on_two_streams_use_their_own_counters(gpu):
    """Merges by the last workgroup to arrive, on two streams at once."""
    B, h, C, P = 1, 4, 6000, 8
    device, g = torch.device(gpu), torch.Generator(device=gpu).manual_seed(1)
    codes = (torch.randint(0, 255, (B, G, C, D), generator=g, device=gpu) % 0x50).to(torch.uint8).view(torch.float8_e4m3fn)
    exps = torch.full((B, G, -(-C // 64)), 122, dtype=torch.uint8, device=gpu)
    cache = QuantCache(codes, codes, exps, exps)
    qs = [torch.randn(B, G, h, 1, D, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2)]
    want = [quant_attention(q, cache, partitions=P) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    counters = set()
    for s in streams:
        with torch.cuda.stream(s):
            counters.add(hip_range._split_k(P, B * G, h, device, s.cuda_stream, True)[2])
    assert None not in counters and len(counters) == 2
    for _ in range(5):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append([quant_attention(q, cache, partitions=P) for _ in range(4)])
        torch.cuda.synchronize()
        for g4, w in zip(got, want):
            assert all(torch.equal(x, w) for x in g4)
