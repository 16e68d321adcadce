"""The 8-bit cache and the windowed read where a model meets them: the sparse decode step over an 8-bit cache, and the
Qwen3 wrapper with kv_format "e4m3" and with mode "window", on a bf16 tiny Qwen3 with head_dim 128.

The windowed wrapper is compared with the unmodified model on the CPU under the same mask (the wrapper tests' bf16
tolerances); the 8-bit one with its own full read where they must agree, with the bfloat16 cache where rounding bounds
them, and by what a read must not see.
"""
from __future__ import annotations

import copy
import math

import numpy as np
import pytest
import torch

from attention_lab import QuantCache, dequantize_rows, prepare_request, sparse_decode_step_kernel, sparse_decode_step_quant
from attention_lab.indexer import GroupedIndexer
from oracle import quant as oq

transformers = pytest.importorskip("transformers")

from attention_lab.qwen_wrap import (LabCache, LabRunner, LabState, make_cache, make_state, tiny_qwen3,  # noqa: E402
                                     wrap_model)

pytestmark = pytest.mark.gpu
VOCAB = 256


def codes(gpu, seed, *shape):
    x = torch.randint(0, 255, shape, generator=torch.Generator().manual_seed(seed)).to(torch.uint8)
    return ((x & 128) | (x & 127) % 0x50).to(gpu)     # magnitudes up to 7.5


def f64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,h,C,L,rho", [(1, 2, 4096, 4000, 1 / 32), (2, 4, 2120, 2119, 1 / 8), (1, 1, 304, 300, 1.0),
                                         (2, 2, 80, 60, 1 / 4), (1, 8, 40000, 39001, 1 / 64)])
@pytest.mark.parametrize("canonical", [False, True])
def test_sparse_step_selects_as_the_bfloat16_step_and_reads_the_codes(gpu, dtype, B, h, C, L, rho, canonical):
    """Row list and z column are bit for bit those of sparse_decode_step_kernel on the same table (whose K/V play no
    part in them); the output is the oracle's over the listed values: bf16, half a step, and weights good to 2^-15."""
    G, r, d = 2, 32, 128
    gen = torch.Generator().manual_seed(C)
    t = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    idx = GroupedIndexer(G, h, d, r, device=gpu, dtype=dtype, seed=3)
    q, q_pre = t(B, G, h, 1, d).to(torch.bfloat16).to(gpu), t(B, G, h, 1, d).to(dtype).to(gpu)
    k_new = t(B, G, 1, d).to(dtype).to(gpu)
    z1 = t(B, G, r, C).to(dtype).to(gpu)
    z2 = z1.clone()
    kc, vc = codes(gpu, 1, B, G, C, d), codes(gpu, 2, B, G, C, d)
    e = torch.randint(120, 126, (B, G, -(-C // 32)), generator=gen).to(torch.uint8).to(gpu)
    cache = QuantCache(kc.view(torch.float8_e4m3fn), vc.view(torch.float8_e4m3fn), e, e, block=32)
    kb, vb = dequantize_rows(cache)
    req = prepare_request(B, G, C, valid_length=L, query_position=L - 1, rho=rho, device=gpu)
    lay = req.layout
    args = (req.fixed_rows, req.off_lo, lay.candidate_lo, lay.candidate_hi, req.k, req.selected_count)
    kw = dict(k_pre_new=k_new, write_col=req.write_col, canonical_order=canonical)
    _, want_rows = sparse_decode_step_kernel(q, q_pre, kb, vb, z1, idx.wq_t_scaled, idx.wk, *args, return_rows=True, **kw)
    out, rows = sparse_decode_step_quant(q, q_pre, cache, z2, idx.wq_t_scaled, idx.wk, *args, return_rows=True, **kw)
    alone = sparse_decode_step_quant(q, q_pre, cache, z2, idx.wq_t_scaled, idx.wk, *args, **kw)
    assert torch.equal(rows, want_rows)
    assert torch.equal(z1, z2)
    pos = (rows.view(B, G, -1) - req.offsets).cpu().numpy()
    qf, kf, vf = f64(q)[:, :, :, 0], f64(kb), f64(vb)
    want = oq.listed_attention(qf, kf, vf, pos, 1 / math.sqrt(d))[:, :, :, None]
    A = oq.listed_attention(qf, kf, np.abs(vf), pos, 1 / math.sqrt(d))[:, :, :, None]
    for got in (out, alone):
        assert (np.abs(f64(got) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * A).all()


def test_sparse_step_refusals(gpu):
    G, d = 2, 128
    cache = QuantCache.empty(1, G, 400, device=gpu)
    idx = GroupedIndexer(G, 2, d, 32, device=gpu, dtype=torch.bfloat16, seed=3)
    q = torch.zeros(1, G, 2, 1, d, dtype=torch.bfloat16, device=gpu)
    z = torch.zeros(1, G, 32, 400, dtype=torch.bfloat16, device=gpu)
    req = prepare_request(1, G, 400, valid_length=300, query_position=299, rho=0.1, device=gpu)
    lay = req.layout
    args = (req.fixed_rows, req.off_lo, lay.candidate_lo, lay.candidate_hi, req.k, req.selected_count)
    w = (idx.wq_t_scaled, idx.wk)
    for call, match in (
            (lambda: sparse_decode_step_quant(q.expand(1, G, 2, 2, d), q, cache, z, *w, *args), "one new query"),
            (lambda: sparse_decode_step_quant(q, q, cache, z[..., :392].contiguous(), *w, *args), "matching the cache"),
            (lambda: sparse_decode_step_quant(q, q, cache, z, *w, req.fixed_rows + 1, *args[1:]), "fixed_rows"),
            (lambda: sparse_decode_step_quant(q, q, cache, z, *w, *args, k_pre_new=q[:, :, :1, 0], write_col=100),
             "write_col"),
            (lambda: sparse_decode_step_quant(q, q[:, :, :1], cache, z, *w, *args), "elements")):
        with pytest.raises(ValueError, match=match):
            call()


def test_a_refused_sparse_step_leaves_the_table(gpu):
    """The read's own refusals come before the new key's column is written."""
    G, d = 2, 128
    cache = QuantCache.empty(1, G, 400, device=gpu)
    req = prepare_request(1, G, 400, valid_length=300, query_position=299, rho=0.1, device=gpu)
    lay = req.layout
    args = (req.fixed_rows, req.off_lo, lay.candidate_lo, lay.candidate_hi, req.k, req.selected_count)
    for h, dtype, kw, match in ((2, torch.float32, {}, "bfloat16"), (2, torch.bfloat16, dict(partitions=257), "partitions"),
                                (9, torch.bfloat16, {}, "h <= 8")):
        idx = GroupedIndexer(G, h, d, 32, device=gpu, dtype=torch.bfloat16, seed=3)
        q = torch.ones(1, G, h, 1, d, dtype=torch.bfloat16, device=gpu)
        z = torch.zeros(1, G, 32, 400, dtype=torch.bfloat16, device=gpu)
        with pytest.raises(ValueError, match=match):
            sparse_decode_step_quant(q.to(dtype), q, cache, z, idx.wq_t_scaled, idx.wk, *args, k_pre_new=q[:, :, :1, 0],
                                     write_col=299, **kw)
        assert not z.any()


# ---------------------------------------------------------------------------------------------------------------------
# the wrapper
# ---------------------------------------------------------------------------------------------------------------------
def tiny_pair(gpu, seed=0):
    cpu = tiny_qwen3(seed=seed, layers=2, hidden=256, heads=4, groups=2, head_dim=128, intermediate=256, vocab=VOCAB,
                     dtype=torch.bfloat16)
    return copy.deepcopy(cpu).to(gpu), cpu


def token_ids(n, seed=0):
    return torch.randint(0, VOCAB, (1, n), generator=torch.Generator().manual_seed(1000 + seed))


def poison_unwritten(cache):
    L = cache.valid_length
    for l in range(cache.layers):
        for t in (cache.k[l], cache.v[l]):
            if cache.quant is not None:
                t.view(torch.uint8)[:, :, L:] = 0x7f
            else:
                t[:, :, L:] = float("nan")
        if cache.z is not None:
            cache.z[l][..., L:] = float("nan")


def close(a, b, atol, rel, what):
    a, b = a.detach().float().cpu(), b.detach().float().cpu()
    assert torch.isfinite(a).all(), what
    d = (a - b).abs()
    r = float(d.norm() / b.norm())
    assert float(d.max()) <= atol and r <= rel, f"{what}: max {float(d.max()):.3e} rel {r:.3e}"


@pytest.mark.parametrize("L,window,sinks,chunk", [(40, 64, 4, 40), (150, 32, 4, 150), (150, 32, 0, 37), (97, 1, 2, 50)])
def test_window_mode_is_the_model_under_that_mask(gpu, L, window, sinks, chunk):
    m, ref_model = tiny_pair(gpu)
    ids = token_ids(L + 4)
    T = L + 4
    i, j = torch.arange(T).view(-1, 1), torch.arange(T).view(1, -1)
    seen = (j <= i) & ((j > i - window) | (j < sinks))
    mask = torch.zeros(1, 1, T, T, dtype=torch.bfloat16).masked_fill_(~seen, torch.finfo(torch.bfloat16).min)
    with torch.inference_mode():
        ref = ref_model(ids, attention_mask={"full_attention": mask}).logits
        run = LabRunner(m, wrap_model(m), make_state(m, T + 8, "window", window=window, sinks=sinks))
        poison_unwritten(run.cache)
        got = [run.prefill(ids[:, :L].to(gpu), chunk, keep_logits=True)]
        for t in range(L, T):
            got.append(run.step(ids[:, t:t + 1].to(gpu)))
    close(torch.cat(got, dim=1), ref, 5e-2, 2e-2, "windowed wrapper")


def test_window_mode_over_the_whole_history_is_the_full_mode(gpu):
    m, _ = tiny_pair(gpu)
    ids = token_ids(90).to(gpu)
    with torch.inference_mode():
        holder = wrap_model(m)
        a = LabRunner(m, holder, make_state(m, 100, "full"))
        b = LabRunner(m, holder, make_state(m, 100, "window", window=100))
        close(a.prefill(ids, 32, keep_logits=True), b.prefill(ids, 32, keep_logits=True), 2e-2, 1e-2, "prefill")
        close(a.step(ids[:, :1]), b.step(ids[:, :1]), 2e-2, 1e-2, "step")


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("chunk", [200, 64, 45])
def test_8bit_cache_holds_the_bfloat16_caches_rows(gpu, block, chunk):
    """Layer 0's K/V do not depend on any read: the values are the bfloat16 cache's, each off by half a step of e4m3
    (2^-4 of the value, or 2^-10 of the block's scale among the subnormals), and by a second rounding where a later
    chunk moved them."""
    m, _ = tiny_pair(gpu)
    L = 200
    ids = token_ids(L).to(gpu)
    with torch.inference_mode():
        holder = wrap_model(m)
        a = LabRunner(m, holder, make_state(m, L + 10, "full"))
        b = LabRunner(m, holder, make_state(m, L + 10, "full", kv_format="e4m3", kv_block=block))
        poison_unwritten(b.cache)
        la, lb = a.prefill(ids, chunk, keep_logits=True), b.prefill(ids, chunk, keep_logits=True)
    k, v = dequantize_rows(b.cache.quant[0], 0, L, dtype=torch.float32)
    for got, want, e in ((k, a.cache.k[0], b.cache._store["k_exp"][0]), (v, a.cache.v[0], b.cache._store["v_exp"][0])):
        scale = torch.exp2(e.float() - 127).repeat_interleave(block, dim=2)[:, :, :L, None]
        w = want[:, :, :L].float()
        assert bool(((got - w).abs() <= 2.0 ** -4 * w.abs() + 2 * 2.0 ** -10 * scale).all())
    # the logits of the two runs: e4m3's rms rounding is about 2.6 % of K and V, a few layers' worth of it
    rel = float((la.float() - lb.float()).norm() / la.float().norm())
    assert torch.isfinite(lb).all() and rel < 0.2, rel
    assert b.cache.bytes()["kv_bytes"] < 0.51 * a.cache.bytes()["kv_bytes"]


@pytest.mark.parametrize("selector", ["index", "recent", "uniform"])
def test_8bit_sparse_reading_everything_is_the_8bit_full_read(gpu, selector):
    m, _ = tiny_pair(gpu)
    L = 150
    ids = token_ids(L + 3).to(gpu)
    with torch.inference_mode():
        holder = wrap_model(m)
        full = LabRunner(m, holder, make_state(m, L + 8, "full", kv_format="e4m3"))
        sp = LabRunner(m, holder, make_state(m, L + 8, "sparse", selector=selector, kv_format="e4m3"))
        poison_unwritten(full.cache)
        poison_unwritten(sp.cache)
        assert torch.equal(full.prefill(ids[:, :L], 64), sp.prefill(ids[:, :L], 64))
        sp.state.begin_request(1.0, k0=L + 8)
        for t in range(3):
            close(sp.step(ids[:, L + t:L + t + 1]), full.step(ids[:, L + t:L + t + 1]), 2e-2, 1e-2, f"step {t}")


def test_8bit_unselected_rows_are_never_read(gpu):
    m, _ = tiny_pair(gpu)
    L = 300
    ids = token_ids(L + 1).to(gpu)
    with torch.inference_mode():
        holder = wrap_model(m)
        run = LabRunner(m, holder, make_state(m, L + 8, "sparse", kv_format="e4m3", canonical_order=True))
        run.prefill(ids[:, :L], 128)
        run.state.begin_request(1 / 16)
        run.state.record_selection = True
        want = run.step(ids[:, L:])
        rows = [r.clone() for r in run.state.last_rows]
        run.rollback(L)
        for l in range(run.cache.layers):
            B, G = run.cache.batch, run.cache.groups
            keep = torch.zeros(B * G * run.cache.slots, dtype=torch.bool, device=gpu)
            keep[rows[l]] = True
            keep[(torch.arange(B * G, device=gpu) * run.cache.slots + L)] = True      # the new row
            drop = ~keep.view(B, G, run.cache.slots)
            for t in (run.cache.k[l], run.cache.v[l]):
                t.view(torch.uint8)[drop] = 0x7f
        got = run.step(ids[:, L:])
    assert torch.equal(got, want)


@pytest.mark.parametrize("mode,kw", [("full", {}), ("window", dict(window=30, sinks=4)), ("sparse", {})])
def test_8bit_rollback_and_clone(gpu, mode, kw):
    m, _ = tiny_pair(gpu)
    ids = token_ids(140).to(gpu)
    with torch.inference_mode():
        holder = wrap_model(m)
        st = make_state(m, 160, mode, kv_format="e4m3", kv_block=32, **kw)
        run = LabRunner(m, holder, st)
        run.prefill(ids[:, :100], 50)
        if mode == "sparse":
            st.begin_request(0.25)
        branch = st.cache.clone()
        assert branch.quant[0].k.data_ptr() != st.cache.quant[0].k.data_ptr()
        first = [run.step(ids[:, 100 + t:101 + t]) for t in range(5)]
        run.rollback(100)
        again = [run.step(ids[:, 100 + t:101 + t]) for t in range(5)]
        # the same tokens after a rollback: the same rows (their blocks' scales can only have kept or grown)
        for a, b in zip(first, again):
            close(a, b, 0.2, 0.05, "after the rollback")
        st2 = LabState(branch, st.indexers, mode=mode, **kw)
        other = LabRunner(m, holder, st2)
        if mode == "sparse":
            st2.begin_request(0.25)
        for t in range(5):
            assert torch.equal(other.step(ids[:, 100 + t:101 + t]), first[t])


def test_configurations_that_do_not_fit_are_refused(gpu):
    m, _ = tiny_pair(gpu)
    c = make_cache(m, 64, with_index=False)
    for kw in (dict(mode="window"), dict(mode="full", window=4), dict(mode="window", window=0),
               dict(mode="window", window=4, sinks=-1), dict(mode="other")):
        with pytest.raises(ValueError):
            LabState(c, **kw)
    for kw in (dict(kv_format="int8"), dict(kv_format="e4m3", kv_block=128)):
        with pytest.raises(ValueError):
            make_cache(m, 64, with_index=False, **kw)
    with pytest.raises(ValueError, match="128"):
        LabCache(layers=1, batch=1, groups=1, capacity=64, head_dim=64, device=gpu, dtype=torch.bfloat16, kv_format="e4m3")
