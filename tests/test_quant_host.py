"""The 8-bit cache and the windowed read without a GPU: the oracle against known answers, and what the C entries and
their Python callers refuse before any launch (the pointers below are never touched)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import attention_lab
from attention_lab import _native, hip_range
from attention_lab.quant import QuantCache
from oracle import quant as oq


def test_oracle_codes():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(oq.TABLE, t)
    fin = oq.TABLE[~np.isnan(oq.TABLE)]
    codes = oq.encode(fin)
    np.testing.assert_array_equal(oq.TABLE[codes], fin)
    # halfway between 1 (even mantissa) and 1.125, between 1.125 and 1.25 (even), and below the smallest step
    np.testing.assert_array_equal(oq.TABLE[oq.encode(np.array([1.0625, 1.1875, 2.0 ** -10, 1.5 * 2.0 ** -9, -2.0 ** -11]))],
                                  [1.0, 1.25, 0.0, 2.0 ** -8, -0.0])
    assert oq.encode(np.array([np.nan]))[0] == 127
    rng = np.random.default_rng(0)
    x = rng.uniform(-440, 440, 4000).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(oq.encode(x.astype(np.float64)), want)


@pytest.mark.parametrize("top,x", [(0.0, 17), (448.0, 127), (448.0000001, 128), (1.0, 119), (1.75, 119),
                                   (1.7500001, 120), (2.0 ** -140, 17), (oq.LARGEST, 247)])
def test_oracle_scale(top, x):
    assert oq.scale_byte(top) == x


def test_oracle_append_keeps_and_moves_codes():
    codes, exps = np.zeros((1, 1, 32, 2), np.uint8), np.zeros((1, 1, 2), np.uint8)
    oq.append(codes, exps, np.full((1, 1, 3, 2), 1.0), 0, 16)
    assert exps[0, 0].tolist() == [119, 0]
    oq.append(codes, exps, np.full((1, 1, 14, 2), 4.0), 3, 16)     # louder: the block's scale grows, its rows follow
    assert exps[0, 0].tolist() == [121, 121]
    v = oq.values(codes, exps, 16)[0, 0, :, 0]
    assert v[:3].tolist() == [1.0] * 3 and v[3:17].tolist() == [4.0] * 14
    oq.append(codes, exps, np.full((1, 1, 1, 2), 0.5), 17, 16)      # quieter: the scale stays
    assert exps[0, 0, 1] == 121 and oq.values(codes, exps, 16)[0, 0, 17, 0] == 0.5


def test_oracle_visible():
    assert oq.visible(5, 10, None, 0).tolist() == [0, 1, 2, 3, 4, 5]
    assert oq.visible(5, 10, 2, 1).tolist() == [0, 4, 5]
    assert oq.visible(9, 6, 2, 1).tolist() == [0]
    assert oq.visible(9, 6, 2, 0).tolist() == []
    assert oq.visible(3, 6, 100, 100).tolist() == [0, 1, 2, 3]


def test_exported():
    for name in ("QuantCache", "quantize_append", "dequantize_rows", "quant_attention", "quant_gather_attention",
                 "window_attention"):
        assert name in attention_lab.__all__ and hasattr(attention_lab, name)


APPEND = dict(k=16, kb=1024, kg=256, kt=128, v=16, vb=1024, vg=256, vt=128, dtype=0, kc=16, vc=16, ke=16, ve=16,
              starts=None, start=0, B=1, G=2, T=4, C=64, block=16, stream=None)
READ = dict(kc=16, vc=16, ke=16, ve=16, ko=16, vo=16, dtype=0, starts=None, start=0, B=1, G=2, T=4, C=64, block=16,
            stream=None)
DECODE = dict(K=16, V=16, ke=16, ve=16, block=16, q=16, lengths=None, length=10, q_pos=9, window=0, sinks=0, B=1, G=2,
              h=2, C=64, P=1, scale=0.1, out=16, out_bf16=1, part=None, arrive=None, stream=None)
ROWS = dict(K=16, V=16, ke=16, ve=16, block=16, q=16, rows=16, rows_stride=8, B=1, G=2, h=2, S=8, C=64, P=1, scale=0.1,
            out=16, out_bf16=1, part=None, arrive=None, stream=None)
CHUNK = dict(q=16, K=16, V=16, ke=16, ve=16, block=16, out=16, B=1, G=2, h=2, T=4, q_pos0=0, legal=4, C=64, window=0,
             sinks=0, scale=0.1, splits=1, part=None, part_bytes=0, stream=None)
REFUSED = [
    ("attnlab_quant_append", APPEND, dict(block=48), "block=48"), ("attnlab_quant_append", APPEND, dict(block=0), "block"),
    ("attnlab_quant_append", APPEND, dict(dtype=3), "dtype"), ("attnlab_quant_append", APPEND, dict(T=-1), "negative"),
    ("attnlab_quant_append", APPEND, dict(start=61), "outside"), ("attnlab_quant_append", APPEND, dict(start=-1), "outside"),
    ("attnlab_quant_append", APPEND, dict(start=2 ** 31 - 1), "outside"),
    ("attnlab_quant_append", APPEND, dict(k=None), "pointers"), ("attnlab_quant_append", APPEND, dict(ke=None), "pointers"),
    ("attnlab_quant_append", APPEND, dict(kt=129), "aligned"), ("attnlab_quant_append", APPEND, dict(v=24), "aligned"),
    ("attnlab_quant_append", APPEND, dict(kc=8), "aligned"), ("attnlab_quant_append", APPEND, dict(B=0), "positive"),
    ("attnlab_quant_append", APPEND, dict(B=2 ** 15, G=2 ** 15, starts=16), "too large"),
    ("attnlab_quant_read", READ, dict(start=61), "outside"), ("attnlab_quant_read", READ, dict(dtype=7), "dtype"),
    ("attnlab_quant_read", READ, dict(ko=None), "pointers"), ("attnlab_quant_read", READ, dict(vo=8), "aligned"),
    ("attnlab_quant_read", READ, dict(T=-2), "negative"), ("attnlab_quant_read", READ, dict(block=128), "block"),
    ("attnlab_range_decode", DECODE, dict(h=9), "h=9"), ("attnlab_range_decode", DECODE, dict(h=0), "h=0"),
    ("attnlab_range_decode", DECODE, dict(P=0), "partitions"), ("attnlab_range_decode", DECODE, dict(P=257), "partitions"),
    ("attnlab_range_decode", DECODE, dict(P=2), "partial"), ("attnlab_range_decode", DECODE, dict(length=65), "length"),
    ("attnlab_range_decode", DECODE, dict(q_pos=-1), "position"),
    ("attnlab_range_decode", DECODE, dict(window=-1), "window"), ("attnlab_range_decode", DECODE, dict(sinks=-1), "sinks"),
    ("attnlab_range_decode", DECODE, dict(q=8), "aligned"), ("attnlab_range_decode", DECODE, dict(ve=None), "pointers"),
    ("attnlab_range_decode", DECODE, dict(ke=None, ve=None, K=None), "pointers"),
    ("attnlab_range_decode", DECODE, dict(block=8), "block"),
    ("attnlab_quant_attend", ROWS, dict(S=0), "at least one row"), ("attnlab_quant_attend", ROWS, dict(rows=None), "rows"),
    ("attnlab_quant_attend", ROWS, dict(rows_stride=7), "rows"), ("attnlab_quant_attend", ROWS, dict(ke=None, ve=None), "scale"),
    ("attnlab_quant_attend", ROWS, dict(h=12), "h=12"),
    ("attnlab_range_prefill", CHUNK, dict(h=17), "h=17"), ("attnlab_range_prefill", CHUNK, dict(q_pos0=-1), "q_pos0"),
    ("attnlab_range_prefill", CHUNK, dict(legal=65), "legal"), ("attnlab_range_prefill", CHUNK, dict(splits=17), "splits"),
    ("attnlab_range_prefill", CHUNK, dict(splits=2), "part"), ("attnlab_range_prefill", CHUNK, dict(window=-3), "window"),
    ("attnlab_range_prefill", CHUNK, dict(q_pos0=2 ** 31 - 2), "2\\^31"), ("attnlab_range_prefill", CHUNK, dict(T=-1), "T"),
    ("attnlab_range_prefill", CHUNK, dict(out=4), "aligned"), ("attnlab_range_prefill", CHUNK, dict(ve=None), "pointers"),
    ("attnlab_range_prefill", CHUNK, dict(splits=2, part=16, part_bytes=64), "part"),
]


@pytest.mark.parametrize("entry,args,change,match", REFUSED)
def test_refused_before_any_launch(native_lib, entry, args, change, match):
    assert len(args) == len(_native.SIGNATURES[entry][1])
    with pytest.raises(ValueError, match=match):
        _native.call(entry, *dict(args, **change).values())


def test_nothing_to_do_is_no_launch(native_lib):
    _native.call("attnlab_quant_append", *dict(APPEND, T=0, k=None, v=None).values())
    _native.call("attnlab_quant_read", *dict(READ, T=0, ko=None, vo=None).values())
    _native.call("attnlab_range_prefill", *dict(CHUNK, T=0, q=None).values())


def test_partials(native_lib):
    f = native_lib.attnlab_range_prefill_part_bytes
    assert f(1, 2, 3, 5, 1) == 0 and f(1, 2, 3, 5, 4) == 30 * 4 * 132 * 4 and f(1, 2, 3, 5, 0) == -1
    assert f(32, 8, 16, 65536, 16) == 32 * 8 * 16 * 65536 * 16 * 528


def test_python_refusals_without_a_device():
    k = torch.zeros(1, 2, 64, 128, dtype=torch.float8_e4m3fn)
    e = torch.zeros(1, 2, 1, dtype=torch.uint8)
    with pytest.raises(ValueError, match="HIP device"):
        QuantCache(k, k, e, e)
    with pytest.raises(ValueError, match="block"):
        QuantCache(k, k, e, e, block=128)
    with pytest.raises(ValueError, match="block"):
        QuantCache.empty(1, 2, 64, block=8, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        QuantCache.empty(1, 0, 64, device="cpu")
    bf = torch.zeros(1, 2, 64, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="HIP device"):
        attention_lab.window_attention(bf[:, :, None, :1], bf, bf, window=4)
    with pytest.raises(ValueError, match="window"):
        hip_range.check_window(0, 4)
    with pytest.raises(ValueError, match="sinks"):
        hip_range.check_window(None, -1)
    assert hip_range.check_window(None, 4) == (0, 0) and hip_range.check_window(2 ** 40, 2 ** 40) == (2 ** 31 - 1,) * 2


@pytest.mark.parametrize("BG", [1, 3, 8, 128, 1000])
@pytest.mark.parametrize("n", [0, 1, 127, 128, 4100, 131072])
def test_split_rules_stay_in_range(BG, n):
    assert 1 <= hip_range.decode_partitions(BG, n) <= 256
    assert 1 <= hip_range.decode_partitions(BG, n, listed=True) <= 256
    assert 2 <= hip_range.decode_partitions(BG, n, ragged=True) <= 256
    for h in (1, 3, 16):
        for T in (1, 33, 8192):
            assert 1 <= hip_range.chunk_splits(BG, h, T, n) <= hip_range.MAX_SPLITS


def test_argument_types_survive_the_binding():
    """64-bit arguments are declared as such: a query position past 2^31 is not cut to 32 bits."""
    assert _native.SIGNATURES["attnlab_range_decode"][1][8] is ctypes.c_int64
    assert _native.SIGNATURES["attnlab_quant_attend"][1][7] is ctypes.c_int64
    assert [i for i, t in enumerate(_native.SIGNATURES["attnlab_quant_append"][1]) if t is ctypes.c_int64] == [1, 2, 3, 5,
                                                                                                                6, 7]


@pytest.mark.parametrize("block", [0, 8, 48, 128, -64])
def test_wrapper_cache_refuses_other_blocks(block):
    pytest.importorskip("transformers")
    from attention_lab.qwen_wrap import LabCache
    with pytest.raises(ValueError, match="kv_block must be one of"):
        LabCache(layers=1, batch=1, groups=1, capacity=64, head_dim=128, device="cpu", dtype=torch.bfloat16,
                 kv_format="e4m3", kv_block=block)


@pytest.mark.parametrize("entry,args", [("attnlab_range_decode", DECODE), ("attnlab_quant_attend", ROWS)])
@pytest.mark.parametrize("out,bf16", [(18, 1), (17, 1), (20, 0), (18, 0)])
def test_outputs_off_their_pairs_are_refused(native_lib, entry, args, out, bf16):
    with pytest.raises(ValueError, match="out must be aligned"):
        _native.call(entry, *dict(args, out=out, out_bf16=bf16).values())


def test_rows_are_copied_only_where_their_address_or_strides_are_odd():
    from attention_lab.quant import _rows
    x = torch.zeros(2, 3, 5, 128, dtype=torch.bfloat16)
    odd = torch.zeros(x.numel() + 1, dtype=torch.bfloat16)[1:].view(x.shape)
    wide = torch.zeros(1, 1, 1, 131, dtype=torch.bfloat16)[..., :128]
    for t, kept in ((x, True), (x.transpose(1, 2), True), (x[:, :, :1], True), (wide, True), (odd, False),
                    (x.transpose(2, 3).contiguous().transpose(2, 3), False)):
        got, at, *strides = _rows(t, 8)
        assert (got is t) == kept and at % 16 == 0 and not any(s % 8 for s in strides) and torch.equal(got, t)


def test_steps_that_share_a_stream_take_turns(monkeypatch):
    """Two host threads on one stream: no launch of one comes between the other's score and select, which meet in the
    select state; the launches are stand-ins here."""
    import contextlib
    import threading
    import time
    from types import SimpleNamespace
    from attention_lab import decode, hip_score, hip_select
    events = []

    def score(zT, lo, hi, *, state, **kw):
        events.append(("score", threading.get_ident(), state.data_ptr()))
        time.sleep(0.02)
        return torch.zeros(1, 1, hi - lo)

    def select(s, *args, rows, **kw):
        events.append(("select", threading.get_ident(), 0))
        return rows, None

    monkeypatch.setattr(hip_score, "score_grouped", score)
    monkeypatch.setattr(hip_select, "select_rows", select)
    monkeypatch.setattr(hip_select, "reserve", lambda *a: None)
    monkeypatch.setattr(hip_range, "capturing", lambda device: False)
    monkeypatch.setattr(hip_range, "check_listed", lambda *a: 1)
    monkeypatch.setattr(hip_range, "listed_attention", lambda q, *a, **k: q)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    stream = threading.local()
    monkeypatch.setattr(_native, "stream_of", lambda device: getattr(stream, "of", 0))
    monkeypatch.setattr(decode, "_QUANT_WS", {})
    cache = SimpleNamespace(capacity=400, batch=1, groups=1, device=torch.device("cpu"))
    q = torch.zeros(1, 1, 1, 1, 128, dtype=torch.bfloat16)
    req = decode.prepare_request(1, 1, 400, valid_length=300, query_position=299, rho=0.1, device="cpu")
    lay = req.layout

    def run(of):
        stream.of = of
        for _ in range(4):
            decode.sparse_decode_step_quant(q, q, cache, torch.zeros(1, 1, 32, 400, dtype=torch.bfloat16),
                                            torch.zeros(1, 128, 32), torch.zeros(1, 32, 128), req.fixed_rows, req.off_lo,
                                            lay.candidate_lo, lay.candidate_hi, req.k, req.selected_count)

    for streams, shared in (((7, 7), True), ((7, 8), False)):
        events.clear()
        threads = [threading.Thread(target=run, args=(s,)) for s in streams]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len(events) == 16 and len({p for n, _, p in events if n == "score"}) == (1 if shared else 2)
        if shared:
            assert all(a[0] == "score" and b[0] == "select" and a[1] == b[1] for a, b in zip(events[::2], events[1::2]))
    assert isinstance(decode._step_workspace(cache.device, object())[1], contextlib.nullcontext)


KEPT = dict(k=16, kb=1024, kg=256, kt=128, v=16, vb=1024, vg=256, vt=128, kc=16, vc=16, ke=16, ve=16, start=0, B=1, G=2,
            T=4, C=64, block=16, kk=16, vk=16, rows=32, stream=None)


@pytest.mark.parametrize("change,match", [(dict(kk=None), "kept rows"), (dict(vk=8), "kept rows"), (dict(rows=0), "kept rows"),
                                          (dict(start=61), "outside"), (dict(start=-1), "outside"), (dict(k=8), "aligned"),
                                          (dict(T=-1), "negative"), (dict(block=8), "block")])
def test_kept_rows_refused_before_any_launch(native_lib, change, match):
    assert len(KEPT) == len(_native.SIGNATURES["attnlab_quant_append_kept"][1])
    with pytest.raises(ValueError, match=match):
        _native.call("attnlab_quant_append_kept", *dict(KEPT, **change).values())
    _native.call("attnlab_quant_append_kept", *dict(KEPT, T=0).values())


def test_configurations_the_reads_do_not_take_are_refused_before_a_state_is_built():
    """At construction, and not in the first layer's read, which comes after its rows were written."""
    pytest.importorskip("transformers")
    from types import SimpleNamespace
    from attention_lab.qwen_wrap import LabCache, LabState, make_state, tiny_qwen3
    size = dict(layers=1, batch=1, groups=2, capacity=64, device="cpu")
    for kw in (dict(head_dim=128, dtype=torch.float32), dict(head_dim=128, dtype=torch.float16), dict(head_dim=128),
               dict(head_dim=64, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="bfloat16 rows of head_dim 128"):
            LabCache(**size, kv_format="e4m3", **{"dtype": torch.float32, **kw})
    for kw in (dict(head_dim=128, dtype=torch.float32), dict(head_dim=64, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="bfloat16 rows of head_dim 128"):
            LabState(LabCache(**size, **kw), mode="window", window=8)
    LabState(LabCache(**size, head_dim=128, dtype=torch.bfloat16), mode="window", window=8)

    def model(h, groups=1):
        return tiny_qwen3(seed=0, layers=1, hidden=64, heads=h * groups, groups=groups, head_dim=128, intermediate=64,
                          vocab=32, dtype=torch.bfloat16)

    for h, mode, kw, most in ((9, "sparse", dict(kv_format="e4m3"), 8), (17, "full", dict(kv_format="e4m3"), 16),
                              (9, "sparse", dict(kv_format="e4m3", selector="recent"), 8), (17, "window", dict(window=4), 16)):
        with pytest.raises(ValueError, match=f"at most {most} query heads"):
            make_state(model(h), 64, mode, **kw)
    make_state(model(16), 64, "window", window=4)
    make_state(model(17), 64, "full")
    cache = SimpleNamespace(layers=1, dtype=torch.bfloat16, head_dim=128, kv_format="e4m3", has_index=True)
    index = SimpleNamespace(wq_t_scaled=torch.zeros(2, 9 * 128, 32))
    with pytest.raises(ValueError, match="at most 8 query heads"):
        LabState(cache, [index], mode="sparse")
    LabState(cache, [index], mode="full")
