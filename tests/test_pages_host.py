"""The paged cache without a GPU: the oracle against known answers, and what the C entries and their Python callers refuse
before any launch (the pointers below are never touched)."""
from __future__ import annotations

import pytest
import torch

import attention_lab
from attention_lab import _native
from attention_lab.pages import PagedCache
from oracle.pages import Pages


def model(S=3, pages=8, W=4, page=4):
    k = torch.arange(pages * page, dtype=torch.float32).view(1, pages, 1, page, 1).expand(1, pages, 1, page, 2).clone()
    return Pages(k, -k, [[-1] * W for _ in range(S)], [0] * S)


def test_oracle_shares_and_takes_apart():
    m = model()
    m.reserve([6, 0, 0])
    assert m.table[0] == [0, 1, -1, -1] and m.lengths == [6, 0, 0] and m.refs[:3] == [1, 1, 0]
    m.fork([0, 0, 0])
    assert m.refs[:2] == [3, 3] and m.lengths == [6] * 3
    m.reserve([1, 0, 1])                       # slot 1 holds page 1 too: both writers leave
    assert [r[:2] for r in m.table] == [[0, 2], [0, 1], [0, 3]] and m.lengths == [7, 6, 7]
    assert torch.equal(m.k[0, 2, 0, :, 0], torch.tensor([4.0, 5.0, 10.0, 11.0]))   # two rows copied, the rest as it was
    m.fork([0, 0, -1])
    assert m.table[2] == [-1] * 4 and m.refs == [2, 0, 2, 0, 0, 0, 0, 0]
    m.reserve([1, 1, 0])                       # all holders write: the last keeps the page
    assert m.table[0][1] == 1 and m.table[1][1] == 2


def test_oracle_runs_out_and_truncates():
    m = model(S=2, pages=3, W=3)
    m.reserve([5, 9])                          # two pages, then three: one is left, and the table has room
    assert m.table == [[0, 1, -1], [2, -1, -1]] and m.missing == 2
    m.reserve([8, 0])                          # positions 5 .. 12 begin entry 2 (no page) and entry 3 (no entry)
    assert m.missing == 4 and m.lengths == [13, 9]
    m.truncate([4, -3])
    assert m.table == [[0, -1, -1], [-1, -1, -1]] and m.lengths == [4, 0]


def test_oracle_compacts():
    m = model(S=2)
    m.table, m.lengths = [[5, 1, -1, -1], [5, 7, 0, -1]], [8, 11]
    m.compact()                                # four in use: 5 and 7 go to 2 and 3
    assert m.table == [[2, 1, -1, -1], [2, 3, 0, -1]] and m.refs == [1, 1, 2, 1, 0, 0, 0, 0]
    assert m.k[0, 2, 0, 0, 0] == 20 and m.v[0, 3, 0, 1, 1] == -29


def test_exported():
    for name in ("PagedCache", "page_fork", "page_reserve", "page_append", "page_truncate", "page_compact"):
        assert name in attention_lab.__all__ and hasattr(attention_lab, name)


FORK = dict(table=16, lengths=16, refs=16, parents=1024, S=2, W=4, pages=8, stream=None)
ALIKE = dict(FORK, lengths=4096, refs=8192, parents=12288)   # table [16, 48), lengths [4096, 4104), refs [8192, 8224)
TRUNCATE = dict(table=16, lengths=16, refs=16, to=None, length=3, S=2, W=4, pages=8, page=16, stream=None)
RESERVE = dict(k=16, v=16, layers=2, pages=8, G=2, page=16, table=16, lengths=16, refs=16, tokens=None, each=1, S=2, W=4,
               missing=None, scratch=16, scratch_bytes=4096, stream=None)
APPEND = dict(k=16, kb=1024, kg=512, kt=128, v=16, vb=1024, vg=512, vt=128, kp=16, vp=16, pages=8, G=2, page=16, table=16,
              lengths=16, tokens=None, S=2, W=4, T=4, stream=None)
COMPACT = dict(k=16, v=16, layers=2, pages=8, G=2, page=16, table=16, lengths=16, refs=16, S=2, W=4, scratch=16,
               scratch_bytes=4096, stream=None)
EVERY = (("attnlab_page_fork", FORK), ("attnlab_page_truncate", TRUNCATE), ("attnlab_page_reserve", RESERVE),
         ("attnlab_page_append", APPEND), ("attnlab_page_compact", COMPACT))
REFUSED = [(e, a, c, m) for e, a in EVERY for c, m in (
    (dict(S=0), "slots"), (dict(S=1025), "slots"), (dict(W=0), "positive"), (dict(pages=0), "positive"),
    (dict(table=None), "pointers"), (dict(lengths=None), "pointers"), (dict(S=1024, W=1 << 21), "2\\^31 entries"))]
REFUSED += [(e, a, c, m) for e, a in EVERY[1:] for c, m in (
    (dict(page=48), "power of two"), (dict(page=0), "power of two"), (dict(page=1 << 17), "power of two"),
    (dict(W=1 << 27), "2\\^31"))]
REFUSED += [(e, a, c, m) for e, a in EVERY[2:] for c, m in (
    (dict(G=0), "positive"), (dict(pages=1 << 26), "2\\^31"), (dict(k=None), "pointers"), (dict(v=24), "pointers"))]
REFUSED += [
    ("attnlab_page_fork", FORK, dict(parents=None), "parents"), ("attnlab_page_fork", FORK, dict(refs=None), "pointers"),
    *(("attnlab_page_fork", ALIKE, dict(parents=p), "own tensors") for p in (12, 44, 4096, 4092, 4100, 8188, 8220)),
    ("attnlab_page_truncate", TRUNCATE, dict(length=-1), "negative"),
    ("attnlab_page_reserve", RESERVE, dict(each=-1), "negative"), ("attnlab_page_reserve", RESERVE, dict(layers=0), "positive"),
    ("attnlab_page_reserve", RESERVE, dict(scratch=None), "scratch"), ("attnlab_page_reserve", RESERVE, dict(scratch=8), "scratch"),
    ("attnlab_page_reserve", RESERVE, dict(scratch_bytes=16), "scratch"),
    ("attnlab_page_append", APPEND, dict(T=-1), "negative"), ("attnlab_page_append", APPEND, dict(kt=132), "aligned"),
    ("attnlab_page_append", APPEND, dict(kp=8), "pointers"), ("attnlab_page_append", APPEND, dict(k=18), "aligned"),
    ("attnlab_page_compact", COMPACT, dict(scratch_bytes=64), "scratch"),
]


@pytest.mark.parametrize("entry,args,change,match", REFUSED)
def test_refused_before_any_launch(native_lib, entry, args, change, match):
    assert len(args) == len(_native.SIGNATURES[entry][1])
    with pytest.raises(ValueError, match=match):
        _native.call(entry, *dict(args, **change).values())


def test_nothing_to_do_is_no_launch(native_lib):
    _native.call("attnlab_page_append", *dict(APPEND, T=0, k=None, v=None).values())


def test_scratch(native_lib):
    size = native_lib.attnlab_page_scratch_bytes
    assert size(3, 100) == 16 + 12 * 100 and size(1024, 5) == 16 + 12 * 1024
    assert size(0, 5) == size(5, 0) == -1


def test_python_makes_the_scratch(native_lib, monkeypatch):
    """The Python side's scratch is what the C side asks for."""
    seen = []
    monkeypatch.setattr(_native, "call_on", lambda device, entry, *args: seen.append((entry, args)))
    monkeypatch.setattr(_native, "stream_of", lambda device: None)
    for sizes in (dict(), dict(pages=1, S=5), dict(pages=33, S=1)):
        c = PagedCache(**parts(**sizes))
        attention_lab.page_reserve(c)
        attention_lab.page_compact(c)
        need = native_lib.attnlab_page_scratch_bytes(c.slots, c.num_pages)
        assert [args[len(_native.SIGNATURES[entry][1]) - 2] for entry, args in seen] == [need, need]
        seen.clear()


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on a HIP device: for the checks, which look no further."""
    is_cuda = True


def parts(layers=2, pages=8, G=2, page=16, S=3, W=4):
    k = torch.zeros(layers, pages, G, page, 128, dtype=torch.bfloat16).as_subclass(OnDevice)
    ints = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    return dict(k=k, v=k.clone(), table=ints(S, W), lengths=ints(S), refs=ints(pages))


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(2, 8, 2, 16, 128, dtype=torch.bfloat16)), "HIP device"),
    (dict(k=torch.zeros(2, 8, 2, 16, 64, dtype=torch.bfloat16).as_subclass(OnDevice)), "k must be"),
    (dict(k=torch.zeros(2, 8, 2, 16, 128).as_subclass(OnDevice)), "k must be"),
    (dict(v=torch.zeros(2, 8, 2, 8, 128, dtype=torch.bfloat16)), "match k"),
    (dict(table=torch.zeros(3, 4, dtype=torch.int64)), "table"), (dict(table=torch.zeros(12, dtype=torch.int32)), "table"),
    (dict(table=torch.zeros(4, 3, dtype=torch.int32).t()), "table"),
    (dict(table=torch.zeros(1025, 4, dtype=torch.int32)), "slots"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)), "lengths"), (dict(refs=torch.zeros(7, dtype=torch.int32)), "refs"),
    (dict(missing=torch.zeros(2, dtype=torch.int32)), "missing"),
])
def test_cache_refuses(change, match):
    PagedCache(**parts())
    with pytest.raises(ValueError, match=match):
        PagedCache(**dict(parts(), **change))


@pytest.mark.parametrize("sizes,match", [((0, 1, 1, 1, 1, 1), "positive"), ((1, 1025, 1, 1, 1, 1), "positive"),
                                         ((1, 1, 1, 1, 24, 1), "power of two"), ((1, 1, 1, 1, 16, 1 << 28), "2\\^31"),
                                         ((1, 1, 8, 1 << 24, 16, 1), "2\\^31"), ((1, 1024, 1, 1, 1, 1 << 21), "2\\^31")])
def test_empty_refuses(sizes, match):
    with pytest.raises(ValueError, match=match):
        PagedCache.empty(*sizes, device="cpu")


def test_operators_refuse():
    c = PagedCache(**parts())
    rows = torch.zeros(3, 2, 5, 128, dtype=torch.bfloat16)
    for call, match in (
        (lambda: attention_lab.page_fork(c, torch.zeros(2, dtype=torch.int32)), "parents"),
        (lambda: attention_lab.page_fork(c, torch.zeros(3, dtype=torch.int64)), "parents"),
        (lambda: attention_lab.page_reserve(c, -1), "tokens"), (lambda: attention_lab.page_reserve(c, 2 ** 31), "tokens"),
        (lambda: attention_lab.page_reserve(c, torch.zeros(3)), "tokens"),
        (lambda: attention_lab.page_truncate(c, -1), "lengths"),
        (lambda: attention_lab.page_truncate(c, torch.zeros(4, dtype=torch.int32)), "lengths"),
        (lambda: attention_lab.page_append(c, 2, rows, rows), "layer"), (lambda: attention_lab.page_append(c, -1, rows, rows), "layer"),
        (lambda: attention_lab.page_append(c, 0, rows[:2], rows[:2]), "slots"),
        (lambda: attention_lab.page_append(c, 0, rows.float(), rows.float()), "bfloat16"),
        (lambda: attention_lab.page_append(c, 0, rows, rows[:, :, :4]), "match k"),
        (lambda: attention_lab.page_append(c, 0, rows, rows, torch.zeros(2, dtype=torch.int32)), "tokens"),
    ):
        with pytest.raises(ValueError, match=match):
            call()
