"""The paged cache where no GPU is needed: page bookkeeping, and what the C ABI and the binding refuse."""
import ctypes as C
import os
import random

import pytest
import torch

from daisy_b200 import _lib
from daisy_b200.kv_cache import PageBook


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from daisy_b200.build import build
        build()
    return _lib.lib()


def _consistent(book, pages):
    held = [p for row, f, e in zip(book.table, book.first, book.end) for p in row[f:e]]
    assert sorted(held + book.free) == list(range(pages))
    for slot, n in enumerate(book.length):
        row = book.table[slot]
        assert all(p == -1 for p in row[:book.first[slot]] + row[book.end[slot]:])
        assert n < 0 or n <= book.end[slot] * book.page


def test_page_book_random_traffic():
    rng = random.Random(7)
    book = PageBook(40, 5, 300, 16)
    for _ in range(3000):
        live = [s for s, n in enumerate(book.length) if n >= 0]
        what = rng.random()
        if what < 0.1 and len(live) < 5:
            assert book.claim() not in live
        elif what < 0.15 and live:
            book.release(rng.choice(live))
        elif what < 0.3 and live:
            s = rng.choice(live)
            book.forget(s, rng.randrange(-20, book.length[s] + 1))
        elif live:
            slots = rng.sample(live, rng.randint(1, len(live)))
            counts = [min(rng.randrange(40), 300 - book.length[s]) for s in slots]
            before = [list(r) for r in book.table], list(book.free)
            try:
                changed = book.reserve(slots, counts)
            except RuntimeError:
                assert before == (book.table, book.free)             # nothing changed
                continue
            assert set(changed) <= set(slots)
            book.advance(slots, counts)
        _consistent(book, 40)


def test_page_book_refusals():
    book = PageBook(3, 2, 40, 16)
    with pytest.raises(ValueError, match="holds no sequence"):
        book.reserve([0], [1])
    a = book.claim()
    with pytest.raises(ValueError, match="the table holds 40"):
        book.reserve([a], [41])
    with pytest.raises(ValueError, match="no pages for"):
        book.advance([a], [1])
    assert book.reserve([a], [33]) == [a] and book.reserve([a], [40]) == []
    b = book.claim()
    with pytest.raises(RuntimeError, match="0 pages left"):
        book.reserve([b], [1])
    with pytest.raises(RuntimeError, match="slots"):
        book.claim()
    book.advance([a], [33])
    assert book.forget(a, 16) == [a] and book.forget(a, 31) == [] and book.free == [book.free[0]]
    assert book.reserve([b], [16]) == [b]
    book.release(a)
    with pytest.raises(ValueError, match="holds no sequence"):
        book.release(a)


def _pages(a, **over):
    d = dict(k=a, v=a, p_sb=2 * 16 * 128, p_sh=16 * 128, p_sr=128, table=a, table_sb=4, n_pages=8, H=2, page=16, width=4, n_seq=3)
    d.update(over)
    return _lib.Pages(**d)


def _append(lib, a, cache, **over):
    d = dict(k=a, v=a, q=a, ks=(256, 256, 128), vs=(256, 256, 128), qs=(512, 512, 128), q_out=a, start=a, cu=None, cos=a, sin=a, rows=64, ve=None, ves=(0, 0, 0), gate=None,
             B=3, T=1, Hq=4, D=128, flags=15)
    d.update(over)
    return lib.daisy_b200_paged_append(C.byref(cache) if cache else None, d["k"], d["v"], d["q"], *d["ks"], *d["vs"], *d["qs"], d["q_out"], d["start"], d["cu"], d["cos"], d["sin"],
                                       d["rows"], d["ve"], *d["ves"], d["gate"], d["B"], d["T"], d["Hq"], d["D"], 1e-6, d["flags"], None, None)


def _decode(lib, a, cache, **over):
    d = dict(q=a, k=a, v=a, s=(512, 128, 256, 128, 256, 128), lens=a, window=0, cos=a, sin=a, rows=64, out=a, os=(512, 128), ve=None, gate=None, Hq=4, D=128, flags=15, ws=a, n=1 << 40)
    d.update(over)
    return lib.daisy_b200_paged_decode_step(C.byref(cache), d["q"], d["k"], d["v"], *d["s"], d["lens"], d["window"], d["cos"], d["sin"], d["rows"], d["out"], *d["os"], d["ve"], 256, 128,
                                            d["gate"], d["Hq"], d["D"], 0.12, 1e-6, d["flags"], d["ws"], d["n"], None, None)


def _attend(lib, a, cache, few=False, **over):
    d = dict(q=a, qs=(512, 512, 128), lens=a, cu=None, window=0, out=a, os=(512, 512, 128), B=3, T=1, Hq=4, D=128, scale=0.12, flags=0, ws=a, n=1 << 40)
    d.update(over)
    fn = lib.daisy_b200_paged_attend_few if few else lib.daisy_b200_paged_attend
    return fn(C.byref(cache), d["q"], *d["qs"], d["lens"], d["cu"], d["window"], d["out"], *d["os"], d["B"], d["T"], d["Hq"], d["D"], d["scale"], d["flags"], d["ws"], d["n"], None, None)


@pytest.fixture(scope="module")
def address():
    buf = (C.c_char * 8192)()
    yield (C.addressof(buf) + 255) & ~255                            # never dereferenced
    del buf


@pytest.mark.parametrize("over,code", [(dict(k=None), "EINVAL"), (dict(table=None), "EINVAL"), (dict(n_pages=0), "EINVAL"), (dict(H=0), "EINVAL"), (dict(width=0), "EINVAL"),
                                       (dict(n_seq=0), "EINVAL"), (dict(table_sb=-1), "EINVAL"), (dict(page=8), "EUNSUPPORTED"), (dict(page=48), "EUNSUPPORTED"),
                                       (dict(page=512), "EUNSUPPORTED"), (dict(width=1 << 30), "EUNSUPPORTED"), (dict(p_sr=132), "EALIGN"), (dict(p_sr=120), "EINVAL"),
                                       (dict(p_sh=0), "EINVAL"), (dict(p_sb=0), "EINVAL")])
def test_pools_that_are_refused(lib, address, over, code):
    for call in (_append, _decode, _attend, lambda *x: _attend(*x, few=True)):
        assert call(lib, address, _pages(address, **over)) == getattr(_lib, code)
    assert _append(lib, address, _pages(address + 2)) == _lib.EALIGN
    assert _append(lib, address, None) == _lib.EINVAL


@pytest.mark.parametrize("over,code", [(dict(k=None), "EINVAL"), (dict(start=None), "EINVAL"), (dict(q=None), "EINVAL"), (dict(q_out=None), "EINVAL"), (dict(Hq=0), "EINVAL"),
                                       (dict(T=0), "EINVAL"), (dict(B=2), "EINVAL"), (dict(flags=16), "EINVAL"), (dict(flags=256 | 15), "EINVAL"), (dict(cos=None), "EINVAL"),
                                       (dict(rows=0), "EINVAL"), (dict(ve="a"), "EINVAL"), (dict(ve="a", gate="a", flags=11), "EINVAL"), (dict(D=64), "EUNSUPPORTED"),
                                       (dict(T=1 << 29), "EUNSUPPORTED"), (dict(ks=(256, 260, 128)), "EALIGN"), (dict(qs=(512, 516, 128)), "EALIGN"), (dict(cu="a"), "EINVAL")])
def test_appends_that_are_refused(lib, address, over, code):
    over = {n: address if v == "a" else v for n, v in over.items()}
    assert _append(lib, address, _pages(address), **over) == getattr(_lib, code)


@pytest.mark.parametrize("over,code", [(dict(q=None), "EINVAL"), (dict(lens=None), "EINVAL"), (dict(out=None), "EINVAL"), (dict(ws=None), "EINVAL"), (dict(Hq=3), "EINVAL"),
                                       (dict(flags=32), "EINVAL"), (dict(sin=None), "EINVAL"), (dict(ve="a"), "EINVAL"), (dict(D=96), "EUNSUPPORTED"),
                                       (dict(s=(512, 128, 256, 128, 256, 100)), "EALIGN"), (dict(os=(512, 126)), "EALIGN"), (dict(n=1000), "EWORKSPACE")])
def test_decode_steps_that_are_refused(lib, address, over, code):
    over = {n: address if v == "a" else v for n, v in over.items()}
    assert _decode(lib, address, _pages(address), **over) == getattr(_lib, code)


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("over,code", [(dict(q=None), "EINVAL"), (dict(lens=None), "EINVAL"), (dict(out=None), "EINVAL"), (dict(ws=None), "EINVAL"), (dict(Hq=5), "EINVAL"), (dict(B=1), "EINVAL"),
                                       (dict(T=0), "EINVAL"), (dict(scale=0.0), "EINVAL"), (dict(flags=512), "EINVAL"), (dict(D=64), "EUNSUPPORTED"), (dict(qs=(512, 512, 100)), "EALIGN"),
                                       (dict(os=(512, 510, 128)), "EALIGN"), (dict(cu="a"), "EINVAL")])
def test_attends_that_are_refused(lib, address, few, over, code):
    over = {n: address if v == "a" else v for n, v in over.items()}
    assert _attend(lib, address, _pages(address), few, **over) == getattr(_lib, code)


def test_attend_refuses_broadcast_queries_and_few_refuses_many(lib, address):
    assert _attend(lib, address, _pages(address), T=40, qs=(512 * 40, 0, 128)) == _lib.EINVAL
    assert _attend(lib, address, _pages(address), T=40, qs=(0, 512, 128)) == _lib.EINVAL
    assert _attend(lib, address, _pages(address), few=True, T=5) == _lib.EUNSUPPORTED                # 5 x 2 heads of a group
    assert _attend(lib, address, _pages(address), few=True, n=100) == _lib.EWORKSPACE


def test_which_chunks_are_few(lib):
    rows = lib.daisy_b200_paged_attend_few_rows
    assert [rows(t, 3, 0, 16, 16) for t in (1, 8, 9)] == [1, 8, 0]
    assert [rows(t, 3, 0, 32, 8) for t in (1, 2, 3)] == [4, 8, 0]
    assert [rows(t, 8, 1, 16, 16) for t in (22, 32, 33)] == [22, 32, 0]      # packed: up to 32 ...
    assert [rows(t, 2, 1, 16, 16) for t in (8, 9)] == [8, 0]                 # ... and 4 a sequence on average
    assert rows(1, 3, 0, 16, 5) == 0 and rows(0, 3, 0, 16, 16) == 0


def test_workspaces_do_not_shrink_for_more(lib):
    d = lib.daisy_b200_paged_decode_workspace_bytes
    assert d(1, 6, 6, 128) < d(1000, 16, 16, 128) and d(1, 6, 4, 128) == 0 and d(0, 6, 6, 128) == 0 and d(1, 6, 6, 64) == 0
    w = lib.daisy_b200_paged_attend_workspace_bytes
    assert w(1, 100, 4, 16, 16) < w(1, 100000, 4, 16, 16) and w(1, 100, 4, 16, 5) == 0 and w(0, 100, 4, 16, 16) == 0


def test_binding_refuses_what_is_not_on_the_gpu():
    from daisy_b200 import B200PagedKVCache, ops
    pool, ids, x = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.paged_append(x, x, pool, pool, ids, ids[0], None, None)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.paged_decode_step(x, x, x, pool, pool, ids, ids[0], None, None, None)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.paged_attend(x, pool, pool, ids, ids[0], None)
    with pytest.raises(ValueError, match="no CPU path"):
        B200PagedKVCache(1, 4, 2, 128, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="16, 32"):
        B200PagedKVCache(1, 4, 2, 128, 1, 64, device="cuda", page=20)
    with pytest.raises(TypeError, match="float16"):
        B200PagedKVCache(1, 4, 2, 128, 1, 64, device="cuda", dtype=torch.float32)
