"""Borders of the paged cache where no GPU is needed."""
import pytest

from daisy_b200 import _lib
from daisy_b200.kv_cache import PageBook
from test_paged_host import _append, _attend, _decode, _pages, address, lib      # noqa: F401


def test_a_negative_limit_is_refused(lib, address):                              # noqa: F811
    for call in (_append, _decode, _attend, lambda *x: _attend(*x, few=True)):
        assert call(lib, address, _pages(address, max_len=-1)) == _lib.EINVAL


@pytest.mark.parametrize("over,call", [(dict(width=1 << 22, page=256, n_seq=64), dict(B=64)), (dict(width=1 << 21, page=256, n_seq=128, H=1), dict(B=1, T=32, Hq=1, cu="a")),
                                       (dict(width=1 << 26, n_seq=1, H=4), dict(B=1, T=32 // 4, Hq=4))])
def test_few_queries_over_a_table_of_too_many_blocks(lib, address, over, call):  # noqa: F811
    """Refused as unsupported before anything else is asked of the device: the caller takes the other form."""
    call = {k: address if v == "a" else v for k, v in call.items()}
    d = dict(width=4, page=16, n_seq=3, H=2)
    d.update(over)
    pages = _pages(address, p_sb=d["H"] * d["page"] * 128, p_sh=d["page"] * 128, **d)
    blocks = d["width"] * d["page"] // 64 * d["n_seq"] * d["H"] * -(-call.get("T", 1) * (call.get("Hq", 4) // d["H"]) // 8)
    assert lib.daisy_b200_paged_attend_few_rows(call.get("T", 1), d["n_seq"], int("cu" in call), call.get("Hq", 4), d["H"]) > 0
    got = _attend(lib, address, pages, few=True, **call)
    assert (got == _lib.EUNSUPPORTED) == (blocks >= 2 ** 31)


def _state(book):
    return list(book.length), [list(r) for r in book.table], list(book.free), list(book.first), list(book.end)


def test_a_refused_advance_changes_nothing():
    book = PageBook(6, 3, 40, 16)
    a, b, c = book.claim(), book.claim(), book.claim()
    book.reserve([a, b], [33, 40])
    before = _state(book)
    for slots, counts, what in (([a, c], [5, 5], "no pages for"), ([a, b], [5, 41], "the table holds 40"), ([b, a], [1, -1], "tokens"), ([a, 3], [1, 1], "holds no sequence"),
                                ([a, b], [1], "1 counts for 2 slots"), ([b, b], [30, 11], "the table holds 40")):
        with pytest.raises(ValueError, match=what):
            book.advance(slots, counts)
        assert _state(book) == before
    book.advance([a, b, a], [20, 40, 13])
    assert book.length == [33, 40, 0]


def test_reserve_adds_up_what_one_slot_asks_for():
    book = PageBook(6, 2, 64, 16)
    a, b = book.claim(), book.claim()
    assert book.reserve([a, a], [10, 10]) == [a] and book.end[a] == 2
    book.advance([a, a], [10, 10])
    before = _state(book)
    with pytest.raises(ValueError, match="20 . 50 tokens, the table holds 64"):
        book.reserve([b, a, a], [1, 25, 25])
    with pytest.raises(ValueError, match="2 counts for 1 slots"):
        book.reserve([b], [1, 1])
    with pytest.raises(RuntimeError, match="4 pages left"):
        book.reserve([b, a, b], [30, 40, 30])
    assert _state(book) == before


def test_forget_keeps_the_pages_of_tokens_to_come():
    """Only what is in the cache can be left behind: reserved pages that wait for their tokens stay."""
    book = PageBook(6, 1, 96, 16)
    a = book.claim()
    book.reserve([a], [80])
    book.advance([a], [33])
    assert book.forget(a, 1000) == [a] and book.first[a] == 2 and len(book.free) == 3
    assert all(p >= 0 for p in book.table[a][2:5])
    book.advance([a], [47])
    assert book.length[a] == 80


def test_results_that_share_rows_are_refused(lib, address):                      # noqa: F811
    for few in (False, True):
        for os in ((0, 512, 128), (512 * 4, 0, 128), (512 * 4, 512, 0)):
            assert _attend(lib, address, _pages(address), few=few, T=4, os=os) == _lib.EINVAL
    for os in ((0, 128), (512, 0)):
        assert _decode(lib, address, _pages(address), os=os) == _lib.EINVAL
