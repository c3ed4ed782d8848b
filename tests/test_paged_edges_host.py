"""Borders of the paged cache where no GPU is needed."""
import pytest

from daisy_b200 import _lib
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
