"""Borders of the paged cache where no GPU is needed."""
import pytest

from daisy_b200 import _lib
from test_paged_host import _append, _attend, _decode, _pages, address, lib      # noqa: F401


def test_a_negative_limit_is_refused(lib, address):                              # noqa: F811
    for call in (_append, _decode, _attend, lambda *x: _attend(*x, few=True)):
        assert call(lib, address, _pages(address, max_len=-1)) == _lib.EINVAL
