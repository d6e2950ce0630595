"""mk_rope_tables refuses positions past 2^31 wherever they begin, without a device."""
import pytest

import malkin_amd as mk_
from test_kv4_refusals import refused, tables


@pytest.mark.parametrize("first,n", [(2 ** 63 - 1, 1), (2 ** 63 - 1, 2 ** 31 - 1), (2 ** 63 - 10, 10), (2 ** 62, 5), (2 ** 31 + 1, 0),
                                     (2 ** 31, 1), (2, 2 ** 31 - 1), (-2 ** 63, 3)])
def test_refused(first, n):
    refused(tables(first=first, n=n), mk_.MK_ERR_INVALID, "positions")


@pytest.mark.parametrize("first,n", [(1, 2 ** 31 - 1), (2 ** 31 - 1, 1), (0, 1)])
def test_taken(first, n):
    refused(tables(first=first, n=n), mk_.MK_ERR_INVALID, "null context")
