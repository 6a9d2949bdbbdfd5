"""Limits of the 8-bit cache's entries and Python classes that need no GPU: what they refuse, and what they leave behind."""
import pytest

from stratacuda_b200 import _lib as L
from test_kv8_host import A, CALLS, cache, refuse
from stratacuda_b200 import kv8


@pytest.mark.parametrize("top", [0x7fffffff // 64 + 1, 1 << 30, 0x7fffffff])
def test_attend_refuses_longer_lists_than_a_table_has_blocks(top):
    """A list is walked with 32-bit indices some steps past its end."""
    assert refuse(kv8.StrataRangeError, "top", lambda: CALLS["attend"](cache(), picks=A, top=top)) == L.ERR_RANGE


@pytest.mark.parametrize("count,heads", [(1 << 24, 128), (1 << 20, 2048), (1 << 16, 32768), ((1 << 24) - 1, 129)])
def test_attend_refuses_runs_of_more_rows_than_32_bits_count(count, heads):
    """A prompt's rows, tokens times query heads a key/value head, are counted in 32 bits."""
    assert refuse(kv8.StrataRangeError, "2\\^31", lambda: CALLS["attend"](cache(kv_heads=1, dim=1), count=count, heads=heads)) == L.ERR_RANGE
