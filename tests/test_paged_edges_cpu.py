"""CPU: what the calls of the cache in pages say of sizes that they do not take."""
import ctypes as C

from test_paged_cpu import HERE, cache
from ytensor_b200 import _lib


def test_a_table_that_is_too_long_for_one_call():
    """The number of positions in the message is the table's, above 32 bits too."""
    L, st = _lib.lib(), (C.c_int64 * 8)(*[128, 64] * 4)
    at = (C.addressof(HERE) + 15) // 16 * 16
    c = cache(slots=1, max_pages=1 << 26, page=1 << 12, kv_heads=1, pages=8)
    rc = L.ytcuda_pages_attend(C.addressof(c), 0, at, at + (1 << 20), None, None, st, at, None, 1000, 2, 0.0, at, 1 << 40, None)
    assert rc == _lib.UNSUPPORTED
    assert f"1000 rows over tables of {1 << 38} positions" in _lib.last_error()
