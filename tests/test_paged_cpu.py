"""CPU: what the entry points of the cache in pages refuse before they touch the device, and the sizes that they ask for."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from ytensor_b200 import _lib  # noqa: E402
from ytensor_b200.paged import PagedCache, _Pages  # noqa: E402

HERE = C.create_string_buffer(64)


def cache(**change):
    at = (C.addressof(HERE) + 15) // 16 * 16
    c = _Pages(at, at, (64, 64, 64, 64), (64, 64, 64, 64), at, at, at, at, at, at, 2, 8, 4, 2, 64, 3, 4, _lib.BF16)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def calls(c, at):
    L, st = _lib.lib(), (C.c_int64 * 8)(*[128, 64] * 4)
    yield L.ytcuda_pages_reserve(c, at, None)
    yield L.ytcuda_pages_append(c, 0, at, at, st, at, 1, None)
    yield L.ytcuda_pages_attend(c, 0, at, at + 16, None, None, st, at, None, 1, 2, 0.0, at, 1 << 40, None)
    yield L.ytcuda_pages_keep(c, at, None, 0, None, None)
    yield L.ytcuda_pages_fork(c, at, None, None)
    yield L.ytcuda_pages_compact(c, c, None)


@pytest.mark.parametrize("change", [dict(dtype=3), dict(layers=0), dict(pages=-1), dict(page=0), dict(kv_heads=0), dict(dim=0),
                                    dict(slots=-1), dict(max_pages=-1), dict(k=None), dict(refs=None), dict(scratch=None),
                                    dict(status=None), dict(page=65537), dict(dim=1 << 17), dict(slots=1 << 20, max_pages=1 << 12),
                                    dict(k_strides=(64, 64, 64, -1)), dict(pages=0)])
def test_bad_caches(change):
    at = (C.addressof(HERE) + 15) // 16 * 16
    c = cache(**change)
    assert all(rc == _lib.INVALID_ARG for rc in calls(C.addressof(c), at))
    assert all(rc == _lib.INVALID_ARG for rc in calls(None, at))


@pytest.mark.parametrize("change", [dict(layers=1 << 14, kv_heads=1 << 10, dim=4), dict(layers=1 << 16, kv_heads=8, dim=64, page=1 << 15),
                                    dict(pages=1 << 30), dict(slots=1 << 30, max_pages=1)])
def test_extents_above_the_limits(change):
    at = (C.addressof(HERE) + 15) // 16 * 16
    c = cache(**change)
    assert all(rc == _lib.INVALID_ARG for rc in calls(C.addressof(c), at))


def test_bad_arguments():
    L, st = _lib.lib(), (C.c_int64 * 8)(*[128, 64] * 4)
    at = (C.addressof(HERE) + 15) // 16 * 16
    c = cache()
    p = C.addressof(c)
    attend = lambda layer=0, q=at, k=None, v=None, o=at + 16, strides=st, starts=at, rows=1, heads=2, work=at, size=1 << 40: (  # noqa: E731
        L.ytcuda_pages_attend(p, layer, q, o, k, v, strides, starts, None, rows, heads, 0.0, work, size, None))
    for change in (dict(layer=2), dict(layer=-1), dict(q=None), dict(k=at), dict(v=at), dict(o=None), dict(o=at), dict(starts=None), dict(strides=None),
                   dict(rows=-1), dict(heads=3), dict(heads=0), dict(work=None), dict(size=16), dict(work=at + 4), dict(q=at + 1)):
        assert attend(**change) == _lib.INVALID_ARG, change
    assert attend(rows=0) == _lib.OK
    for rc in (L.ytcuda_pages_reserve(p, None, None), L.ytcuda_pages_append(p, 2, at, at, st, at, 1, None),
               L.ytcuda_pages_append(p, 0, None, at, st, at, 1, None), L.ytcuda_pages_append(p, 0, at, at, st, None, 1, None),
               L.ytcuda_pages_append(p, 0, at, at, None, at, 1, None), L.ytcuda_pages_append(p, 0, at, at, st, at, -1, None), L.ytcuda_pages_keep(p, None, None, 0, None, None),
               L.ytcuda_pages_keep(p, at, at, -1, None, None), L.ytcuda_pages_fork(p, at, at, None),
               L.ytcuda_pages_fork(p, None, None, None), L.ytcuda_pages_compact(p, None, None), L.ytcuda_pages_compact(p, p, None)):
        assert rc == _lib.INVALID_ARG
    other = cache(dim=32)
    assert L.ytcuda_pages_compact(p, C.addressof(other), None) == _lib.INVALID_ARG
    empty = cache(slots=0)
    assert L.ytcuda_pages_reserve(C.addressof(empty), at, None) == _lib.OK
    big = cache(dim=264)
    assert L.ytcuda_pages_attend(C.addressof(big), 0, at, at + 16, None, None, st, at, None, 1, 2, 0.0, at, 1 << 40, None) == _lib.UNSUPPORTED


def test_sizes():
    L = _lib.lib()
    c = cache()
    assert L.ytcuda_pages_scratch(C.addressof(c)) % 16 == 0 and L.ytcuda_pages_scratch(None) == 0
    small = L.ytcuda_pages_attend_workspace(C.addressof(c), 1, 2)
    assert small > 0 and L.ytcuda_pages_attend_workspace(C.addressof(c), 500, 16) >= small
    assert L.ytcuda_pages_attend_workspace(C.addressof(c), 0, 2) == 0


def test_tensors_off_the_device():
    z = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(1, 4, 2, 4, 8)
    with pytest.raises(ValueError):
        PagedCache.over(k, k.clone(), z(3, 4), z(3), z(3), z(4))
    with pytest.raises(ValueError):
        PagedCache.over(k, k[:, :2], z(3, 4), z(3), z(3), z(4))
