"""GPU tests of the cache in pages at its edges: numbers that are none in front of the nodes, sequences that were shortened, tensors that
share memory, starts that descend. The plain cache and the tolerances are those of test_paged_gpu.py."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import BF16, F16, F32, Both, ints, paged  # noqa: E402,F401

# every form: narrow, tcgen05 with one row block and two, wide, element by element
FORMS = [(F32, 64, 2), (F32, 30, 2), (BF16, 64, 2), (F16, 128, 2), (BF16, 64, 8), (F16, 128, 12), (BF16, 128, 40), (F16, 64, 40), (BF16, 256, 2),
         (F16, 200, 9), (BF16, 30, 9)]


@pytest.mark.parametrize("dtype,dim,groups", FORMS)
@pytest.mark.parametrize("length,places", [(70, [40]), (70, [0]), (300, [10]), (300, [290]), (300, [200, 260, 299]), (1, [0]), (127, [126]), (128, [127]),
                                           (2000, [1990, 3])])
@pytest.mark.parametrize("tree", [True, False])
def test_numbers_in_seen_places(paged, dtype, dim, groups, length, places, tree):
    """Infinities and NaN of the sequence's own positions reach every row, wherever they lie beside the nodes' tile; so do they where a hidden
    node's value is none, too."""
    b = Both(paged, layers=1, heads=1, dim=dim, slots=2, page=16, pages=200, max_pages=150, dtype=dtype, seed=length)
    b.fill([length, 33])
    b.reserve([6, 3])
    q, k, v = b.randn(9, groups, dim), b.randn(9, 1, dim), b.randn(9, 1, dim)
    starts, parents = ints([0, 6, 9]), ints([-1, 0, 0, 1, 2, -1, -1, 0, -1]) if tree else None
    plain = b.d.attend(0, q, starts, k, v, parents=parents)
    kept = b.d.v.clone()
    for bad in (math.nan, math.inf, -math.inf):
        for hidden in (False, True):
            v2 = v.clone()
            if hidden:
                v2[5, 0, 7] = bad  # only node 5 of slot 0 sees it
            b.d.v.copy_(kept)
            for i, at in enumerate(places):
                b.d.v[0, int(b.d.table[0, at // 16]), 0, at % 16, i] = bad
            b.d.append(0, k, v2, starts)
            for fresh in (True, False):
                got = b.d.attend(0, q, starts, k if fresh else None, v2 if fresh else None, parents=parents)
                wrong = torch.zeros_like(got, dtype=torch.bool)
                wrong[:6, :, :len(places)] = True
                wrong[5, :, 7] |= hidden
                assert torch.equal(got[~wrong], plain[~wrong])
                if dtype == F32:  # (an infinity is NaN there)
                    assert not bool(torch.isfinite(got[wrong]).any())
                else:
                    assert bool(torch.isnan(got[wrong]).all()) if math.isnan(bad) else bool((got[wrong] == bad).all())
    # a key that is no number: every weight of every row is none
    b.d.v.copy_(kept)
    b.d.k[0, int(b.d.table[0, places[0] // 16]), 0, places[0] % 16, 1] = math.nan
    got = b.d.attend(0, q, starts, k, v, parents=parents)
    assert bool(torch.isnan(got[:6]).all()) and torch.equal(got[6:], plain[6:])


@pytest.mark.parametrize("dtype,dim,groups", [(BF16, 64, 1), (F16, 128, 4), (BF16, 128, 12)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_one_number_that_is_none_in_a_deep_tree(paged, dtype, dim, groups, bad):
    """1024 nodes, most of them in one line, and a value that those behind it see: the rows are right and the call is not given up."""
    n = 1024
    b = Both(paged, layers=1, heads=2, dim=dim, slots=2, page=32, pages=160, max_pages=100, dtype=dtype, seed=groups)
    b.fill([300, 70])
    b.reserve([n, 40])
    q, k, v = b.randn(n + 40, 2 * groups, dim), b.randn(n + 40, 2, dim), b.randn(n + 40, 2, dim)
    parents = [max(-1, i - (2 if i % 50 == 7 else 1)) for i in range(n)] + [i - 1 for i in range(40)]
    starts, up = ints([0, n, n + 40]), ints(parents)
    plain = b.d.attend(0, q, starts, k, v, parents=up)
    for node in (0, 6, 500):
        v2 = v.clone()
        v2[node, 1, dim - 3] = bad
        got = b.d.attend(0, q, starts, k, v2, parents=up)
        wrong = torch.zeros_like(got, dtype=torch.bool)
        sees = [False] * n
        for i in range(n):
            sees[i] = i == node or (parents[i] >= 0 and sees[parents[i]])
        wrong[:n, groups:, dim - 3] = torch.tensor(sees, device="cuda")[:, None]
        assert torch.equal(got[~wrong], plain[~wrong])
        assert bool(torch.isnan(got[wrong]).all()) if math.isnan(bad) else bool((got[wrong] == bad).all())
    from ytensor_b200 import _lib
    assert _lib.lib().ytcuda_device_status(None) == _lib.OK


@pytest.mark.parametrize("dtype,dim,groups", [(BF16, 64, 1), (F16, 128, 4), (BF16, 128, 4)])
def test_one_number_that_is_none_in_a_long_chain(paged, dtype, dim, groups):
    """A prompt of thousands of tokens: rows from the number on, and no others."""
    n, node, bad = 6000, 2500, math.nan
    b = Both(paged, layers=1, heads=1, dim=dim, slots=1, page=128, pages=60, max_pages=60, dtype=dtype)
    b.fill([200])
    b.reserve([n])
    q, k, v = b.randn(n, groups, dim), b.randn(n, 1, dim), b.randn(n, 1, dim)
    starts = ints([0, n])
    plain = b.d.attend(0, q, starts, k, v)
    v2 = v.clone()
    v2[node, 0, 11] = bad
    got = b.d.attend(0, q, starts, k, v2)
    wrong = torch.zeros_like(got, dtype=torch.bool)
    wrong[node:, :, 11] = True
    assert bool(torch.isnan(got[wrong]).all()) and torch.equal(got[~wrong], plain[~wrong])
    from ytensor_b200 import _lib
    assert _lib.lib().ytcuda_device_status(None) == _lib.OK
