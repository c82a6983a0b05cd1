"""GPU tests of the cache in pages at its edges: numbers that are none in front of the nodes, sequences that were shortened, tensors that
share memory, starts that descend. The plain cache and the tolerances are those of test_paged_gpu.py."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from plain_pages import FULL, INVALID, PlainPages  # noqa: E402
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


class Shortened(PlainPages):
    """`reserve` replaces every page that others hold too among those that the new positions go to, not only the first: a sequence that
    was shortened has such pages behind its length."""

    def reserve(self, counts):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        want = []
        for s, n in enumerate(counts):
            if n <= 0:
                if n < 0:
                    self.status |= INVALID
                continue
            need, table = self._pages(self.lens[s] + n), self.table[s]
            if need > self.max_pages:
                self.status |= FULL
                return
            want += [(s, i) for i in range(self.lens[s] // self.page, need) if i >= len(table) or self.refs[table[i]] > 1]
        if len(want) > len(free):
            self.status |= FULL
            return
        for (s, i), new in zip(want, free):
            if i < len(self.table[s]):
                old, rows = self.table[s][i], max(0, self.lens[s] - i * self.page)
                for pool in (self.k, self.v):
                    pool[:, new, :, :rows] = pool[:, old, :, :rows]
                self.refs[old] -= 1
                self.table[s][i] = new
            else:
                self.table[s].append(new)
            self.refs[new] = 1


def shortened(paged, **how):
    b = Both(paged, **how)
    b.p.__class__ = Shortened
    return b


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,base", [(16, 20), (16, 32), (16, 0), (16, 47), (4, 13), (1, 11), (5, 25)])
def test_a_shortened_copy_goes_on(paged, dtype, page, base):
    """A fork whose length is taken back by more than a page, into a page or to its end: room for new positions is room that can be
    written, and what the other slots hold stays as it is."""
    b = shortened(paged, page=page, slots=3, pages=200, max_pages=80, dtype=dtype)
    b.fill([50, 7, 0])
    b.fork([0, 1, 0])
    b.keep([0, 0, 0], None, [50, 7, base])
    b.same()
    b.reserve([0, 0, 40])
    b.same()
    for layer in range(2):
        b.attend(layer, [0, 0, 40], 2)
    b.same()
    b.keep([0, 0, 40])
    b.attend(0, [0, 0, 0], 2)
    b.same()
    b.d.check()
    b.fork([2, 0, 0])  # all copies shortened, two of them go on at once
    b.keep([0, 0, 0], None, [base, 50, 50 - page])
    b.reserve([3 * page, 0, 2 * page + 1])
    b.same()
    for layer in range(2):
        b.append(layer, [3 * page, 0, 2 * page + 1])
    b.keep([3 * page, 0, 2 * page + 1])
    b.same()
    b.d.check()


def test_a_shortened_copy_without_free_pages(paged):
    """All pages or none: those that would be replaced count, too."""
    b = shortened(paged, page=4, slots=2, pages=7, max_pages=8)
    b.fill([16, 0])
    b.fork([0, 0])
    b.keep([0, 0], None, [16, 2])
    b.reserve([0, 15])  # pages 0 to 3 again and one more: five of three
    assert b.p.status == FULL
    b.same()
    b.d.status.zero_()
    b.p.status = 0
    b.reserve([0, 10])  # three of three
    assert b.same().p.status == 0 and min(b.p.refs) == 1


@pytest.mark.parametrize("page,dim", [(16, 64), (4, 7), (1, 16)])
def test_pages_over_many_steps_with_shortening(paged, page, dim):
    b = shortened(paged, page=page, dim=dim, pages=60, slots=5, max_pages=14, seed=page)
    r = b.rng
    for step in range(60):
        kind = r.choice(["grow", "grow", "fork", "free", "shorten"])
        if kind == "grow":
            counts = [r.choice([0, 1, r.randint(1, 3 * page)]) for _ in range(5)]
            b.reserve(counts)
            if b.p.status & FULL:
                b.same()
                b.d.status.zero_()
                b.p.status = 0
                continue
            for layer in range(2):
                b.append(layer, counts)
            b.keep(counts)
        elif kind == "fork":
            b.fork([r.choice([s, r.randrange(-1, 5)]) for s in range(5)])
        elif kind == "free":
            gone = [int(r.random() < 0.2) for _ in range(5)]
            b.d.free(ints(gone))
            b.p.fork([-1 if x else s for s, x in enumerate(gone)])
        else:
            b.keep([0] * 5, None, [r.choice([n, r.randint(0, n)]) for n in b.p.lens])
        b.same()
        assert b.p.status == 0


def test_many_shared_pages_behind_a_shortened_sequence(paged):
    """More of them than a warp takes at a time, in more slots than a round."""
    slots = 1100
    b = shortened(paged, layers=1, heads=1, dim=2, page=1, slots=slots, pages=40000, max_pages=100)
    b.reserve([90] + [0] * (slots - 1))
    b.append(0, [90] + [0] * (slots - 1))
    b.keep([90] + [0] * (slots - 1))
    b.fork([0 if s % 3 == 0 else s for s in range(slots)])
    b.keep([0] * slots, None, [(s * 7) % 90 if s % 3 == 0 else 0 for s in range(slots)])
    b.reserve([100 - (s * 7) % 90 if s % 3 == 0 else s % 4 for s in range(slots)])
    b.same()
    assert b.p.status == 0


@pytest.mark.parametrize("dtype,dim,groups", [(F32, 64, 2), (F32, 30, 2), (BF16, 64, 1), (F16, 128, 12), (BF16, 256, 2), (F16, 200, 9)])
def test_starts_that_descend(paged, dtype, dim, groups):
    """Slots that claim one another's rows: nothing is computed, the status says so, and the next call is as ever."""
    b = Both(paged, layers=1, heads=1, dim=dim, slots=3, page=16, pages=80, max_pages=20, dtype=dtype)
    b.fill([100, 30, 70])
    b.reserve([8, 8, 8])
    q, k, v = b.randn(8, groups, dim), b.randn(8, 1, dim), b.randn(8, 1, dim)
    plain = b.d.attend(0, q, ints([0, 3, 5, 8]), k, v)
    for starts in ([0, 8, 0, 8], [8, 0, 4, 8], [0, 5, 3, 8], [0, 8, 8, 7]):
        out = torch.full_like(q, 3.0)
        b.d.attend(0, q, ints(starts), k, v, out=out)
        assert int(b.d.status.item()) == INVALID and bool((out == 3).all())
        b.d.status.zero_()
    assert torch.equal(plain, b.d.attend(0, q, ints([0, 3, 5, 8]), k, v))
    b.d.check()


def test_starts_that_descend_over_long_sequences(paged):
    """256 slots of a million positions, every other one with all of 8000 rows: more work than 32 bits count."""
    slots, rows, length = 256, 8000, 1 << 20
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    k = torch.zeros(1, 2, 8, 1024, 8, dtype=BF16, device="cuda")
    c = paged.PagedCache.over(k, k.clone(), z(slots, 1040), z(slots) + length, z(slots) + 1040, z(2) + 1)
    q = torch.zeros(rows, 64, 8, dtype=BF16, device="cuda")
    new = torch.zeros(rows, 8, 8, dtype=BF16, device="cuda")
    out = torch.full_like(q, 3.0)
    c.attend(0, q, ints([0, rows] * (slots // 2) + [rows]), new, new, out=out)
    assert int(c.status.item()) & INVALID and bool((out == 3).all())


def test_check_says_that_a_wait_ran_out(paged):
    """A kernel that gives up a wait leaves it in the device's status word: check() reads that, too, and once."""
    from ytensor_b200 import _lib
    L = _lib.lib()
    b = Both(paged, layers=1, heads=1, slots=1)
    b.d.check()
    old, waited = L.ytcuda_get_wait_limit(), torch.zeros(1, dtype=torch.int64, device="cuda")
    _lib.check(L.ytcuda_set_wait_limit(2_000_000))  # about a millisecond
    try:
        for also in (False, True):
            _lib.check(L.ytcuda_wait_probe(waited.data_ptr(), torch.cuda.current_stream().cuda_stream))
            if also:
                b.d.keep(ints([1]))  # a row without a page
            with pytest.raises(_lib.YtCudaError, match="wait ran out.*tree that is none" if also else "wait ran out") as e:
                b.d.check()
            assert e.value.status == _lib.TIMEOUT
            b.d.check()
    finally:
        _lib.check(L.ytcuda_set_wait_limit(old))


def numpy_of(t, base):
    """The same places of a numpy array that torch's strides give, over the storage of `base`."""
    size, flat = t.element_size(), np.zeros(base.untyped_storage().nbytes() // t.element_size(), f"u{t.element_size()}")
    return np.lib.stride_tricks.as_strided(flat[t.storage_offset():], t.shape, [x * size for x in t.stride()]), flat


def meet(x, y):
    """Whether two views of one storage have an element in common."""
    seen = []
    for t in (x, y):
        view, flat = numpy_of(t, x)
        view[...] = 1
        seen.append(flat)
    return bool((seen[0] & seen[1]).any())


VIEWS = {  # two views of one tensor, [layers, pages, heads, page, dim] each
    "pages": ((2, 24, 2, 4, 16), lambda t: (t[:, :12], t[:, 12:])),
    "pages that overlap": ((2, 24, 2, 4, 16), lambda t: (t[:, :12], t[:, 11:])),
    "layers": ((4, 12, 2, 4, 16), lambda t: (t[:2], t[2:])),
    "the same": ((2, 12, 2, 4, 16), lambda t: (t, t)),
    "layers that overlap": ((3, 12, 2, 4, 16), lambda t: (t[:2], t[1:])),
    "every other page": ((2, 24, 2, 4, 16), lambda t: (t[:, ::2], t[:, 1::2])),
    "every other page, and all from one on": ((2, 24, 2, 4, 16), lambda t: (t[:, ::2], t[:, 3:])),
    "heads": ((2, 12, 4, 4, 16), lambda t: (t[:, :, :2], t[:, :, 2:])),
    "heads that overlap": ((2, 12, 3, 4, 16), lambda t: (t[:, :, :2], t[:, :, 1:])),
    "rows of a page": ((2, 12, 2, 8, 16), lambda t: (t[:, :, :, ::2], t[:, :, :, 1::2])),
    "halves of a row": ((2, 12, 2, 4, 32), lambda t: (t[..., :16], t[..., 16:])),
    "halves of a row that overlap": ((2, 12, 2, 4, 31), lambda t: (t[..., :16], t[..., 15:])),
    "heads behind positions": ((2, 24, 4, 2, 16), lambda t: (t[:, :12].transpose(2, 3), t[:, 12:].transpose(2, 3))),
    "one order in the other": ((2, 12, 4, 4, 16), lambda t: (t[:, :10], t[:, 2:].transpose(2, 3))),
}


@pytest.mark.parametrize("which", VIEWS)
@pytest.mark.parametrize("pool", ["k", "v", "k and v"])
def test_caches_that_are_views_of_one_pool(paged, which, pool):
    """compact() takes two of them that have no element in common, whatever their strides, and refuses them otherwise."""
    shape, views = VIEWS[which]
    g = torch.Generator(device="cuda").manual_seed(1)
    whole = torch.randn(shape, generator=g, device="cuda").to(BF16)
    mine, theirs = views(whole)
    if pool == "k":
        kv, into = (mine, mine.clone()), (theirs, theirs.clone())
    elif pool == "v":
        kv, into = (mine.clone(), mine), (theirs.clone(), theirs)
    else:  # keys of one beside values of the other
        kv, into = (mine, mine.clone()), (theirs.clone(), theirs)
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    a = paged.PagedCache.over(*kv, z(2, 6), z(2), z(2), z(kv[0].shape[1]))
    b = paged.PagedCache.over(*into, z(2, 6), z(2), z(2), z(into[0].shape[1]))
    fresh = paged.PagedCache(*into[0].shape[:2], a.page, a.kv_heads, a.dim, 2, 6)
    a.reserve(ints([3 * a.page - 1, 2 * a.page]))
    a.keep(ints([3 * a.page - 1, 2 * a.page]))
    a.compact(fresh)
    if meet(mine, theirs):
        with pytest.raises(ValueError, match="share memory"):
            a.compact(b)
        return
    a.compact(b)
    for cache in (a, b, fresh):
        cache.check()
    assert torch.equal(b.k[:, :5], fresh.k[:, :5]) and torch.equal(b.v[:, :5], fresh.v[:, :5])
    assert torch.equal(b.refs, fresh.refs) and torch.equal(b.lens, fresh.lens)
    assert all(torch.equal(b.table[s, :n], fresh.table[s, :n]) for s, n in ((0, 3), (1, 2)))


def test_caches_that_share_counts(paged):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    k = lambda: torch.zeros(1, 8, 1, 4, 16, device="cuda")  # noqa: E731
    space = z(100)
    part = lambda at, *s: space[at:at + math.prod(s)].view(s)  # noqa: E731
    a = paged.PagedCache.over(k(), k(), part(0, 2, 5), part(10, 2), part(12, 2), part(14, 8))
    for at in ((30, 42, 44, 46), (22, 32, 34, 36)):
        a.compact(paged.PagedCache.over(k(), k(), part(at[0], 2, 5), part(at[1], 2), part(at[2], 2), part(at[3], 8)))
    for at in ((21, 42, 44, 46), (30, 9, 44, 46), (30, 42, 13, 46), (30, 42, 44, 7), (30, 12, 44, 46), (0, 42, 44, 46)):
        with pytest.raises(ValueError, match="share memory"):
            a.compact(paged.PagedCache.over(k(), k(), part(at[0], 2, 5), part(at[1], 2), part(at[2], 2), part(at[3], 8)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_results_in_the_tensor_of_the_queries(paged, dtype):
    """`out` may be a slice of the tensor that q, k and v are slices of, but has no element in common with them."""
    b = Both(paged, layers=1, heads=2, dim=64, slots=1, page=16, pages=40, max_pages=30, dtype=dtype)
    b.fill([100])
    b.reserve([6])
    starts, whole = ints([0, 6]), b.randn(12, 12, 64)
    want = None
    for q, k, v, out in (
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[:6, 8:]),           # beside them
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[6:, :4]),           # behind them
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[:6, 7:11]),         # a head of v
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[:6, 3:7]),          # q, k and v
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[5:11, 4:8]),        # a row of k and v
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[5:11, 8:]),
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[:6, :4]),           # q
            (lambda t: t[:6, :4], lambda t: t[:6, 4:6], lambda t: t[:6, 6:8], lambda t: t[1:7, :4])):
        t = whole.clone()
        x, y, z, o = q(t), k(t), v(t), out(t)
        if any(meet(o, i) for i in (x, y, z)):
            with pytest.raises(ValueError, match="shares memory"):
                b.d.attend(0, x, starts, y, z, out=o)
            assert torch.equal(t, whole)
        else:
            want = b.d.attend(0, x.clone(), starts, y.clone(), z.clone()) if want is None else want
            assert torch.equal(b.d.attend(0, x, starts, y, z, out=o), want)
    # keys and values that are in the pages already: only q counts
    t = whole.clone()
    assert torch.equal(b.d.attend(0, t[:6, :4], starts, out=t[:6, 4:8]), want)


def test_results_that_lie_in_one_another(paged):
    """Rows and heads of `out` are each written by some CTA: they may stand in any order, but not in one another."""
    b = Both(paged, layers=1, heads=2, dim=64, slots=1, page=16, pages=20, max_pages=8)
    b.fill([40])
    b.reserve([5])
    q, k, starts = b.randn(5, 4, 64), b.randn(5, 2, 64), ints([0, 5])
    want = b.d.attend(0, q, starts, k, k)
    for strides in ((256, 64, 1), (64, 320, 1), (400, 80, 1), (512, 128, 1), (72, 400, 1)):
        out = torch.zeros(4000, dtype=BF16, device="cuda").as_strided((5, 4, 64), strides)
        assert torch.equal(b.d.attend(0, q, starts, k, k, out=out), want)
    for strides in ((0, 64, 1), (256, 0, 1), (192, 64, 1), (256, 63, 1), (64, 64, 1), (32, 320, 1)):
        out = torch.zeros(4000, dtype=BF16, device="cuda").as_strided((5, 4, 64), strides)
        with pytest.raises(ValueError, match="lie in one another"):
            b.d.attend(0, q, starts, k, k, out=out)
        assert not bool(out.any())
    one = torch.zeros(4000, dtype=BF16, device="cuda").as_strided((1, 4, 64), (0, 64, 1))  # (a single row's stride says nothing)
    b.d.attend(0, q[:1], ints([0, 1]), k[:1], k[:1], out=one)


def test_more_slots_than_a_grid_is_high(paged):
    slots = 70001
    c = paged.PagedCache(1, slots, 4, 1, 8, slots, 1, BF16)
    two, starts = torch.full((slots,), 2, dtype=torch.int32, device="cuda"), torch.arange(0, 2 * slots + 1, 2, dtype=torch.int32, device="cuda")
    k = torch.arange(2 * slots * 8, device="cuda").view(2 * slots, 1, 8).remainder(251).to(BF16)
    v = k + 1
    c.reserve(two)
    c.append(0, k, v, starts)
    take = torch.arange(slots, device="cuda") % 2  # every slot keeps one row, the first or the second
    c.keep(torch.ones_like(two), take.to(torch.int32).view(slots, 1))
    c.check()
    rows = torch.arange(slots, device="cuda") * 2 + take
    assert torch.equal(c.k[0, :, 0, 0], k[rows, 0]) and torch.equal(c.v[0, :, 0, 0], v[rows, 0]) and bool((c.lens == 1).all())
    c.keep(two)
    c.check()
    assert bool((c.lens == 3).all())
    c.fork(torch.arange(slots, dtype=torch.int32, device="cuda").flip(0))
    c.keep(torch.zeros_like(two))
    c.reserve(torch.ones_like(two))
    c.check()
    assert torch.equal(c.k[0, c.table[:, 0].long(), 0, 0], k[rows, 0].flip(0))
    q = k[:slots, :, :]
    one = torch.arange(slots + 1, dtype=torch.int32, device="cuda")
    out = c.attend(0, q, one, k[:slots], v[:slots])
    c.check()
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim,groups", [(64, 1), (128, 4), (256, 2), (64, 20), (128, 32), (256, 17), (128, 140), (30, 2), (30, 9)])
def test_many_small_weights_beside_large_ones(paged, dtype, dim, groups):
    """Sixteen keys with a weight of one and a value of zero, 8000 with weights of 2^-25.5 and values of one: what is left of the small
    ones is the whole result. Tolerance: fp16 weights, of which the largest are 2^7 or more, are off by 2^-25 at most where they are
    below 2^-14, so by 2^-32 of the largest; else as ever."""
    n, slots, scale = 8000, 200, 1.0
    page, heads = 32, 1
    c = paged.PagedCache(1, n // page + slots + 9, page, heads, dim, slots, n // page + 1, dtype)
    starts = torch.tensor([0] + [n] * slots, dtype=torch.int32, device="cuda")
    counts = ints([n] + [0] * (slots - 1))
    k, v = torch.zeros(n, 1, dim, dtype=dtype, device="cuda"), torch.ones(n, 1, dim, dtype=dtype, device="cuda")
    heavy = torch.arange(0, 256, 16, device="cuda")  # one for every warp, stream and block of keys
    k[heavy, 0, 0], v[heavy] = 4.421875, 0.0
    c.reserve(counts)
    c.append(0, k, v, starts)
    c.keep(counts)
    c.fork(torch.zeros(slots, dtype=torch.int32, device="cuda"))
    one = torch.ones(slots, dtype=torch.int32, device="cuda")
    c.reserve(one)
    q = torch.zeros(slots, groups, dim, dtype=dtype, device="cuda")
    q[..., 0] = 4.0
    new = torch.zeros(slots, 1, dim, dtype=dtype, device="cuda")
    got = c.attend(0, q, torch.arange(slots + 1, dtype=torch.int32, device="cuda"), new, new + 1, scale=scale)
    c.check()
    w = math.exp(-4.0 * float(torch.tensor(4.421875, dtype=dtype)))
    small = n + 1 - 16
    want = small * w / (16 + small * w)
    tol = (torch.finfo(dtype).eps if dtype != F32 else 0) * want * 1.01 + (n * 2.0 ** -32 if dtype == F16 else 0)
    tol += 2 * (10 * math.sqrt(dim) * 17.7 + 10 * math.sqrt(n)) * 2.0 ** -24 * want
    assert float((got.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("dtype,dim,groups", FORMS)
@pytest.mark.parametrize("tree", [True, False])
def test_the_largest_numbers_in_hidden_places(paged, dtype, dim, groups, tree):
    """A hidden value may be the largest or lowest finite number: it has no part in the rows that do not see it."""
    b = Both(paged, layers=1, heads=1, dim=dim, slots=2, page=16, pages=60, max_pages=30, dtype=dtype)
    b.fill([200, 18])
    b.reserve([6, 3])
    q, k, v = b.randn(9, groups, dim), b.randn(9, 1, dim), b.randn(9, 1, dim)
    starts, parents = ints([0, 6, 9]), ints([-1, 0, 0, 1, 2, -1, -1, 0, -1]) if tree else None
    plain = b.d.attend(0, q, starts, k, v, parents=parents)
    for huge in (torch.finfo(dtype).max, torch.finfo(dtype).min):
        k2, v2 = k.clone(), v.clone()
        v2[5], k2[5], v2[8, 0, 3] = huge, 0, huge  # only the last nodes of the slots see them
        got = b.d.attend(0, q, starts, k2, v2, parents=parents)
        rest = [0, 1, 2, 3, 4, 6, 7]
        assert torch.equal(got[rest], plain[rest])
        if dtype != F32:  # a weight of the node's own of 1 / 206 or so: the result is as large, and finite
            assert bool((got[5] * math.copysign(1, huge) > torch.finfo(dtype).max / 1e7).all()) and bool(torch.isfinite(got[[5, 8]]).all())
