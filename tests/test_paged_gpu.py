"""GPU tests of the cache in pages (ytensor_b200.paged) against plain_pages.py in 64 bits.

Tolerances. Page operations move bits and count: equal. Attention, element by element, relative to A = sum of p |v| over the
row's weights p (so |o| <= A):
  fp32 arithmetic  a score of dim products is off by at most 5 sqrt(dim) u S with u = 2^-24, S the row's sum of |q||k| scale
                   (rounding errors that are independent, five deviations); a weight by that in the numerator and in the sum;
                   the sums over n positions by 5 sqrt(n) u each: (10 sqrt(dim) S + 10 sqrt(n)) u A, and as much again for the
                   factor log2(e) and the exponentials
  16-bit types     half a step eps / 2 of the result, and of every weight where they are operands of a matrix instruction:
                   eps A; fp16 weights below 2^-14 are off by 2^-25 at most, each times |v| (n 2^-25 max|v|)"""
import math
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from plain_pages import FULL, INVALID, SHARED, PlainPages  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from ytensor_b200 import paged
    return paged


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def host(t):
    return t.detach().double().cpu().numpy()


class Both:
    """The same cache twice: on the device and plainly. Rows that nothing was written to are NaN in both."""

    def __init__(self, paged, *, layers=2, pages=64, page=16, heads=2, dim=64, slots=3, max_pages=16, dtype=BF16, layout="heads",
                 seed=0):
        self.g, self.dtype = torch.Generator(device="cuda").manual_seed(seed), dtype
        self.rng = random.Random(seed)
        shape = (layers, pages, heads, page, dim)
        if layout == "heads":
            make = lambda: torch.full(shape, math.nan, dtype=dtype, device="cuda")  # noqa: E731
        elif layout == "rows":  # [layers, pages, page, heads, dim]
            make = lambda: torch.full((layers, pages, page, heads, dim), math.nan, dtype=dtype, device="cuda").transpose(2, 3)  # noqa: E731
        elif layout == "far":  # 1.6 GB from page to page: offsets in bytes and in elements pass 32 bits
            stride = (1600 << 20) // torch.finfo(dtype).bits * 8
            space = torch.empty(layers * pages * stride, dtype=dtype, device="cuda")
            make = lambda: space.as_strided(shape, (pages * stride, stride, page * dim, dim, 1), space_at.pop()).fill_(math.nan)  # noqa: E731
            space_at = [stride // 2, 0]  # (values half way between keys)
        else:  # odd strides: no row starts on more than an element's boundary
            make = lambda: torch.full((*shape[:-1], dim + 3), math.nan, dtype=dtype, device="cuda")[..., 1:dim + 1]  # noqa: E731
        zeros = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.d = paged.PagedCache.over(make(), make(), zeros(slots, max_pages), zeros(slots), zeros(slots), zeros(pages))
        self.p = PlainPages(layers, pages, page, heads, dim, slots, max_pages)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda").to(self.dtype)

    def reserve(self, counts):
        self.d.reserve(ints(counts))
        self.p.reserve(counts)

    def fork(self, source):
        self.d.fork(ints(source))
        self.p.fork(source)

    def keep(self, kept, accepted=None, base=None):
        self.d.keep(ints(kept), None if accepted is None else ints(accepted), base=None if base is None else ints(base))
        self.p.keep(kept, accepted, base)

    def append(self, layer, counts):
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        k, v = (self.randn(starts[-1], self.p.heads, self.p.dim) for _ in range(2))
        self.d.append(layer, k, v, ints(starts))
        self.p.append(layer, host(k), host(v), starts)

    def fill(self, lens):
        """Sequences of the given lengths, pages anywhere."""
        order = list(range(self.p.slots))
        left = list(lens)
        while any(left):  # in pieces, slot by slot in a random order, so that the pages are not in theirs
            self.rng.shuffle(order)
            for s in order:
                n = min(left[s], self.rng.randint(1, 3 * self.p.page))
                if n:
                    counts = [n if i == s else 0 for i in range(self.p.slots)]
                    self.reserve(counts)
                    for layer in range(self.p.layers):
                        self.append(layer, counts)
                    self.keep(counts)
                    left[s] -= n

    def attend(self, layer, counts, groups=2, tree=True, fresh=True, scale=0.0, parents=None, extra=0, sharp=1.0):
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        rows, H, D = starts[-1] + extra, self.p.heads, self.p.dim
        # q, k and v are slices of one projection
        qkv = self.randn(rows, (groups + 2) * H, D)
        q, k, v = qkv[:, :groups * H] * sharp, qkv[:, groups * H:(groups + 1) * H], qkv[:, (groups + 1) * H:]
        if tree and parents is None:
            parents = [max(-1, i - 1 - self.rng.randrange(4)) for n in counts for i in range(n)]
        parents = parents if tree else None
        dp = None if parents is None else ints(list(parents) + [-1] * extra)
        if not fresh:
            self.d.append(layer, k, v, ints(starts))
        out = torch.full((rows, groups * H, D), 7.0, dtype=self.dtype, device="cuda")
        got = self.d.attend(layer, q, ints(starts), k if fresh else None, v if fresh else None, parents=dp, scale=scale, out=out)
        assert got is out
        want, size, big = self.p.attend(layer, host(q), starts, parents, host(k), host(v), scale)
        self.p.append(layer, host(k), host(v), starts)
        self.near(got[:starts[-1]], want[:starts[-1]], size[:starts[-1]], big, max(l + n for l, n in zip(self.p.lens, counts)))
        assert torch.equal(got[starts[-1]:], torch.full_like(got[starts[-1]:], 7.0))  # rows behind the last sequence
        return got

    def near(self, got, want, size, big, n):
        D, u = self.p.dim, 2.0 ** -24
        tol = 2 * (10 * math.sqrt(D) * big + 10 * math.sqrt(n)) * u * size
        if self.dtype != F32:
            tol = tol + torch.finfo(self.dtype).eps * size * 1.01
        if self.dtype == F16:
            tol = tol + n * 2.0 ** -25 * np.nanmax(np.abs(self.p.v), initial=4.0)
        err = np.abs(host(got) - want)
        assert np.all(err <= tol), f"off by {np.max(err / np.maximum(tol, 1e-300))} tolerances"

    def same(self):
        """Every count and every bit."""
        d, p = self.d, self.p
        assert d.lens.tolist() == p.lens and d.held.tolist() == p.held and d.refs.tolist() == p.refs
        table = d.table.tolist()
        assert [row[:h] for row, h in zip(table, p.held)] == p.table
        for x, y in ((d.k, p.k), (d.v, p.v)):
            assert np.array_equal(host(x), y, equal_nan=True)
        assert int(d.status.item()) == p.status
        return self


DTYPES = [F32, BF16, F16]


# ---------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("layout,page,dim", [("heads", 16, 64), ("rows", 5, 24), ("odd", 4, 7), ("heads", 1, 16), ("rows", 64, 130)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_over_many_steps(paged, dtype, layout, page, dim):
    """Random sequences of all the operations: every count, table and bit as in the plain cache."""
    b = Both(paged, page=page, dim=dim, layout=layout, dtype=dtype, pages=40, slots=5, max_pages=12, seed=page)
    other = Both(paged, page=page, dim=dim, layout="heads", dtype=dtype, pages=40, slots=5, max_pages=12)
    r = b.rng
    for step in range(40):
        kind = r.choice(["grow", "grow", "grow", "draft", "fork", "free", "compact"])
        if kind in ("grow", "draft"):
            counts = [r.choice([0, 1, r.randint(1, 2 * page)]) for _ in range(5)]
            before = [list(t) for t in b.p.table]
            b.reserve(counts)
            if b.p.status & FULL:
                assert before == b.p.table
                b.same()
                b.d.status.zero_()
                b.p.status = 0
                continue
            for layer in range(2):
                b.append(layer, counts)
            if kind == "grow":
                b.keep(counts)
            else:
                rows = [sorted(r.sample(range(n), r.randint(0, n))) for n in counts]
                depth = max(1, max(map(len, rows)))
                b.keep([len(x) for x in rows], [x + [0] * (depth - len(x)) for x in rows])
        elif kind == "fork":
            b.fork([r.choice([s, r.randrange(-1, 5)]) for s in range(5)])
        elif kind == "free":
            gone = [int(r.random() < 0.3) for _ in range(5)]
            b.d.free(ints(gone))
            b.p.fork([-1 if x else s for s, x in enumerate(gone)])
        else:
            b.d.compact(other.d)
            b.p.compact(other.p)
            other.same()
            b, other = other, b
        b.same()


def test_more_slots_and_pages_than_a_pass(paged):
    """The counting kernels go through slots and pages in rounds."""
    b = Both(paged, layers=1, pages=20001, page=1, heads=1, dim=2, slots=1500, max_pages=9)
    b.reserve([s % 7 for s in range(1500)])
    b.append(0, [s % 7 for s in range(1500)])
    b.keep([s % 7 for s in range(1500)])
    b.same()
    b.fork([s - 1 if s % 3 == 0 else s for s in range(1500)])
    b.same()
    b.reserve([2 if s % 11 else 0 for s in range(1500)])
    b.same()
    other = Both(paged, layers=1, pages=9000, page=1, heads=1, dim=2, slots=1500, max_pages=9)
    b.d.compact(other.d)
    b.p.compact(other.p)
    other.same()


def test_beams_share_and_copy(paged):
    b = Both(paged, slots=4, page=16)
    b.fill([37, 0, 0, 0])
    used = sum(r > 0 for r in b.p.refs)
    b.fork([0, 0, 0, 0])
    assert sum(r > 0 for r in b.same().p.refs) == used
    b.reserve([1, 1, 0, 1])  # three of four beams go on: each gets the written rows of the last page
    b.same()
    for layer in range(2):
        b.append(layer, [1, 1, 0, 1])
    b.keep([1, 1, 0, 1])
    b.same()
    b.fork([3, 3, -1, 0])
    b.same()


def test_a_full_pool_changes_nothing(paged):
    b = Both(paged, pages=5, page=4, slots=2, max_pages=8)
    b.fill([9, 0])
    b.fork([0, 0])
    b.reserve([1, 12])  # a copy and three pages: one too many for the two that are free
    assert b.p.status == FULL
    b.same()
    with pytest.raises(Exception, match="too few free pages"):
        b.d.check()
    b.d.check()
    b.p.status = 0
    b.reserve([33, 0])  # more pages than a row of the table has
    assert b.p.status == FULL
    b.same()
    small = Both(paged, pages=2, page=4, slots=2, max_pages=8)
    b.d.compact(small.d)
    b.p.compact(small.p)
    assert small.p.status == FULL
    small.same()


def test_what_only_the_device_sees(paged):
    b = Both(paged, pages=8, page=4, slots=3, max_pages=4)
    b.fill([6, 3, 0])
    b.append(0, [5, 1, 1])  # past the pages of slots 0 and 2
    assert b.p.status == INVALID
    b.same()
    for do in (lambda: b.fork([7, 1, -5]), lambda: b.reserve([-1, 1, 0]), lambda: b.keep([3, 0, 1]), lambda: b.keep([2, -1, 0]),
               lambda: b.keep([2, 0, 0], [[1, 1], [0, 0], [0, 0]]), lambda: b.keep([1, 0, 0], [[9], [0], [0]]),
               lambda: b.keep([3, 0, 0], [[0, 1], [0, 0], [0, 0]]), lambda: b.keep([1, 0, 0], None, [-4, 3, 0])):
        b.d.status.zero_()
        b.p.status = 0
        do()
        assert b.p.status == INVALID
        b.same()
    b.d.status.zero_()
    b.p.status = 0
    b.keep([0, 0, 0], None, [5, 3, 0])
    b.fork([0, 0, 0])
    b.append(1, [1, 0, 0])  # a page that three slots hold
    assert b.p.status == SHARED
    b.same()
    b.keep([1, 0, 0], [[1], [0], [0]])
    b.same()


def test_pages_that_do_not_exist(paged):
    """Numbers of pages outside the pool in the table are not followed."""
    b = Both(paged, pages=8, page=4, slots=2, max_pages=4)
    b.fill([8, 4])
    b.d.table[0, 1], b.d.table[1, 0] = 99, -3
    k = b.d.k.clone()
    q = b.randn(2, 4, 64)
    b.d.attend(0, q, ints([0, 1, 2]), b.randn(2, 2, 64), b.randn(2, 2, 64))
    b.d.append(0, b.randn(2, 2, 64), b.randn(2, 2, 64), ints([0, 1, 2]))
    b.d.reserve(ints([1, 1]))
    b.d.keep(ints([0, 0]))
    b.d.fork(ints([1, 0]))
    other = Both(paged, pages=8, page=4, slots=2, max_pages=4)
    b.d.compact(other.d)
    assert int(b.d.status.item()) & INVALID and int(other.d.status.item()) == INVALID
    assert torch.equal(torch.nan_to_num(b.d.k), torch.nan_to_num(k))


@pytest.mark.parametrize("dtype,groups", [(F32, 2), (BF16, 2), (BF16, 40), (F16, 40)])
def test_attention_reads_zeros_where_a_page_does_not_exist(paged, dtype, groups):
    b = Both(paged, layers=1, heads=1, dim=64, page=16, pages=40, slots=1, max_pages=40, dtype=dtype)
    b.fill([400])
    b.reserve([3])
    for i, pg in ((3, 40), (9, -2), (17, 1 << 30)):
        b.p.k[:, b.p.table[0][i]] = b.p.v[:, b.p.table[0][i]] = 0
        b.d.table[0, i] = pg
    q, k, v = b.randn(3, groups, 64), b.randn(3, 1, 64), b.randn(3, 1, 64)
    got = b.d.attend(0, q, ints([0, 3]), k, v)
    assert int(b.d.status.item()) == INVALID
    want, size, big = b.p.attend(0, host(q), [0, 3], None, host(k), host(v))
    b.near(got, want, size, big, 403)


def test_base_of_kept_rows(paged):
    b = Both(paged, slots=2, page=4)
    b.fill([10, 5])
    b.reserve([6, 3])
    for layer in range(2):
        b.append(layer, [6, 3])
    for _ in range(2):  # from the same base twice
        b.keep([3, 2], [[0, 2, 5], [1, 2, 0]], [10, 5])
        b.same()
    b.keep([0, 0], None, [8, 0])
    b.same()


# ---------------------------------------------------------------------------------------------- attention
CASES = [  # slots' lengths, nodes, heads, groups, dim, page
    ([5], [1], 1, 1, 64, 16),
    ([0], [1], 2, 2, 128, 16),
    ([1000], [1], 8, 2, 128, 16),
    ([0, 1, 15, 16, 17, 200], [1, 1, 1, 1, 1, 1], 2, 4, 128, 16),
    ([70, 0, 33], [13, 4, 0], 2, 2, 128, 16),
    ([129, 64, 63], [1, 31, 33], 1, 8, 64, 24),
    ([300, 20], [64, 7], 2, 4, 128, 32),
    ([90, 500], [20, 3], 1, 3, 80, 16),
    ([40, 7], [9, 2], 2, 1, 256, 8),
    ([11, 3], [5, 6], 2, 2, 36, 3),
    ([11, 3], [5, 6], 1, 5, 7, 1),
    ([260], [130], 1, 4, 64, 128),
]


@pytest.mark.parametrize("lens,nodes,heads,groups,dim,page", CASES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tree", [True, False])
def test_attend(paged, dtype, tree, lens, nodes, heads, groups, dim, page):
    n = sum(-(-(l + m) // page) for l, m in zip(lens, nodes))
    b = Both(paged, heads=heads, dim=dim, page=page, pages=n + 9, slots=len(lens), max_pages=n + 1, dtype=dtype, seed=dim + page)
    b.fill(lens)
    b.reserve(nodes)
    b.attend(1, nodes, groups, tree, fresh=True, extra=3)
    b.same()
    b.attend(1, nodes, groups, tree, fresh=False)
    b.same()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout,dim,page", [("rows", 64, 16), ("odd", 64, 16), ("rows", 128, 5), ("odd", 12, 4)])
def test_attend_over_other_layouts(paged, dtype, layout, dim, page):
    b = Both(paged, heads=3, dim=dim, page=page, pages=99, slots=3, max_pages=60, dtype=dtype, layout=layout)
    b.fill([50, 0, 131])
    b.reserve([6, 3, 9])
    b.attend(0, [6, 3, 9], 2)
    b.same()


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_chains_and_long_sequences(paged, dtype):
    """A piece of a prompt behind a sequence (more nodes than a tree may have), and one slot that all CTAs share."""
    b = Both(paged, layers=1, heads=1, dim=64, page=64, pages=120, slots=2, max_pages=110, dtype=dtype)
    b.fill([300, 0])
    b.reserve([1100, 40])
    b.attend(0, [1100, 40], 2, tree=False)
    b.keep([1100, 40])
    b.reserve([3000, 1])
    b.append(0, [3000, 0])
    b.keep([3000, 0])
    b.reserve([2, 1])
    b.attend(0, [2, 1], 4)
    b.same()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_trees_of_every_shape(paged, dtype):
    """A chain, a star, two roots, the widest tree, a deep one."""
    n = 1024
    b = Both(paged, layers=1, heads=1, dim=64, page=64, pages=40, slots=1, max_pages=40, dtype=dtype)
    b.fill([100])
    b.reserve([n])
    for parents in ([-1, 0, 1, 2], [-1, 0, 0, 0], [-1, -1, 0, 1], [-1] * 5, [-1], [-1] + [(i - 1) // 2 for i in range(1, n)],
                    list(range(-1, n - 1)), [-1, 0, -1, 2, 1, 4, 3]):
        b.attend(0, [len(parents)], 1, parents=parents)
    b.same()


def test_bad_trees(paged):
    """Parents that are none count as -1; a tree of too many nodes is left out: its rows are not written."""
    b = Both(paged, layers=1, heads=1, dim=64, page=64, pages=40, slots=2, max_pages=20)
    b.fill([20, 30])
    b.reserve([1025, 4])
    q, kv = b.randn(1029, 2, 64), b.randn(1029, 1, 64)
    out = torch.full_like(q, 3.0)
    b.d.attend(0, q, ints([0, 1025, 1029]), kv, kv, parents=ints([-1] * 1029), out=out)
    assert int(b.d.status.item()) == INVALID
    assert bool((out[:1025] == 3).all()) and bool((out[1025:] != 3).any())
    b.d.status.zero_()
    for parents in ([0, 0, 1, 5], [-7, 0, 1, -1]):
        right = [-1, 0, 1, -1]
        x = b.d.attend(0, q[:4], ints([0, 0, 4]), kv[:4], kv[:4], parents=ints(parents))
        assert int(b.d.status.item()) == INVALID
        b.d.status.zero_()
        assert torch.equal(x, b.d.attend(0, q[:4], ints([0, 0, 4]), kv[:4], kv[:4], parents=ints(right)))
        b.d.check()
    for starts in ([0, 5, 2], [-1, 2, 4], [0, 2, 9]):  # not rows of the call
        out = torch.full_like(q[:4], 3.0)
        b.d.attend(0, q[:4], ints(starts), kv[:4], kv[:4], out=out)
        assert int(b.d.status.item()) == INVALID
        b.d.status.zero_()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,groups", [(64, 2), (64, 8), (64, 30), (128, 40), (256, 8)])
def test_sharp_scores_and_scales(paged, dtype, dim, groups):
    b = Both(paged, heads=2, dim=dim, pages=60, slots=2, dtype=dtype, max_pages=30)
    b.fill([300, 77])
    b.reserve([7, 2])
    for scale, sharp in ((0.0, 30.0), (1.0, 1.0), (-0.5, 1.0), (1e-6, 1.0)):
        b.attend(0, [7, 2], groups, scale=scale, sharp=sharp)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page", [1, 7, 8, 16, 24, 48, 64, 100, 128, 256])
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_many_rows_over_every_page(paged, dtype, page, dim):
    """Whole key tiles by TMA boxes of what divides a page, or row by row; one row tile and two, in one piece and in several."""
    b = Both(paged, layers=2, heads=2, dim=dim, page=page, pages=3300 // page + 20, slots=4, max_pages=1400 // page + 6, dtype=dtype, seed=page)
    b.fill([700, 0, 128, 1279])
    b.reserve([20, 40, 9, 65])
    b.attend(1, [20, 40, 9, 65], 4)
    b.attend(1, [20, 0, 9, 65], 4, tree=False)
    b.same()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,groups", [(64, 2), (20, 2), (64, 8), (64, 40), (128, 40), (128, 2), (128, 7), (80, 33), (256, 2), (256, 9)])
def test_numbers_in_hidden_places(paged, dtype, dim, groups):
    """What a node does not see may be infinite or no number: siblings, rows behind the end, pages of others."""
    b = Both(paged, layers=1, heads=1, dim=dim, slots=2, page=16, dtype=dtype)
    b.fill([30, 18])
    b.reserve([5, 3])
    q, k, v = b.randn(8, groups, dim), b.randn(8, 1, dim), b.randn(8, 1, dim)
    parents = [-1, 0, 0, 1, 2, -1, 0, -1]
    starts = [0, 5, 8]
    plain = b.d.attend(0, q, ints(starts), k, v, parents=ints(parents))
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[2], v2[2] = bad, bad  # nodes 2 and 4 of slot 0 see it
        v2[7, 0, 3] = bad        # node 2 of slot 1 sees it
        got = b.d.attend(0, q, ints(starts), k2, v2, parents=ints(parents))
        for row in range(8):
            if row in (2, 4):
                assert not bool(torch.isfinite(got[row]).any())
            elif row == 7:
                assert not bool(torch.isfinite(got[row, :, 3]).any())
            else:
                assert torch.equal(got[row], plain[row]), row


@pytest.mark.parametrize("dtype,dim,groups", [(F32, 64, 1), (F32, 20, 2), (BF16, 64, 1), (BF16, 64, 4), (F16, 128, 3), (BF16, 128, 12), (BF16, 30, 4),
                                              (BF16, 256, 2), (F16, 200, 5)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_numbers_in_hidden_places_of_a_chain(paged, dtype, dim, groups, bad):
    """Pieces of prompts: what is no number reaches the rows that see it, whole tiles of keys behind it, and no row in front."""
    b = Both(paged, layers=1, heads=1, dim=dim, slots=3, page=32, pages=60, max_pages=30, dtype=dtype)
    b.fill([70, 0, 5])
    b.reserve([500, 333, 3])
    q, k, v = b.randn(836, groups, dim), b.randn(836, 1, dim), b.randn(836, 1, dim)
    starts = ints([0, 500, 833, 836])
    plain = b.d.attend(0, q, starts, k, v)
    v2 = v.clone()
    v2[100, 0, 5] = v2[300, 0, 3] = v2[700, 0, 2] = bad
    got = b.d.attend(0, q, starts, k, v2)
    touched = torch.zeros(836, dim, dtype=torch.bool, device="cuda")
    touched[100:500, 5] = touched[300:500, 3] = touched[700:833, 2] = True
    touched = touched[:, None].expand_as(got)
    assert not bool(torch.isfinite(got[touched]).any())
    assert torch.equal(got[~touched], plain[~touched])


@pytest.mark.parametrize("dtype,groups", [(F32, 4), (BF16, 4), (BF16, 16), (F16, 16)])
def test_results_are_the_same_every_time(paged, dtype, groups):
    """The same call twice gives the same bits."""
    b = Both(paged, heads=2, dim=128, pages=200, slots=3, max_pages=150, dtype=dtype)
    b.fill([700, 45, 1300])
    b.reserve([9, 1, 30])
    q, k, v = b.randn(40, 2 * groups, 128), b.randn(40, 2, 128), b.randn(40, 2, 128)
    first = b.d.attend(0, q, ints([0, 9, 10, 40]), k, v)
    for _ in range(20):
        assert torch.equal(first, b.d.attend(0, q, ints([0, 9, 10, 40]), k, v))


@pytest.mark.parametrize("dtype,dim,groups", [(BF16, 64, 2), (BF16, 64, 30), (F16, 128, 30), (BF16, 256, 30), (F16, 256, 2), (F32, 128, 2),
                                              (F32, 30, 3), (BF16, 30, 9)])
def test_offsets_above_32_bits(paged, dtype, dim, groups):
    b = Both(paged, layers=2, heads=2, dim=dim, page=32, pages=7, slots=2, max_pages=6, dtype=dtype, layout="far")
    b.fill([90, 20])
    b.reserve([5, 8])
    b.attend(1, [5, 8], groups)
    b.append(0, [5, 8])
    b.keep([3, 4], [[0, 2, 4, 0], [1, 2, 5, 7]])
    b.attend(1, [1, 3], groups)
    b.fork([0, 0])
    b.reserve([7, 9])
    b.append(0, [7, 9])
    b.attend(1, [7, 9], groups)
    b.keep([7, 9])
    b.same()
    other = Both(paged, layers=2, heads=2, dim=dim, page=32, pages=7, slots=2, max_pages=6, dtype=dtype)
    b.d.compact(other.d)
    b.p.compact(other.p)
    other.same()
    torch.cuda.empty_cache()


def test_accepted_without_columns(paged):
    """No row can be kept of none: a kept row is refused, as it is of a shorter list."""
    b = Both(paged, pages=20, page=4, slots=3, max_pages=4)
    b.fill([3, 5, 2])
    b.reserve([2, 2, 2])
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    b.d.keep(ints([0, 1, 0]), none)
    assert b.d.lens.tolist() == [3, 5, 2]
    with pytest.raises(RuntimeError):
        b.d.check()
    b.d.keep(ints([0, 0, 0]), none, base=ints([2, 4, 0]))
    assert b.d.lens.tolist() == [2, 4, 0]
    b.d.check()


def test_rows_of_q_that_overlap(paged):
    """Queries are only read: they may lie in one another, and the result is a tensor of its own."""
    b = Both(paged, layers=1, heads=2, dim=64, page=16, pages=20, slots=1, max_pages=8)
    b.fill([40])
    b.reserve([5])
    flat = b.randn(400)
    k = b.randn(5, 2, 64)
    for strides in ((1, 1, 1), (1, 64, 1), (0, 64, 1), (64, 0, 1), (0, 0, 1)):
        q = flat.as_strided((5, 2, 64), strides)
        got = b.d.attend(0, q, ints([0, 5]), k, k)
        assert got.stride(2) == 1
        b.near(got, *b.p.attend(0, host(q), [0, 5], None, host(k), host(k), 0.0), 45)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nodes,groups", [(1, 1), (1, 7), (5, 3), (16, 1), (33, 2), (64, 5), (200, 3)])
@pytest.mark.parametrize("dim", [64, 130, 256])
def test_one_sequence_over_all_processors(paged, dtype, nodes, groups, dim):
    """One key head: every tile of rows is cut into as many pieces as there are keys for."""
    b = Both(paged, layers=1, heads=1, dim=dim, page=64, pages=180, slots=1, max_pages=180, dtype=dtype, seed=nodes)
    b.fill([900])
    b.reserve([9000])
    b.append(0, [9000])
    b.keep([9000])
    b.reserve([nodes])
    b.attend(0, [nodes], groups)
    b.same()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups", [2, 12])
def test_attend_over_many_slots(paged, dtype, groups):
    """More slots than lanes, idle ones among them, ragged lengths."""
    slots = 70
    lens, nodes = [(s * 37) % 90 for s in range(slots)], [s % 4 for s in range(slots)]
    b = Both(paged, layers=1, heads=2, dim=64, page=16, pages=600, slots=slots, max_pages=8, dtype=dtype)
    b.reserve(lens)
    b.append(0, lens)
    b.keep(lens)
    b.reserve(nodes)
    b.attend(0, nodes, groups, tree=True, extra=2)
    b.attend(0, [0] * 69 + [3], groups, tree=False)
    b.same()


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_speculative_steps(paged, dtype):
    """Draft, attend, accept, beam by beam: at the end every slot's keys are those of its own history, and attention over the
    pages is attention over that history."""
    b = Both(paged, layers=2, heads=2, dim=64, page=8, pages=90, slots=4, max_pages=30, dtype=dtype, seed=5)
    b.fill([21, 8, 0, 40])
    r = b.rng
    for step in range(8):
        counts = [r.choice([0, 1, 6, 12]) for _ in range(4)]
        b.reserve(counts)
        parents = [max(-1, i - 1 - r.randrange(3)) for n in counts for i in range(n)]
        for layer in range(2):
            b.attend(layer, counts, 2, parents=parents)
        rows, at = [], 0
        for n in counts:  # the path to some node
            path, j = [], r.randrange(n) if n else -1
            while j >= 0:
                path.append(j)
                j = parents[at + j]
            rows.append(path[::-1])
            at += n
        depth = max(1, max(map(len, rows)))
        b.keep([len(x) for x in rows], [x + [0] * (depth - len(x)) for x in rows])
        if step % 3 == 2:
            b.fork([r.choice([s, s, r.randrange(4)]) for s in range(4)])
        b.same()
        b.d.check()


def test_a_captured_step_serves_any_lengths(paged):
    """One graph of a whole step, replayed while the sequences grow; two graphs of the same layer share no workspace."""
    b = Both(paged, layers=1, heads=2, dim=64, page=8, pages=60, slots=2, max_pages=25)
    b.fill([5, 30])
    q, k, v = b.randn(6, 4, 64), b.randn(6, 2, 64), b.randn(6, 2, 64)
    starts, counts, parents = ints([0, 4, 6]), ints([4, 2]), ints([-1, 0, 0, 1, -1, 0])
    kept, accepted = ints([2, 1]), ints([[0, 2], [0, 0]])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                b.d.reserve(counts)
                outs.append(b.d.attend(0, q, starts, k, v, parents=parents))
                b.d.keep(kept, accepted)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(stream)
    for step in range(6):
        q.copy_(b.randn(6, 4, 64)), k.copy_(b.randn(6, 2, 64)), v.copy_(b.randn(6, 2, 64))
        graphs[step % 2].replay()
        b.p.reserve([4, 2])
        want, size, big = b.p.attend(0, host(q), [0, 4, 6], [-1, 0, 0, 1, -1, 0], host(k), host(v))
        b.near(outs[step % 2], want, size, big, 200)
        b.p.append(0, host(k), host(v), [0, 4, 6])
        b.p.keep([2, 1], [[0, 2], [0, 0]])
        b.same()


def test_captured_page_operations(paged):
    """append, fork, free and compact in one graph, replayed on other states."""
    b = Both(paged, layers=2, heads=2, dim=64, page=4, pages=60, slots=3, max_pages=12)
    other = Both(paged, layers=2, heads=2, dim=64, page=4, pages=50, slots=3, max_pages=12)
    b.fill([9, 5, 0])
    k, v, starts = b.randn(3, 2, 64), b.randn(3, 2, 64), [0, 2, 3, 3]
    source, gone, kept, counts, dstarts = ints([0, 0, 1]), ints([0, 1, 0]), ints([2, 1, 0]), ints([2, 1, 1]), ints(starts)
    g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=stream):
        b.d.reserve(counts)
        b.d.append(1, k, v, dstarts)
        b.d.keep(kept)
        b.d.fork(source)
        b.d.free(gone)
        b.d.compact(other.d)
    torch.cuda.current_stream().wait_stream(stream)
    for step in range(4):
        k.copy_(b.randn(3, 2, 64))
        source.copy_(ints([[0, 0, 1], [2, 1, 0], [1, 0, 2], [-1, 2, 2]][step]))
        g.replay()
        b.p.reserve([2, 1, 1])
        b.p.append(1, host(k), host(v), starts)
        b.p.keep([2, 1, 0])
        b.p.fork([[0, 0, 1], [2, 1, 0], [1, 0, 2], [-1, 2, 2]][step])
        b.p.fork([0, -1, 2])
        b.p.compact(other.p)
        b.same()
        other.same()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout,dim,heads,groups", [("rows", 128, 3, 20), ("rows", 64, 1, 40), ("odd", 64, 2, 20), ("rows", 256, 2, 10)])
def test_many_rows_over_other_layouts(paged, dtype, layout, dim, heads, groups):
    b = Both(paged, heads=heads, dim=dim, page=16, pages=99, slots=3, max_pages=60, dtype=dtype, layout=layout)
    b.fill([400, 0, 131])
    b.reserve([6, 3, 9])
    b.attend(0, [6, 3, 9], groups)
    b.same()


def test_an_axis_of_one_element_has_any_stride(paged):
    """One head, one layer: their strides say nothing, and the result is that of the plain layout."""
    b = Both(paged, layers=1, heads=1, dim=64, page=16, pages=20, slots=1)
    b.fill([100])
    b.reserve([20])
    q, kv = b.randn(20, 4, 64), b.randn(20, 1, 64)
    want = b.d.attend(0, q, ints([0, 20]), kv, kv)
    odd = paged.PagedCache.over(*(x.as_strided(x.shape, (3, x.stride(1), 5, x.stride(3), 1)) for x in (b.d.k, b.d.v)), b.d.table,
                                b.d.lens, b.d.held, b.d.refs)
    assert torch.equal(want, odd.attend(0, q, ints([0, 20]), kv, kv))


def test_two_streams_and_two_graphs_at_once(paged):
    """Attention in two layers at the same time."""
    b = Both(paged, layers=2, heads=2, dim=128, page=16, pages=420, slots=2, max_pages=210)
    b.fill([3000, 1500])
    b.reserve([3, 2])
    q, k, v = b.randn(5, 8, 128), b.randn(5, 2, 128), b.randn(5, 2, 128)
    starts = ints([0, 3, 5])
    want = [b.d.attend(layer, q, starts, k, v) for layer in range(2)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for _ in range(20):
        for layer, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs.append((layer, b.d.attend(layer, q, starts, k, v)))
    torch.cuda.synchronize()
    for layer in range(2):  # both captured on one stream, replayed on two
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            outs.append((layer, b.d.attend(layer, q, starts, k, v)))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[layer]) for layer, o in outs)


def test_refusals(paged):
    b = Both(paged, layers=2, heads=2, dim=64, slots=3)
    c, st = b.d, ints([0, 1, 2, 3])
    q, k = b.randn(3, 4, 64), b.randn(3, 2, 64)
    bad = ValueError
    for call in (lambda: c.attend(2, q, st, k, k), lambda: c.attend(-1, q, st, k, k), lambda: c.attend(0, q[:, :3], st, k, k),
                 lambda: c.attend(0, q.float(), st, k, k), lambda: c.attend(0, q, st[:3], k, k), lambda: c.attend(0, q, st.long(), k, k),
                 lambda: c.attend(0, q, st, k), lambda: c.attend(0, q, st, k[:2], k[:2]), lambda: c.attend(0, q, st, k, k, out=q),
                 lambda: c.attend(0, q, st, k, k, parents=st[:2]), lambda: c.attend(0, q, st.cpu(), k, k),
                 lambda: c.attend(0, q.transpose(1, 2)[:, :, :4], st, k, k), lambda: c.attend(0, q[0], st),
                 lambda: c.append(0, k, k[:2], st), lambda: c.append(5, k, k, st), lambda: c.reserve(st), lambda: c.reserve(st[:3].cpu()),
                 lambda: c.fork(st[:2]), lambda: c.free(st), lambda: c.keep(st), lambda: c.keep(st[:3], st), lambda: c.keep(st[:3], base=st),
                 lambda: c.compact(c), lambda: c.compact(Both(paged, layers=1, heads=2, dim=64, slots=3).d)):
        with pytest.raises(bad):
            call()
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    for over in (lambda: paged.PagedCache.over(c.k[0], c.v[0], c.table, c.lens, c.held, c.refs),
                 lambda: paged.PagedCache.over(c.k, c.v.float(), c.table, c.lens, c.held, c.refs),
                 lambda: paged.PagedCache.over(c.k[..., ::2], c.v[..., ::2], c.table, c.lens, c.held, c.refs),
                 lambda: paged.PagedCache.over(c.k, c.v, c.table[:2], c.lens, c.held, c.refs),
                 lambda: paged.PagedCache.over(c.k, c.v, c.table, c.lens, c.held, z(3)),
                 lambda: paged.PagedCache.over(c.k, c.v, c.table.long(), c.lens, c.held, c.refs),
                 lambda: paged.PagedCache.over(c.k.cpu(), c.v.cpu(), c.table, c.lens, c.held, c.refs),
                 lambda: paged.PagedCache.over(*(x.cpu() for x in (c.k, c.v, c.table, c.lens, c.held, c.refs)))):
        with pytest.raises(bad):
            over()
    with pytest.raises(bad):
        paged.PagedCache(1, 4, 4, 0, 64, 1, 4)
    wide = paged.PagedCache(1, 4, 4, 1, 264, 1, 4)
    with pytest.raises(bad, match="at most 256"):
        wide.attend(0, torch.zeros(1, 1, 264, dtype=BF16, device="cuda"), ints([0, 1]))
    # nothing to do: no launch
    from ytensor_b200._lib import lib
    n = lib().ytcuda_launch_count()
    assert c.attend(0, q[:0], st, k[:0], k[:0]).shape == (0, 4, 64)
    c.append(0, k[:0], k[:0], st)
    assert lib().ytcuda_launch_count() == n
