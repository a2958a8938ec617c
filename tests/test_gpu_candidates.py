"""The operators that decode several candidates of a chunk (shared-prefix attention, paged tails, logit penalties) against
plain implementations in 64 bits (tests/candidates_ref.py), and a decode that uses them together."""

import random

import numpy as np
import pytest
import torch

from candidates_ref import PoolRef, attend_bounds, attend_ref, penalize_ref

pytestmark = pytest.mark.gpu

BF, HF, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32
INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _errors_clear():
    from viktor_b200._lib import check_device_errors
    yield
    torch.cuda.synchronize()
    check_device_errors()


def i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


# ------------------------------------------------------------------------------------------------ attention
class Attend:
    """Inputs of one call; what lies behind every length holds NaN, and the table behind a row's last page nonsense."""

    def __init__(self, seed, dtype, heads, sizes, lens, tails, page, S=None, pad=0, n_pages=None, nonsense=True):
        H, HK, D = heads
        g = torch.Generator("cuda").manual_seed(seed)
        rs = np.random.RandomState(seed)
        B, P, S = sum(sizes) + pad, len(sizes), S or max(1, *lens)

        def randn(*shape):
            return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)

        self.q, self.k, self.v = randn(B, H, D) * 1.5, randn(P, S, HK, D), randn(P, S, HK, D)
        need = [-(-t // page) for t in tails] + [0] * pad
        n_pages = n_pages or max(1, sum(need)) + 2
        self.kp, self.vp = randn(n_pages, page, HK, D), randn(n_pages, page, HK, D)
        table = np.full((B, max(1, *need) + 1), 2 ** 31 - 1 if nonsense else 0, dtype=np.int64)
        free = rs.permutation(n_pages)
        for b, n in enumerate(need):
            table[b, :n], free = free[:n], free[n:]
        if nonsense:
            for x in (self.k, self.v):
                x[torch.arange(S, device="cuda")[None] >= i32(lens)[:, None]] = NAN
            keep = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
            for b, t in enumerate(tails):
                for j in range(need[b]):
                    keep[table[b, j], :min(page, t - j * page)] = True
            for x in (self.kp, self.vp):
                x[~keep] = NAN
        self.table, self.lens, self.tails = i32(table), i32(lens), i32(list(tails) + [1] * pad)
        self.offsets, self.pad = i32(np.concatenate([[0], np.cumsum(sizes)])), pad
        self.most = max(lens) + max([0, *tails])

    def args(self):
        return self.q, self.k, self.v, self.lens, self.offsets, self.kp, self.vp, self.table, self.tails

    def check(self, scale=None, args=None):
        from viktor_b200.ops import shared_prefix_attention
        args = self.args() if args is None else args
        out = torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device="cuda")
        got, lse = shared_prefix_attention(*args, scale=scale, out=out, return_lse=True)
        n, D = self.q.shape[0] - self.pad, self.q.shape[2]
        want, want_lse, spread, span = attend_ref(*args, scale=scale)
        tol, tol_lse = attend_bounds(want, spread, span, self.most, D, self.q.dtype)
        err = (got.double() - want).abs()
        assert got is out and bool((err <= tol)[:n].all()), f"out off by up to {float((err / tol)[:n].max()):.3g} of the bound"
        empty = want_lse[:n] == -INF
        assert bool((lse[:n] == -INF)[empty].all()) and bool((got[:n][empty] == 0).all())
        e = (lse[:n].double() - want_lse[:n]).abs()[~empty]
        assert bool((e <= tol_lse[:n][~empty] + 2.0 ** -22 * want_lse[:n][~empty].abs()).all()), f"lse off by {float(e.max()):.3g}"
        assert bool((got[n:] == 7.0).all()), "rows behind the last group were written"
        return got, lse


HEADS = [(8, 2, 64), (8, 2, 128), (4, 4, 64), (16, 1, 128), (6, 3, 128), (12, 1, 64), (24, 1, 64), (40, 2, 128)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads", HEADS)
def test_attention_heads_and_types(dtype, heads):
    Attend(1, dtype, heads, [3, 1, 5], [70, 33, 129], [0, 1, 15, 16, 17, 40, 31, 5, 64], 16, S=140).check()


@pytest.mark.parametrize("heads", [(8, 2, 64), (6, 3, 128)])
@pytest.mark.parametrize("n", [0, 1, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1025])
def test_attention_prefix_lengths(heads, n):
    Attend(n, BF, heads, [2, 3], [n, max(0, n - 1)], [0, 1, 2, 3, 0], 8, S=n + 3).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("n", [0, 1, 15, 16, 33, 127, 129, 500, 1100])
def test_attention_tail_lengths(page, n):
    Attend(n, HF, (8, 2, 64), [4], [5], [n, max(0, n - 1), 1, 0], page).check()


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 64, 65, 100, 257])
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 1, 128)])
def test_attention_group_sizes(rows, heads):
    """Every number of rows that share a prefix, next to a group of one row and an empty one."""
    tails = [b % 5 for b in range(rows + 1)]
    Attend(rows, BF, heads, [rows, 0, 1], [300, 4, 77], tails, 16, pad=3).check()


@pytest.mark.parametrize("sizes", [[300], [0, 300, 0, 7], [150, 90, 60, 1], [0, 0, 3]])
@pytest.mark.parametrize("heads", [(8, 2, 64), (32, 4, 128), (5, 1, 128)])
def test_attention_wide_groups(sizes, heads):
    rs = np.random.RandomState(5)
    Attend(2, HF, heads, sizes, [1700, 130, 0, 257][:len(sizes)], rs.randint(0, 90, sum(sizes)), 32, pad=5).check()


@pytest.mark.parametrize("rows,heads,n", [(2, (8, 8, 64), 70001), (3, (8, 2, 64), 40000), (40, (8, 1, 128), 20011)])
def test_attention_long_prefix(rows, heads, n):
    a = Attend(3, HF, heads, [rows], [n], [9] * rows, 16)
    a.check()


def test_attention_long_tails():
    Attend(4, BF, (8, 2, 64), [2, 1], [3, 0], [9000, 0, 4097], 64).check()


def test_attention_many_rows():
    rs = np.random.RandomState(6)
    sizes = rs.randint(0, 9, 300)
    Attend(5, BF, (8, 2, 64), list(sizes), list(rs.randint(0, 400, 300)), rs.randint(0, 200, sizes.sum()), 64, pad=11).check()


def test_attention_no_tails_and_no_table():
    a = Attend(7, BF, (8, 2, 64), [3, 2], [100, 17], [0] * 5, 16)
    a.table = a.table[:, :0]
    a.check()


def test_attention_every_row_empty():
    got, lse = Attend(8, BF, (8, 2, 64), [2, 2], [0, 0], [0] * 4, 16, S=20).check()
    assert not got.any() and bool((lse == -INF).all())


def test_attention_no_rows():
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(9, BF, (8, 2, 64), [2], [4], [1, 1], 16)
    out, lse = shared_prefix_attention(a.q[:0], a.k, a.v, a.lens, i32([0, 0]), a.kp, a.vp, a.table[:0], a.tails[:0], return_lse=True)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)


@pytest.mark.parametrize("scale", [1.0, 0.02, 1e-6])
def test_attention_scale(scale):
    Attend(10, HF, (8, 2, 64), [3, 9], [90, 300], [4] * 12, 16).check(scale=scale)


@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_attention_peaked_and_flat(size):
    """Scores of up to some thousands, where one position takes all, and next to none, where all count the same."""
    a = Attend(11, BF, (8, 2, 64), [3, 60], [90, 700], [20] * 63, 16)
    a.q *= size
    a.check()


def test_attention_growing_scores():
    """The running maximum rises from tile to tile, and falls again."""
    a = Attend(12, BF, (8, 2, 64), [3, 70], [900, 900], [30] * 73, 16)
    a.k[:, :, :, 0] = torch.linspace(-40, 40, 900, device="cuda").to(BF)[None, :, None]
    a.k[1] = a.k[1].flip(0)
    a.q[:, :, 0] = 8
    a.check()


def test_attention_infinite_values():
    """An infinite V in a used place gives what the formula gives; one behind a length gives nothing (test inputs have
    NaN there already)."""
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(13, BF, (8, 2, 64), [3, 40], [90, 80], [4] * 43, 16)
    a.v[0, 3, 0, 5] = INF
    a.v[1, 79, 1, 6] = -INF
    out = shared_prefix_attention(*a.args())
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[:3, :4, 5] = True
    want[3:, 4:, 6] = True
    assert bool((bad == want).all()) and bool((out[:3, :4, 5] == INF).all()) and bool((out[3:, 4:, 6] == -INF).all())


def test_attention_nan_scores():
    """A NaN key in a used place makes the rows and heads that see it NaN, and no others."""
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(14, BF, (8, 2, 64), [3, 40], [90, 80], [4] * 43, 16)
    a.k[1, 70, 0, 3] = NAN
    out, lse = shared_prefix_attention(*a.args(), return_lse=True)
    want = torch.zeros_like(lse, dtype=torch.bool)
    want[3:, :4] = True
    assert bool((torch.isnan(lse) == want).all()) and bool((torch.isnan(out).all(-1) == want).all())


def test_attention_strided():
    """A layer and a range of rows of larger caches, rows of q inside a wider buffer, columns of a larger table."""
    a = Attend(15, BF, (8, 2, 64), [3, 6], [90, 300], [21] * 9, 16)
    k = torch.full((2, 4, 310, 3, 64), NAN, dtype=BF, device="cuda")
    v = k.clone()
    k[1, 2:, :300, :2], v[1, 2:, :300, :2] = a.k, a.v
    q = torch.full((9, 12, 64), NAN, dtype=BF, device="cuda")
    q[:, 2:10] = a.q
    kp = torch.full((a.kp.shape[0], 2, *a.kp.shape[1:]), NAN, dtype=BF, device="cuda")
    vp = kp.clone()
    kp[:, 1], vp[:, 1] = a.kp, a.vp
    table = torch.full((9, 11), -5, dtype=I32, device="cuda")
    table[:, 4:7] = a.table
    a.check(args=(q[:, 2:10], k[1, 2:, :300, :2], v[1, 2:, :300, :2], a.lens, a.offsets, kp[:, 1], vp[:, 1], table[:, 4:7], a.tails))


def test_attention_past_31_bits():
    """Prefix rows and pages whose offsets pass 2^31 elements."""
    a = Attend(16, BF, (8, 2, 64), [2, 2], [50, 50], [20] * 4, 16)
    S = (1 << 31) // 128 + 1000
    k = torch.empty(2, S, 2, 64, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    k[:, :50], v[:, :50] = a.k, a.v
    n = (1 << 31) // (16 * 128) + 100
    kp = torch.empty(n, 16, 2, 64, dtype=BF, device="cuda")
    vp = torch.empty_like(kp)
    m = a.kp.shape[0]
    kp[-m:], vp[-m:] = a.kp, a.vp
    a.check(args=(a.q, k, v, a.lens, a.offsets, kp, vp, torch.where(a.table < m, a.table + (n - m), a.table), a.tails))


def test_attention_same_bits_again():
    """The order of the sums does not depend on the run."""
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(17, BF, (8, 2, 64), [40, 3, 9], [2000, 300, 77], [150] * 52, 16)
    first = shared_prefix_attention(*a.args())
    for _ in range(5):
        assert torch.equal(first, shared_prefix_attention(*a.args()))


@pytest.mark.parametrize("heads", [(6, 3, 128), (8, 2, 64)])
@pytest.mark.parametrize("each", [19, 70])
def test_attention_same_bits_under_load(heads, each):
    """Many groups with prefixes of many tiles, so that the loads of one tile may come long after those of later ones."""
    from viktor_b200.ops import shared_prefix_attention
    rs = np.random.RandomState(each)
    sizes = rs.randint(0, 2 * each, 86)
    a = Attend(22, HF, heads, list(sizes), list(rs.randint(0, 4500, 86)), rs.randint(0, 17, sizes.sum()), 64, nonsense=False)
    a.check()
    first, lse = shared_prefix_attention(*a.args(), return_lse=True)
    for _ in range(60):
        got = [shared_prefix_attention(*a.args(), return_lse=True) for _ in range(10)]
        assert all(torch.equal(o, first) and torch.equal(l, lse) for o, l in got)


def test_attention_streams_and_graphs():
    """Two calls at once on two streams, and a captured call replayed with other lengths."""
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(18, BF, (8, 2, 64), [30, 3], [1500, 300], [150] * 33, 16, nonsense=False)
    b = Attend(19, BF, (8, 2, 64), [30, 3], [1500, 300], [150] * 33, 16, nonsense=False)
    want = [shared_prefix_attention(*x.args()) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(shared_prefix_attention(*x.args()))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    graphs, outs = [], []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(shared_prefix_attention(*x.args()))
        graphs.append(graph)
    for step in range(3):
        for x in (a, b):
            x.lens.sub_(100 * step)
            x.tails.sub_(step)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, o in zip((a, b), outs):
            assert torch.equal(o, shared_prefix_attention(*x.args()))


def test_attention_own_workspace():
    from viktor_b200._lib import load
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(20, BF, (8, 2, 64), [3, 2], [100, 17], [40] * 5, 16)
    n = load().vk_shared_attention_workspace_bytes(5, 8, 2, 64, 2, 100, a.table.shape[1] * 16)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    want = shared_prefix_attention(*a.args())
    for _ in range(2):
        assert torch.equal(shared_prefix_attention(*a.args(), workspace=ws), want)


@pytest.mark.parametrize("what", ["page", "tail", "prefix", "offset", "negative"])
def test_attention_reports_bad_indices(what):
    """Pages, lengths and offsets out of range are kept out of the reads and reported; the other rows are right."""
    from viktor_b200._lib import check_device_errors
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(21, BF, (8, 2, 64), [2, 2], [100, 17], [40] * 4, 16, nonsense=False)
    want = shared_prefix_attention(*a.args())
    check_device_errors()
    spoilt = {"page": [3], "tail": [3], "prefix": [2, 3], "offset": [2, 3], "negative": [3]}[what]
    if what == "page":
        a.table[3, 1] = a.kp.shape[0]
    elif what == "negative":
        a.table[3, 0] = -1
    elif what == "tail":
        a.tails[3] = a.table.shape[1] * 16 + 1
    elif what == "prefix":
        a.lens[1] = 101
    else:
        a.offsets[2] = 5
    got = shared_prefix_attention(*a.args())
    with pytest.raises(RuntimeError, match="out of range"):
        check_device_errors()
    rest = [b for b in range(4) if b not in spoilt]
    assert torch.equal(got[rest], want[rest])


# ------------------------------------------------------------------------------------------------ pages
def pool(layers=2, n_pages=40, page=8, rows=10, max_pages=6, hk=2, d=64, dtype=BF, seed=0):
    from viktor_b200.ops import KVPages
    p = KVPages.empty(layers, n_pages, page, rows, max_pages, hk, d, dtype)
    g = torch.Generator("cuda").manual_seed(seed)
    for x in (p.k, p.v):
        x.copy_(torch.empty(x.shape, device="cuda").normal_(generator=g).to(dtype))
    return p


def errors():
    from viktor_b200._lib import read_device_errors
    return read_device_errors(clear=True)


@pytest.mark.parametrize("page,dtype,hk,d", [(8, BF, 2, 64), (16, HF, 1, 8), (64, F32, 3, 20), (256, BF, 1, 128)])
def test_pages_random_steps(page, dtype, hk, d):
    """Long random runs of all operations against the whole-number model."""
    from viktor_b200.ops import pages_compact, pages_extend, pages_fork, pages_free
    rng = random.Random(page)
    p = pool(2, 60, page, 12, 7, hk, d, dtype)
    ref = PoolRef(p)
    for step in range(60):
        op = rng.choice(["extend", "extend", "extend", "fork", "fork", "free", "compact"])
        rows = rng.sample(range(12), rng.randint(1, 12))
        if op == "extend":
            count = rng.choice([1, 1, 2, page - 1, page, page + 1, 2 * page + 3])
            rows = None if rng.random() < 0.3 else rows
            page_at, slot = pages_extend(p, count, None if rows is None else i32(rows))
            want = ref.extend(count, rows)
            np.testing.assert_array_equal(page_at.cpu().numpy(), want[0])
            np.testing.assert_array_equal(slot.cpu().numpy(), want[1])
        elif op == "fork":
            src = [rng.randrange(12) for _ in rows]
            pages_fork(p, i32(src), i32(rows))
            ref.fork(src, rows)
        elif op == "free":
            rows = rows[:4] if rng.random() < 0.9 else None
            pages_free(p, None if rows is None else i32(rows))
            ref.free(rows)
        else:
            assert int(pages_compact(p)) == ref.compact()
        ref.check(p)
    errors()  # rows that were full or found no page were reported


@pytest.mark.parametrize("rows,n_pages,max_pages", [(1, 1, 1), (1030, 5000, 3), (2500, 9001, 2), (3, 70001, 5)])
def test_pages_sizes(rows, n_pages, max_pages):
    """More rows and pages than a block has threads, and one of each."""
    from viktor_b200.ops import pages_compact, pages_extend, pages_fork, pages_free
    p = pool(1, n_pages, 8, rows, max_pages, 1, 8)
    ref = PoolRef(p)
    rs = np.random.RandomState(rows)
    for count in (3, 1, 5, 8):
        page, slot = pages_extend(p, count)
        want = ref.extend(count)
        np.testing.assert_array_equal(page.cpu().numpy(), want[0])
        np.testing.assert_array_equal(slot.cpu().numpy(), want[1])
        gone = rs.permutation(rows)[:rows // 2]
        pages_free(p, i32(gone))
        ref.free(gone)
        src, dst = rs.randint(0, rows, rows), rs.permutation(rows)
        pages_fork(p, i32(src), i32(dst))
        ref.fork(src, dst)
        ref.check(p)
    assert int(pages_compact(p)) == ref.compact()
    ref.check(p)
    errors()


def test_pages_fork_swaps_and_chains():
    """Rows that are source and target at once are copied as they were before the call."""
    from viktor_b200.ops import pages_extend, pages_fork
    p = pool()
    ref = PoolRef(p)
    for rows, count in (([0, 1, 2], 13), ([1], 4), ([2], 3)):
        pages_extend(p, count, i32(rows))
        ref.extend(count, rows)
    for src, dst in (([0, 1], [1, 0]), ([0, 1, 2], [1, 2, 3]), ([3, 3, 3], [3, 0, 4]), ([5], [1]), ([2, 2], [5, 6])):
        pages_fork(p, i32(src), i32(dst))
        ref.fork(src, dst)
        ref.check(p)
    assert errors() == 0


def test_pages_same_row_twice():
    """A row that a list names twice is served once and reported; freed twice it is empty."""
    from viktor_b200.ops import pages_extend, pages_fork, pages_free
    p = pool()
    ref = PoolRef(p)
    page, slot = pages_extend(p, 3, i32([4, 4, 1]))
    want = ref.extend(3, [4, 4, 1])
    assert errors() == 8 and page[1].tolist() == [-1] * 3
    np.testing.assert_array_equal(page.cpu().numpy(), want[0])
    pages_fork(p, i32([4, 1]), i32([2, 2]))
    ref.fork([4, 1], [2, 2])
    assert errors() == 8
    ref.check(p)
    pages_free(p, i32([4, 4, 2]))
    ref.free([4, 4, 2])
    assert errors() == 0
    ref.check(p)


def test_pages_out_of_range_and_out_of_pages():
    from viktor_b200.ops import pages_extend, pages_fork, pages_free
    p = pool(n_pages=5, rows=4, max_pages=3)
    ref = PoolRef(p)
    for rows in ([0, 9, -1, 1], [0, 1, 2]):
        page, slot = pages_extend(p, 10, i32(rows))
        want = ref.extend(10, rows)
        np.testing.assert_array_equal(page.cpu().numpy(), want[0])
        assert errors() & 8 if 9 in rows else errors() == 16
        ref.check(p)
    pages_fork(p, i32([0, 1, 7, 0]), i32([2, 3, 1, -3]))
    ref.fork([0, 1, 7, 0], [2, 3, 1, -3])
    assert errors() == 8 | 16
    ref.check(p)
    pages_free(p, i32([1, 4, -1]))
    ref.free([1])
    assert errors() == 8
    ref.check(p)
    page, slot = pages_extend(p, 20, i32([0, 3]))  # row 0 would pass its table
    want = ref.extend(20, [0, 3])
    np.testing.assert_array_equal(page.cpu().numpy(), want[0])
    assert errors() & 8
    ref.check(p)


def test_pages_captured():
    """A captured step replayed goes on from where the pages stand."""
    from viktor_b200.ops import pages_compact, pages_extend, pages_fork, pages_free
    p = pool(rows=6)
    ref = PoolRef(p)
    src, dst = i32([0, 1, 0]), i32([3, 4, 5])

    def step():
        page, slot = pages_extend(p, 3, dst)
        pages_extend(p, 5, src[:2])
        pages_free(p, dst[:1])
        pages_fork(p, src[:2], dst[:2])
        return page, pages_compact(p)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        page, live = step()
    for _ in range(4):
        graph.replay()
        want = ref.extend(3, [3, 4, 5])[0]
        ref.extend(5, [0, 1])
        ref.free([3])
        ref.fork([0, 1], [3, 4])
        n = ref.compact()
        np.testing.assert_array_equal(page.cpu().numpy(), want)
        assert int(live) == n
        ref.check(p)


def test_pages_copies_past_31_bits():
    """Pages whose bytes lie past 2^32 of their layer."""
    from viktor_b200.ops import KVPages, pages_compact, pages_extend, pages_fork
    n = (1 << 32) // (256 * 8 * 128 * 2) + 8
    shape = (1, n, 256, 8, 128)
    k, v = torch.zeros(shape, dtype=BF, device="cuda"), torch.zeros(shape, dtype=BF, device="cuda")
    refs = torch.ones(n, dtype=I32, device="cuda")
    refs[-4:] = 0
    p = KVPages(k, v, torch.full((3, 2), -1, dtype=I32, device="cuda"), i32([0, 0, 0]), refs)
    page, _ = pages_extend(p, 300, i32([0]))
    assert page[0].unique().tolist() == [n - 4, n - 3]
    g = torch.Generator("cuda").manual_seed(1)
    data = torch.empty(2, 2, 256, 8, 128, dtype=BF, device="cuda").normal_(generator=g)
    k[0, n - 4:n - 2], v[0, n - 4:n - 2] = data[0], data[1]
    pages_fork(p, i32([0]), i32([1]))
    assert p.table[1].tolist() == [n - 4, n - 2]
    assert torch.equal(k[0, n - 2, :44], data[0, 1, :44]) and torch.equal(v[0, n - 2, :44], data[1, 1, :44])
    assert not k[0, n - 2, 44:].any()
    refs[:n - 4] = 0
    assert int(pages_compact(p)) == 3 and p.table[:2].tolist() == [[0, 1], [0, 2]]
    assert torch.equal(k[0, :2], data[0]) and torch.equal(v[0, :2], data[1]) and torch.equal(k[0, 2, :44], data[0, 1, :44])


# ------------------------------------------------------------------------------------------------ penalties
def penal_inputs(B, V, T, dtype, seed, masks=5):
    g = torch.Generator().manual_seed(seed)
    lo = -3 if V > 5 else 0
    return dict(logits=(torch.randn(B, V, generator=g) * 4).to(dtype), history=torch.randint(lo, V + 3, (B, T), generator=g),
                history_lens=torch.randint(0, T + 1, (B,), generator=g).int(), repetition=torch.rand(B, generator=g) + 0.5,
                presence=torch.randn(B, generator=g), frequency=torch.randn(B, generator=g) * 0.2, bias=torch.randn(V, generator=g),
                mask=torch.randint(-(1 << 31), 1 << 31, (masks, -(-V // 32)), generator=g).int(),
                mask_index=torch.randint(-1, masks, (B,), generator=g).int())


def check_penal(a, **more):
    from viktor_b200.ops import penalize_logits
    names = dict(history_lens="lens")
    want = penalize_ref(**{names.get(k, k): v for k, v in a.items()})
    x = a["logits"]
    got = penalize_logits(**{k: v if v is None else v.cuda() for k, v in a.items()}, **more).cpu()
    assert got.dtype == x.dtype
    # five operations of half a step of float32 each, on values of at most `size` in between, then one rounding
    T = a["history"].shape[1] if a.get("history") is not None else 0
    size = x.double().abs() * 2.0 + 8.0 + T * 1.0
    size = torch.where(torch.isfinite(size), size, 0.0)
    tol = 5 * 2.0 ** -24 * size + torch.finfo(x.dtype).eps / 2 * want.abs() + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    same = got.double() == want
    both_nan = torch.isnan(got) & torch.isnan(want)
    ok = same | both_nan | ((got.double() - want).abs() <= tol)
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off"
    return got


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("B,V,T", [(1, 1, 1), (3, 7, 20), (5, 343, 1100), (2, 8191, 33), (2, 8193, 300), (3, 32, 5), (2, 33, 4),
                                   (2, 50021, 4097), (1, 131072, 513), (9, 16384, 70)])
def test_penalties_sizes(dtype, B, V, T):
    check_penal(penal_inputs(B, V, T, dtype, V + T))


@pytest.mark.parametrize("drop", [("repetition",), ("presence",), ("frequency",), ("bias",), ("mask", "mask_index"),
                                  ("repetition", "presence", "frequency", "history", "history_lens"),
                                  ("repetition", "presence", "frequency"), ("presence", "bias", "mask", "mask_index")])
def test_penalties_parts(drop):
    a = penal_inputs(4, 1000, 50, F32, 3)
    check_penal({k: v for k, v in a.items() if k not in drop})


def test_penalties_masks_and_rows():
    """One mask for all, one for each row, a bias for each row, no tokens at all."""
    a = penal_inputs(4, 1000, 50, F32, 4, masks=4)
    a["bias"] = torch.randn(4, 1000)
    del a["mask_index"]
    check_penal(a)
    check_penal({**a, "mask": a["mask"][:1]})
    check_penal({**a, "history": a["history"][:, :0], "history_lens": torch.zeros(4, dtype=I32)})
    check_penal({**a, "history_lens": torch.zeros(4, dtype=I32)})


def test_penalties_nothing_allowed_and_infinities():
    """A mask without a bit gives a row of -inf whatever the logits hold; elsewhere infinities and NaN go by the formula."""
    a = penal_inputs(3, 100, 20, F32, 5)
    a["logits"][:, 7], a["logits"][:, 8], a["logits"][:, 9] = INF, -INF, NAN
    a["history"][:, :3] = torch.tensor([7, 8, 9])
    a["history_lens"][:] = 3
    a["mask"][0], a["mask"][1] = 0, -1
    a["mask_index"] = torch.tensor([0, 1, -1], dtype=I32)
    got = check_penal(a)
    assert bool((got[0] == -INF).all()) and got[1, 7] == INF and got[1, 8] == -INF and bool(torch.isnan(got[1:, 9]).all())


def test_penalties_one_token_many_times():
    a = penal_inputs(2, 70000, 70000, F32, 6)
    a["history"][0], a["history"][1, ::2] = 69999, 3
    a["history_lens"][:] = 70000
    check_penal(a)


def test_penalties_in_place_and_strided():
    """In place, with rows inside wider buffers: what lies between the rows stays."""
    from viktor_b200.ops import penalize_logits
    a = penal_inputs(3, 343, 40, F32, 7)
    want = check_penal(a).cuda()
    wide = torch.full((3, 352), 9.0, device="cuda")
    wide[:, 1:344] = a["logits"]
    hist = torch.full((3, 50), 5, dtype=torch.int64, device="cuda")
    hist[:, 7:47] = a["history"]
    rest = {k: v.cuda() for k, v in a.items() if k not in ("logits", "history")}
    view = wide[:, 1:344]
    assert penalize_logits(view, hist[:, 7:47], out=view, **rest) is view
    assert torch.equal(view, want) and bool((wide[:, 0] == 9).all()) and bool((wide[:, 344:] == 9).all())


def test_penalties_past_31_bits():
    from viktor_b200.ops import penalize_logits
    V, B = 131072, 16500
    x = torch.zeros(B, V, dtype=BF, device="cuda")
    hist = torch.zeros(B, 1, dtype=torch.int64, device="cuda")
    hist[-1] = V - 1
    pres = torch.zeros(B, device="cuda")
    pres[-1] = 2.0
    out = penalize_logits(x, hist, torch.ones(B, dtype=I32, device="cuda"), presence=pres, out=x)
    assert out[-1, -1] == -2.0 and not out[:-1].any() and not out[-1, :-1].any()


def test_penalties_report_bad_indices():
    from viktor_b200._lib import check_device_errors
    a = penal_inputs(3, 343, 40, F32, 8)
    for name, bad in (("mask_index", 5), ("mask_index", -2), ("history_lens", 41), ("history_lens", -1)):
        b = {k: v.clone() for k, v in a.items()}
        b[name][1] = bad
        from viktor_b200.ops import penalize_logits
        penalize_logits(**{k: v.cuda() for k, v in b.items()})
        with pytest.raises(RuntimeError, match="out of range"):
            check_device_errors()


# ------------------------------------------------------------------------------------------------ together
class Candidates:
    """Decodes N candidates of each chunk that an engine has prefilled: the chunk's row of the engine's cache is the shared
    prefix, every candidate's own tokens live in pages."""

    def __init__(self, eng, n, page, n_pages):
        from viktor_b200.ops import KVPages
        self.eng, self.w, self.n = eng, eng.w, n
        B, cfg = eng.B * n, eng.cfg
        self.B = B
        self.pages = KVPages.empty(cfg.n_layers, n_pages, page, B, -(-eng.max_new // page))
        self.offsets = i32(range(0, B + 1, n))
        self.plens = (eng.plen + 1).int()
        self.base = self.plens.repeat_interleave(n)
        self.x, self.ssq = eng._xcat.repeat_interleave(n, 0), eng._scat.repeat_interleave(n, 0)
        self.q = torch.empty(B, 8, 64, dtype=BF, device="cuda")
        self.g = torch.empty(B, cfg.ffn_dim, dtype=BF, device="cuda")
        self.history = torch.zeros(B, eng.max_new, dtype=torch.int64, device="cuda")

    def logits(self):
        from viktor_b200 import ops
        return ops.linear_rmsnorm(self.x, self.ssq, self.w.eps, self.w.lm_head, out_dtype=F32)[:, :self.w.vocab]

    def step(self, tok):
        from viktor_b200 import ops
        p, w = self.pages, self.w
        pos = self.base + p.lens
        page, slot = ops.pages_extend(p)
        page, slot = page.flatten(), slot.flatten()
        self.x = w.embed[tok]
        self.ssq = ops.row_ssq(self.x)
        for i, L in enumerate(w.layers):
            ops.linear_qkv_rope_cache(self.x, L["qkv"], L["q_norm"], L["k_norm"], w.cos, w.sin, slot, page, p.k[i], p.v[i], w.eps,
                                      rope_pos=pos, q_out=self.q, ssq=self.ssq, norm_eps=w.eps)
            o = ops.shared_prefix_attention(self.q, self.eng.cache.k[i], self.eng.cache.v[i], self.plens, self.offsets, p.k[i],
                                            p.v[i], p.table, p.lens)
            ops.linear_residual(o.view(self.B, 512), L["o"], self.x, ssq_out=self.ssq)
            g = ops.linear_rmsnorm(self.x, self.ssq, w.eps, L["gate_up"], swiglu=True)
            ops.linear_residual(g, L["down"], self.x, ssq_out=self.ssq)

    def select(self, logits, t, noise, temperature=0.8, **penalties):
        from viktor_b200 import ops
        lens = torch.full((self.B,), t, dtype=I32, device="cuda")
        z = ops.penalize_logits(logits, self.history, lens, bias=self.eng.bias, **penalties)
        tok = (z / temperature - (-(noise.clamp(min=1e-20).log())).log()).argmax(-1)
        self.history[:, t] = tok
        return tok


def test_candidates_of_chunks_decode_together():
    """Prefill two chunks with the engine, sample three candidates of each from pages with penalties and a grammar mask, let
    the best take the place of others on the way (fork), compact, and go on.  At every step the logits equal those of the
    engine's teacher forcing over each candidate's own tokens, within the noise of two bf16 paths (the bound of
    tests/test_gpu_engine.py)."""
    from golden_io import load
    from test_gpu_engine import build
    from viktor_b200 import ops
    gold = load("base_theta1e6")
    lens, steps, n = gold["meta"]["lens"][:2], 21, 3
    frames = torch.from_numpy(gold["frames"][:sum(lens)])
    eng = build(gold, B=len(lens), max_new=steps, graph=False, max_frames=max(lens))
    eng.prefill(frames, lens)
    c = Candidates(eng, n, page=8, n_pages=40)
    g = torch.Generator("cuda").manual_seed(3)
    mask = torch.full((2, 1), 0b1111000, dtype=I32, device="cuda")  # bases only
    mask[1] = 0b0101000
    pen = dict(repetition=torch.full((c.B,), 1.1, device="cuda"), frequency=torch.full((c.B,), 0.05, device="cuda"))
    seen, order = [], torch.arange(c.B, device="cuda")
    logits = c.logits()
    for t in range(steps):
        seen = [s[order] for s in seen] + [logits]
        order = torch.arange(c.B, device="cuda")
        state = i32([(t + b) % 3 - 1 for b in range(c.B)])
        tok = c.select(logits, t, torch.rand(c.B, eng.w.vocab, device="cuda", generator=g), mask=mask, mask_index=state, **pen)
        assert bool(((tok >= 3) | (state < 0)).all()) and bool(((tok == 3) | (tok == 5) | (state != 1)).all())
        if t == steps - 1:
            break
        c.step(tok)
        logits = c.logits()
        if t in (4, 9, 12):  # the second candidate of each chunk takes the place of its neighbours
            src, dst = i32([1, 1, 4, 4]), i32([0, 2, 3, 5])
            ops.pages_fork(c.pages, src, dst)
            order[dst.long()] = src.long()
            c.history, c.x, logits = c.history[order], c.x[order], logits[order]
            c.ssq = c.ssq[order]
        if t in (6, 13):
            assert int(ops.pages_compact(c.pages)) == int((c.pages.refs > 0).sum())
    got = torch.stack(seen, 1)
    tokens = torch.cat([torch.ones(c.B, 1, dtype=torch.int64, device="cuda"), c.history[:, :steps - 1]], 1)
    big = build(gold, B=c.B, max_new=steps, graph=False, max_frames=max(lens))
    per = [frames[sum(lens[:i]):sum(lens[:i + 1])] for i in range(len(lens)) for _ in range(n)]
    want = big.teacher_forced_logits(torch.cat(per), [lens[i] for i in range(len(lens)) for _ in range(n)], tokens)
    assert (c.history[0] != c.history[1]).any()
    assert float((got - want).abs().max()) < 2.5e-2
