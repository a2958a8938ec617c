"""The operators that decode several candidates of a chunk at the ends of what their entry points accept."""

import math

import pytest
import torch

from candidates_ref import attend_bounds, attend_ref
from test_gpu_candidates import BF, F32, HF, I32, INF, NAN, Attend, check_penal, errors, i32, penal_inputs, pool

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _errors_clear():
    from viktor_b200._lib import check_device_errors
    yield
    torch.cuda.synchronize()
    check_device_errors()


# ------------------------------------------------------------------------------------------------ attention
def check_attend(a):
    """As Attend.check, with the bound on the rounding of fp16 probabilities completed: one that is below 2^-14 next to its
    reference is not off by u relative but by up to 2^-25, half the step of the smallest fp16 values.  The reference of a chunk is at
    least 11 (base 2) below its largest score, so the sum of all probabilities is at least 2^11 there, and every position adds at
    most 2^-36 |v_j|."""
    from viktor_b200.ops import shared_prefix_attention
    out = torch.full(a.q.shape, 7.0, dtype=a.q.dtype, device="cuda")
    got, lse = shared_prefix_attention(*a.args(), out=out, return_lse=True)
    n, D, dtype = a.q.shape[0] - a.pad, a.q.shape[2], a.q.dtype
    want, want_lse, spread, span = attend_ref(*a.args())
    tol, tol_lse = attend_bounds(want, spread, span, a.most, D, dtype)
    if dtype is HF:
        largest = max(float(torch.nan_to_num(x.float(), nan=0.0).abs().max()) for x in (a.v, a.vp))
        tol = tol + 2.0 ** -36 * a.most * largest
    err = (got.double() - want).abs()
    assert bool((err <= tol)[:n].all()), f"out off by up to {float((err / tol)[:n].max()):.3g} of the bound"
    empty = want_lse[:n] == -INF
    assert bool((lse[:n] == -INF)[empty].all()) and bool((got[:n][empty] == 0).all())
    e = (lse[:n].double() - want_lse[:n]).abs()[~empty]
    assert bool((e <= tol_lse[:n][~empty] + 2.0 ** -22 * want_lse[:n][~empty].abs()).all()), f"lse off by {float(e.max()):.3g}"
    assert bool((got[n:] == 7.0).all()), "rows behind the last group were written"


# few rows of each group; more than 32 of a KV head; more than 128
FORMS = [((2, 1, 64), [1] * 300), ((2, 1, 128), [1] * 300), ((40, 1, 64), [1] * 148), ((40, 1, 128), [1] * 148), ((40, 1, 64), [4] * 148),
         ((40, 1, 128), [4] * 148)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,sizes", FORMS)
@pytest.mark.parametrize("gap", [13.0, 20.6, 25.05, 27.5])
def test_attention_dominant_positions_of_small_value(dtype, heads, sizes, gap):
    """A few positions whose scores are 2^gap above all others, with values of 0: what the others add up to is not lost.  They
    stand where every warp and stream that goes through a prefix meets one first."""
    D = heads[2]
    a = Attend(31, dtype, heads, sizes, [700 - g % 7 for g in range(len(sizes))], [5] * sum(sizes), 16)
    a.q *= 0.05
    a.k[..., 0] = a.kp[..., 0] = 0.0
    a.q[..., 0] = 4.0
    for x in (a.v, a.vp):
        x.mul_(0.1).add_(1.0).mul_(64.0)
    for at in (0, 16, 32, 48, 64, 96):
        a.k[:, at, :, 0] = gap * math.log(2.0) * math.sqrt(D) / 4.0
        a.v[:, at] = 0.0
    check_attend(a)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("heads,rows", [((8, 2, 64), 7), ((2, 1, 128), 2500)])
def test_attention_dominant_positions_in_tails(dtype, page, heads, rows):
    """The same in the tails, for few and for many rows."""
    D = heads[2]
    a = Attend(32, dtype, heads, [rows], [3], [200 - b % 9 for b in range(rows)], page)
    a.q *= 0.05
    a.k[..., 0] = a.kp[..., 0] = 0.0
    a.q[..., 0] = 4.0
    for x in (a.v, a.vp):
        x.mul_(0.1).add_(1.0).mul_(64.0)
    for at in (0, 16, 32, 48, 64, 96):
        pages = a.table[:, at // page].long()
        a.kp[pages, at % page, :, 0] = 21.0 * math.log(2.0) * math.sqrt(D) / 4.0
        a.vp[pages, at % page] = 0.0
    check_attend(a)


@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_attention_peaked_and_flat_in_fp16(size):
    a = Attend(33, HF, (8, 2, 64), [3, 60], [90, 700], [20] * 63, 16)
    a.q *= size
    check_attend(a)


def test_attention_growing_scores_in_fp16():
    """The running maximum rises from tile to tile, by more and by less than the reference may lag behind, and falls again."""
    for top in (3.0, 12.0, 40.0):
        a = Attend(34, HF, (8, 2, 64), [3, 70], [900, 900], [30] * 73, 16)
        a.k[:, :, :, 0] = torch.linspace(-top, top, 900, device="cuda").to(HF)[None, :, None]
        a.k[1] = a.k[1].flip(0)
        a.q[:, :, 0] = 8
        check_attend(a)


@pytest.mark.parametrize("heads,B,P,lo", [((1, 1, 64), 180, 6, 60), ((1, 1, 64), 1000, 3, 100), ((2, 1, 128), 40, 6, 8),
                                          ((2, 1, 128), 500, 3, 50)])
def test_attention_offsets_that_descend(heads, B, P, lo):
    """Offsets 0, B, lo, B, ...: the second group is refused, the first and the third have rows and tiles in common.  That is
    reported, rows below lo are right, and nothing is written behind the workspace."""
    from viktor_b200._lib import load
    from viktor_b200.ops import shared_prefix_attention
    a = Attend(30, BF, heads, [B] + [0] * (P - 1), [300, 70, 150, 4, 5, 6][:P], [b % 4 for b in range(B)], 16)
    n = load().vk_shared_attention_workspace_bytes(B, *heads, P, 300, a.table.shape[1] * 16)
    ws = torch.full((n + (1 << 20),), 255, dtype=torch.uint8, device="cuda")
    want = shared_prefix_attention(*a.args(), workspace=ws)
    assert errors() == 0 and bool((ws[n:] == 255).all())
    a.offsets[2] = lo
    for _ in range(20):
        got = shared_prefix_attention(*a.args(), workspace=ws)
        assert errors() == 8 and torch.equal(got[:lo], want[:lo]) and bool((ws[n:] == 255).all())


# groups whose rows of a KV head are more than 32 (two streams take turns), and more than 128 (two streams of rows)
WIDE = [((40, 1, 64), 1), ((40, 1, 128), 1), ((40, 1, 64), 4), ((20, 1, 128), 9), ((80, 2, 64), 3), ((40, 2, 128), 5)]


@pytest.mark.parametrize("heads,each", WIDE)
@pytest.mark.parametrize("more", [0, 3])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 192, 193, 255, 256, 257, 511, 513])
def test_attention_wide_prefix_lengths(heads, each, n, more):
    """Prefixes that end before, at and behind the ends of tiles, with a cache that ends there too or has NaN behind."""
    check_attend(Attend(n, HF if n % 2 else BF, heads, [each, each + 1], [n, n - 1], [b % 4 for b in range(2 * each + 1)], 8, S=n + more))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,each", WIDE)
def test_attention_wide_chunks_of_many_tiles(heads, each, dtype):
    """As many groups as there are SMs, so that a chunk is a whole prefix: every number of tiles up to 12, and odd ends."""
    lens = [0, 1, 63, 64, 65, 705] + [5 * g % 769 for g in range(146)]
    check_attend(Attend(40, dtype, heads, [each] * len(lens), lens, [3] * (each * len(lens)), 8))


@pytest.mark.parametrize("heads,sizes", [((8, 2, 64), [20, 0, 11]), ((8, 2, 64), [70, 0, 40]), ((6, 3, 128), [30, 0, 40]), ((8, 1, 128), [33, 0, 40])])
def test_attention_wide_workspace_of_any_contents(heads, sizes):
    """What the workspace holds does not matter: prefixes, tails and rows without tokens write no values."""
    from viktor_b200._lib import load
    from viktor_b200.ops import shared_prefix_attention
    B = sum(sizes)
    a = Attend(41, BF, heads, sizes, [900, 70, 0], [b % 3 * 20 for b in range(B)], 16, pad=2)
    n = load().vk_shared_attention_workspace_bytes(B + 2, *heads, 3, 900, a.table.shape[1] * 16)
    want, want_lse = shared_prefix_attention(*a.args(), return_lse=True)
    for fill in (255, 0, 127):
        ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        for _ in range(2):
            got, lse = shared_prefix_attention(*a.args(), workspace=ws, return_lse=True)
            assert torch.equal(got[:B], want[:B]) and torch.equal(lse[:B], want_lse[:B])
    check_attend(a)


@pytest.mark.parametrize("sizes", [[20, 25], [40, 50]])
def test_attention_wide_past_31_bits(sizes):
    """Prefix rows and pages whose offsets pass 2^31 elements."""
    a = Attend(42, BF, (8, 2, 64), sizes, [150, 150], [20] * sum(sizes), 16)
    S = (1 << 31) // 128 + 1000
    k = torch.full((2, S, 2, 64), NAN, dtype=BF, device="cuda")
    v = torch.full((2, S, 2, 64), NAN, dtype=BF, device="cuda")
    k[:, :150], v[:, :150] = a.k, a.v
    n = (1 << 31) // (16 * 128) + 100
    kp = torch.full((n, 16, 2, 64), NAN, dtype=BF, device="cuda")
    vp = torch.full((n, 16, 2, 64), NAN, dtype=BF, device="cuda")
    m = a.kp.shape[0]
    kp[-m:], vp[-m:] = a.kp, a.vp
    a.table = torch.where(a.table < m, a.table + (n - m), a.table)
    a.k, a.v, a.kp, a.vp = k, v, kp, vp
    check_attend(a)


@pytest.mark.parametrize("heads", [(8, 2, 64), (6, 3, 128)])
def test_attention_one_large_group_among_many(heads):
    """The mean of the rows of a group chooses the kernel: here the large group goes through the one for few rows."""
    check_attend(Attend(43, BF, heads, [1] * 40 + [300] + [1] * 160, [70 + g for g in range(201)], [b % 5 for b in range(500)], 16))


# ------------------------------------------------------------------------------------------------ pages
def test_extend_rows_near_31_bits():
    """A row of almost 2^31 tokens: `count` more than it has room for are refused, as many as it has room for are placed."""
    from viktor_b200.ops import KVPages, pages_extend
    page, max_pages = 256, (1 << 23) - 1
    most = page * max_pages
    k = torch.zeros(1, 6, page, 1, 8, dtype=BF, device="cuda")
    table = torch.full((1, max_pages), -1, dtype=I32, device="cuda")
    table[0, -2], table[0, -1] = 4, 2
    p = KVPages(k, k.clone(), table, i32([most - 100]), i32([0, 0, 1, 0, 1, 0]))
    for count in (101, 512, 1 << 20):  # the last two pass 2^31 with the length
        before = [t.clone() for t in (p.table, p.lens, p.refs)]
        places, slots = pages_extend(p, count)
        assert errors() == 8 and bool((places == -1).all()) and bool((slots == -1).all())
        assert all(torch.equal(a, b) for a, b in zip(before, (p.table, p.lens, p.refs)))
    places, slots = pages_extend(p, 100)
    assert places.unique().tolist() == [2] and slots[0].tolist() == list(range(156, 256)) and p.lens.tolist() == [most]
    table[0, -1] = -1
    p.lens.fill_(most - 300)
    p.refs.copy_(i32([1, 0, 0, 0, 1, 0]))
    places, slots = pages_extend(p, 300)
    assert places[0].tolist() == [4] * 44 + [1] * 256 and p.table[0, -2:].tolist() == [4, 1] and p.refs.tolist() == [1, 1, 0, 0, 1, 0]
    assert slots[0].tolist() == list(range(212, 256)) + list(range(256)) and errors() == 0


@pytest.mark.parametrize("rows", [4, 1000])
def test_extend_with_too_few_pages(rows):
    """The first row that needs more pages than are left stops every later one of the call that needs a page; rows that need
    none are served, and what is left is there for the next call."""
    from viktor_b200.ops import pages_extend
    p = pool(n_pages=rows + 1, rows=rows, max_pages=4, layers=1, hk=1)
    pages_extend(p, 3, i32(range(2, rows)))  # one page each
    p.refs[rows - 2:] = 1
    p.refs[rows] = 0  # one free page
    p.lens[1], p.table[1, 0] = 7, rows - 1
    table, lens, refs = p.table.clone(), p.lens.clone(), p.refs.clone()
    # 9 tokens: row 0 needs two pages, the others one each
    places, slots = pages_extend(p, 9)
    assert errors() == 16 and bool((places == -1).all()) and bool((slots == -1).all())
    assert torch.equal(p.table, table) and torch.equal(p.lens, lens) and torch.equal(p.refs, refs)
    # 5 tokens: rows 0 and 1 need one page each, and row 0 gets it; the others have room
    places, slots = pages_extend(p, 5)
    assert errors() == 16 and places[0].tolist() == [rows] * 5 and places[1].tolist() == [-1] * 5
    assert torch.equal(places[2:], table[2:, :1].expand(-1, 5)) and slots[2:].unique().tolist() == [3, 4, 5, 6, 7]
    table[0, 0], refs[rows] = rows, 1
    lens += 5
    lens[1] = 7
    assert torch.equal(p.table, table) and torch.equal(p.lens, lens) and torch.equal(p.refs, refs)
    # a free page again: without the row that needs two, row 1 gets it
    p.refs[rows], p.table[0, 0], p.lens[0] = 0, -1, 0
    places, slots = pages_extend(p, 9, i32([1, 0]))
    assert errors() == 16 and places.tolist() == [[rows - 1] + [rows] * 8, [-1] * 9] and slots[0].tolist() == [7, 0, 1, 2, 3, 4, 5, 6, 7]


@pytest.mark.parametrize("bad", [-1, -7, 40, 2 ** 31 - 1])
@pytest.mark.parametrize("max_pages", [6, 3000])
def test_fork_of_a_row_whose_last_page_is_out_of_range(bad, max_pages):
    """Nothing can be copied, so the row stays as it was, and no page is spent on it; other rows are served."""
    from viktor_b200.ops import pages_extend, pages_fork
    p = pool(max_pages=max_pages)
    pages_extend(p, 13, i32([0, 1, 2]))
    p.table[0, 1] = bad
    p.refs[1] = 0
    before = p.table.clone(), p.lens.clone(), p.refs.clone(), p.k.clone(), p.v.clone()
    pages_fork(p, i32([0, 2, 0]), i32([1, 3, 4]))
    assert errors() == 8
    table, lens, refs, k, v = before
    table[3, :2] = i32([4, 1])  # the lowest free page is 1
    lens[3], refs[4], refs[1] = 13, 2, 1
    k[:, 1, :5], v[:, 1, :5] = k[:, 5, :5], v[:, 5, :5]
    assert torch.equal(p.table, table) and torch.equal(p.lens, lens) and torch.equal(p.refs, refs)
    assert torch.equal(p.k, k) and torch.equal(p.v, v)
    p.table[0, 1] = 7  # repaired: served
    p.refs[7] = 1
    pages_fork(p, i32([0]), i32([4]))
    assert errors() == 0 and p.table[4, :2].tolist() == [0, 6] and p.lens[4] == 13
    assert torch.equal(p.k[:, 6, :5], p.k[:, 7, :5])


@pytest.mark.parametrize("lens,last", [(-1, 1), (-(2 ** 31), 1), (6 * 8 + 1, 1), (2 ** 31 - 1, 1), (13, -1), (13, 40)])
def test_extend_and_fork_of_a_row_out_of_range(lens, last):
    """A row whose length or partly filled last page is out of range is left as it is and reported; the others are served."""
    from viktor_b200.ops import pages_extend, pages_fork
    p = pool()
    pages_extend(p, 13, i32([0, 1, 2]))
    p.lens[0], p.table[0, 1] = lens, last
    table, lengths, refs = p.table.clone(), p.lens.clone(), p.refs.clone()
    places, slots = pages_extend(p, 4, i32([0, 1]))
    assert errors() == 8 and places.tolist() == [[-1] * 4, [3, 3, 3, 6]] and slots.tolist() == [[-1] * 4, [5, 6, 7, 0]]
    table[1, 2], lengths[1], refs[6] = 6, 17, 1
    assert torch.equal(p.table, table) and torch.equal(p.lens, lengths) and torch.equal(p.refs, refs)
    pages_fork(p, i32([0, 2]), i32([3, 4]))
    assert errors() == 8
    table[4, :2], lengths[4], refs[4], refs[7] = i32([4, 7]), 13, 2, 1
    assert torch.equal(p.table, table) and torch.equal(p.lens, lengths) and torch.equal(p.refs, refs)
    pages_fork(p, i32([2]), i32([0]))  # over the damaged row: well again
    assert errors() == 0 and p.lens[0] == 13


def test_compact_with_a_table_that_names_a_free_page():
    """Such an entry is left as it is and reported, whatever the workspace held; the others follow their pages."""
    from viktor_b200.ops import pages_compact, pages_extend, pages_free
    p = pool(n_pages=400)
    pages_extend(p, 13, i32([0, 1, 2]))
    pages_free(p, i32([0]))
    p.table[5, :3] = i32([399, 7, 401])
    for _ in range(3):
        filled = [torch.full((1 << k,), 5, dtype=I32, device="cuda") for k in (9, 10, 11, 12)]
        del filled
        p.table[2, :2], p.refs[:6] = i32([4, 5]), i32([0, 0, 1, 1, 1, 1])
        assert int(pages_compact(p)) == 4 and errors() == 8
        assert p.table[1, :2].tolist() == [2, 3] and p.table[2, :2].tolist() == [0, 1] and p.table[5, :3].tolist() == [399, 7, 401]
        assert p.refs.nonzero().flatten().tolist() == [0, 1, 2, 3]


# ------------------------------------------------------------------------------------------------ penalties
@pytest.mark.parametrize("V", [7, 1000])
def test_penalties_of_any_size(V):
    """Repetition penalties whose inverse is no normal number: a logit over 1e-40 is not infinite as long as the quotient is a
    number.  The inverse, the product and the result are off by half a step each, results below the normal numbers by half of
    their step."""
    from viktor_b200.ops import penalize_logits
    g = torch.Generator().manual_seed(V)
    reps = torch.tensor([2.0 ** -149, 1e-40, 1.1e-38, 2.0 ** -126, 1e-37, 0.5, 1.3, 8e37, 2.0 ** 126, 1.8e38, 3.4e38, INF, 0.0])
    B = len(reps)
    x = torch.randn(B, V, generator=g) * torch.randint(-140, 127, (B, V), generator=g).double().exp2()
    x = x.float()
    history = torch.randint(0, V, (B, 2 * V), generator=g)
    lens = torch.full((B,), 2 * V, dtype=I32)
    got = penalize_logits(x.cuda(), history.cuda(), lens.cuda(), repetition=reps.cuda()).cpu()
    seen = torch.zeros(B, V, dtype=torch.bool).scatter_(1, history, True)
    d, r = x.double(), reps.double()[:, None]
    want = torch.where(seen, torch.where(d > 0, d / r, d * r), d)
    most = float(torch.finfo(torch.float32).max)
    beyond = want.abs() > most * (1 + 2.0 ** -22)
    assert torch.equal(got[beyond], torch.where(want > 0, INF, -INF)[beyond].float())
    inside = want.abs() < most * (1 - 2.0 ** -22)
    assert bool((torch.isnan(got) == torch.isnan(want)).all())
    off = (got.double() - want).abs() <= 3 * 2.0 ** -24 * want.abs() + 2.0 ** -149
    assert bool(off[inside].all()), f"{int((~off[inside]).sum())} of {int(inside.sum())} off"


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("B,V,T,wide", [(3, 7, 20, 16), (5, 343, 1100, 352), (33, 343, 40, 352), (2, 50021, 4097, 50048), (1, 131071, 513, 131080),
                                        (9, 16385, 70, 16400), (2, 33000, 70000, 33024)])
def test_penalties_on_logits_of_a_wider_head(dtype, B, V, T, wide):
    """The first V columns of rows that are padded: rows of logits and of out lie differently relative to 16 bytes, in several
    slices and steps.  The arithmetic is the same, so the bits are those of contiguous logits; what lies between rows stays."""
    from viktor_b200.ops import penalize_logits
    a = penal_inputs(B, V, T, dtype, V + B)
    want = check_penal(a).cuda()
    rest = {k: v.cuda() for k, v in a.items() if k != "logits"}
    rows = torch.full((B, wide), NAN, dtype=dtype, device="cuda")
    rows[:, :V] = a["logits"].cuda()
    got = penalize_logits(rows[:, :V], **rest)
    assert got.is_contiguous() and torch.equal(got, want)
    out = torch.full((B, wide + 1), 9.0, dtype=dtype, device="cuda")
    penalize_logits(a["logits"].cuda(), out=out[:, 1:V + 1], **rest)
    assert torch.equal(out[:, 1:V + 1], want) and bool((out[:, 0] == 9).all()) and bool((out[:, V + 1:] == 9).all())
    penalize_logits(rows[:, :V], out=rows[:, :V], **rest)
    assert torch.equal(rows[:, :V], want) and bool(torch.isnan(rows[:, V:]).all())
