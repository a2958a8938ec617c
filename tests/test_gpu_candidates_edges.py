"""The operators that decode several candidates of a chunk at the ends of what their entry points accept."""

import pytest
import torch

from test_gpu_candidates import BF, I32, Attend, errors, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _errors_clear():
    from viktor_b200._lib import check_device_errors
    yield
    torch.cuda.synchronize()
    check_device_errors()


# ------------------------------------------------------------------------------------------------ attention
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
