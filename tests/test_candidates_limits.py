"""The largest sizes that the operators for several candidates of a chunk accept, checked without a GPU."""

import pytest
import torch

from viktor_b200 import _lib, ops

MOST = 2 ** 31 - 2 ** 16  # positions of a prefix and a tail together


def _attend(S, max_pages, page):
    """Tensors without storage: nothing is read before a refusal."""
    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")

    ints = dict(dtype=torch.int32)
    return dict(q=empty(1, 1, 64), k_prefix=empty(1, S, 1, 64), v_prefix=empty(1, S, 1, 64), prefix_lens=empty(1, **ints),
                group_offsets=empty(2, **ints), k_pages=empty(1, page, 1, 64), v_pages=empty(1, page, 1, 64),
                page_table=empty(1, max_pages, **ints), tail_lens=empty(1, **ints))


@pytest.mark.parametrize("S,max_pages,page", [(1, (MOST >> 3), 8), (8, (MOST >> 3), 8), (7, 2 ** 28 - 1, 8), (1, 2 ** 23 - 1, 256),
                                              (MOST, 1, 8), (2 ** 31 - 1, 0, 8), (5, 2 ** 24, 128), (5, 2 ** 31, 256)])
def test_shared_prefix_attention_refuses_more_positions(S, max_pages, page):
    """Past this the end of the last chunk, and the places that are looked at behind it, would pass 2^31."""
    with pytest.raises(ValueError, match="max_pages"):
        ops.shared_prefix_attention(**_attend(S, max_pages, page))


def test_entry_point_refuses_more_positions():
    lib = _lib.load()
    for S, max_pages, page in ((1, MOST >> 3, 8), (7, 2 ** 28 - 1, 8), (1, 2 ** 23 - 1, 256), (MOST + 1, 0, 8), (2 ** 31 - 1, 0, 8)):
        assert lib.vk_shared_attention_workspace_bytes(1, 1, 1, 64, 1, S, max_pages * page) == 0
        assert lib.vk_shared_attention(16, 64, 0, 16, 16, 16, 16, 1, S, 64 * S, 64, 16, 16, 1, page, 64 * page, 16, max_pages, max_pages,
                                       16, 1 << 20, None, 1, 1, 1, 64, 0.125, 16, 2 ** 62, None) == _lib.VK_ERR_ARG
    assert lib.vk_shared_attention_workspace_bytes(1, 1, 1, 64, 1, 8, MOST - 8) > 0
