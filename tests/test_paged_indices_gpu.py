"""What new tokens with an index outside its table leave behind, and how they are reported."""

import pytest
import torch

import serving_util as su
from dlmrt_b200.ops.paged_kv import PagedKV, rotary_table
from test_paged_append_gpu import tokens, untouched

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
PAGE, PAGES, ROWS = 16, 3, 10


@pytest.mark.parametrize("slot, text", [(48, "slot 3 * 16 + 0"), (61, "slot 3 * 16 + 13"), ((1 << 40) + 5, "slot at least 2147483647 * 16 + 5"),
                                        ((1 << 35) - 1, "slot at least 2147483647 * 16 + 15"), ((1 << 35) - 17, "slot 2147483646 * 16 + 15"),
                                        ((1 << 63) - 1, "slot at least 2147483647 * 16 + 15")])
def test_a_slot_is_named_by_its_page_and_place(slot, text):
    kv = PagedKV(*su.pool(PAGES, 1, PAGE, 64, BF16, 1, device="cuda"))
    _, k, v = tokens(3, 1, 1, 64, BF16, 2)
    before = kv.keys.clone(), kv.values.clone()
    kv.append(k, v, None, torch.tensor([-1, slot, -1], device="cuda"))
    with pytest.raises(IndexError) as raised:
        kv.check()
    assert f"row 1: {text} lies outside" in str(raised.value)
    assert torch.equal(before[0], kv.keys) and torch.equal(before[1], kv.values)
    kv.check()
