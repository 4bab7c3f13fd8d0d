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


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("bad, what", [({3: (PAGE * PAGES, None)}, "row 3: slot 3"), ({0: (1 << 40, None)}, "row 0: slot"),
                                       ({9: (None, ROWS)}, "row 9: position 10"), ({4: (None, -1)}, "row 4: position -1"),
                                       ({2: (-1, ROWS)}, "row 2: position 10"), ({5: (99999, 1 << 30)}, "row 5: slot"),
                                       ({1: (None, -(1 << 31)), 6: (PAGE * PAGES + 1, None), 8: (-1, None)}, "row [16]: ")])
def test_rows_with_a_bad_index_leave_everything_as_it_was(bad, what, cache):
    """Their own slot (where that is good), every other place of the pool, and their rotated queries; the other rows are
    stored and rotated as without them."""
    keys, values, ks, vs = su.pool(PAGES, 2, PAGE, 64, cache, 1, device="cuda")
    kv, other = PagedKV(keys, values, ks, vs), PagedKV(keys.clone(), values.clone(), ks, vs)
    was = keys.clone(), values.clone()
    q, k, v = tokens(ROWS, 3, 2, 64, BF16, 2)
    table = rotary_table(64, ROWS, device="cuda")
    slots = torch.randperm(PAGE * PAGES, generator=torch.Generator().manual_seed(3))[:ROWS]
    positions = torch.arange(ROWS).flip(0).int()
    for row, (slot, position) in bad.items():
        slots[row] = slots[row] if slot is None else slot
        positions[row] = positions[row] if position is None else position
    left_out = [r for r, (slot, position) in bad.items() if not (slot == -1 and position is None)]
    good = [r for r in range(ROWS) if r not in left_out]
    out = torch.full_like(q, 7.0)
    kv.append(k, v, positions.cuda(), slots.cuda(), table, q=q, q_out=out)
    with pytest.raises(IndexError, match=what):
        kv.check()
    kv.check()  # read and cleared
    assert bool((out[left_out] == 7).all())
    want = other.append(k[good], v[good], positions[good].cuda(), slots[good].cuda(), table, q=q[good])
    other.check()
    assert torch.equal(out[good], want)
    rest = untouched(keys, slots[good], PAGE)
    for pool, expected, before in zip((keys, values), (other.keys, other.values), was):
        pool, expected, before = (t.cpu().view(torch.uint8).transpose(1, 2) for t in (pool, expected, before))
        assert torch.equal(pool, expected)
        assert torch.equal(pool[rest], before[rest]) and not torch.equal(pool[~rest], before[~rest])
