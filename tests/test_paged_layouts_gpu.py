"""Layouts of queries, keys and values that callers have besides slices of one projection side by side."""

import pytest
import torch

import serving_util as su
from dlmrt_b200.ops.paged_kv import PagedKV, rotary_table
from test_paged_append_gpu import tokens

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("n", [1, 21])
@pytest.mark.parametrize("group", [1, 3])
def test_queries_rotated_in_place_between_keys_and_values(n, group):
    """[n, key heads, (queries of a group, key, value), head dim]: one key head's share of a projection after the other."""
    hk, d = 2, 64
    q, k, v = (t.contiguous() for t in tokens(n, hk * group, hk, d, BF16, 2))
    wide = torch.cat((q.view(n, hk, group, d), k.unsqueeze(2), v.unsqueeze(2)), 2).contiguous()
    if group > 1:  # queries have one stride only where a key head has one: the first of each group
        q = q.view(n, hk, group, d)[:, :, 0].contiguous()
    table, positions = rotary_table(d, 64, device="cuda"), torch.arange(n, device="cuda").int()
    slots = torch.arange(n, device="cuda")
    kv, other = (PagedKV(*su.pool(2, hk, 16, d, BF16, 1, device="cuda")) for _ in range(2))
    want = kv.append(k, v, positions, slots, table, q=q)
    view = wide[:, :, 0]
    before = wide.clone()
    assert other.append(wide[:, :, -2], wide[:, :, -1], positions, slots, table, q=view, q_out=view) is view
    assert torch.equal(view, want) and torch.equal(other.keys, kv.keys) and torch.equal(other.values, kv.values)
    assert torch.equal(wide[:, :, 1:], before[:, :, 1:])
    other.check()
    # results beside the queries of the same rows: every second head
    heads = torch.zeros(n, hk, 2, d, device="cuda", dtype=BF16)
    heads[:, :, 0] = want
    pages, lengths = torch.zeros(n, 1, device="cuda", dtype=torch.int32), torch.full((n,), 5, device="cuda", dtype=torch.int32)
    expected = kv.attend(want, pages, lengths)
    out = heads[:, :, 1]
    assert kv.attend(heads[:, :, 0], pages, lengths, out=out) is out
    assert torch.equal(out, expected) and torch.equal(heads[:, :, 0], want)
