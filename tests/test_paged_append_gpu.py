"""New tokens entering a paged cache on the GPU against 64 bits: norm, rotation, the store into pages."""

import pytest
import torch

import serving_util as su
from dlmrt_b200.ops.paged_kv import PagedKV, rotary_table

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def tokens(n, hq, hk, d, dtype, seed, device="cuda"):
    """q, k, v as slices of one projection's output."""
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(n, (hq + 2 * hk) * d, generator=g) * 2).to(dtype).to(device)
    return [t.view(n, -1, d) for t in qkv.split((hq * d, hk * d, hk * d), 1)]


def norm(d, dtype, seed):
    return (torch.randn(d, generator=torch.Generator().manual_seed(seed)) * 0.2 + 1).to(dtype).cuda()


def untouched(pool, slots, page):
    """Mask [pages, page] of the places that no token was stored in."""
    mask = torch.ones(pool.shape[0], page, dtype=torch.bool)
    s = slots.cpu()
    s = s[s >= 0]
    mask[s // page, s % page] = False
    return mask


CASES = [
    # n, hq, hk, d, page, pages, dtype, cache, rotated, interleaved, norms, layout
    (1, 4, 1, 64, 16, 3, BF16, BF16, 64, False, True, "hnd"),
    (7, 8, 2, 128, 16, 4, BF16, BF16, 128, False, True, "nhd"),
    (33, 3, 3, 256, 8, 9, F16, F16, 128, True, False, "hnd"),
    (130, 6, 2, 128, 8, 18, BF16, E4M3, 64, False, True, "hnd"),
    (65, 2, 1, 64, 64, 4, F16, E4M3, 48, True, True, "nhd"),
    (40, 5, 5, 256, 32, 4, BF16, E4M3, 256, False, False, "hnd"),
    (9, 4, 2, 128, 16, 2, F16, F16, 0, False, True, "hnd"),
    (300, 32, 8, 128, 64, 6, BF16, BF16, 128, True, True, "hnd"),
]


@pytest.mark.parametrize("n, hq, hk, d, page, pages, dtype, cache, rotated, interleaved, norms, layout", CASES)
def test_append_matches_64_bits(n, hq, hk, d, page, pages, dtype, cache, rotated, interleaved, norms, layout):
    keys, values, ks, vs = su.pool(pages, hk, page, d, cache, 1, layout, "cuda")
    before = keys.clone(), values.clone()
    kv = PagedKV(keys, values, ks, vs)
    q, k, v = tokens(n, hq, hk, d, dtype, 2)
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(pages * page, generator=g)[:n].cuda()
    if n > 8:
        slots[[2, n - 1]] = torch.tensor([-1, -7], device="cuda")
    positions = torch.randint(0, 5000, (n,), generator=g).int().cuda()
    positions[0] = 4999
    table = rotary_table(rotated, 5000, 1e6, "cuda") if rotated else None
    wq, wk = (norm(d, dtype, 4), norm(d, dtype, 5)) if norms else (None, None)
    out = kv.append(k, v, positions, slots, table, q=q, q_norm=wq, k_norm=wk, eps=1e-5, interleaved=interleaved)
    kv.check()
    want, bound = su.turned(q, wq, table, positions, 1e-5, interleaved)
    su.assert_within(out, *su.stored(want, bound, dtype), "queries")
    stored = slots.cpu() >= 0
    at = slots.cpu()[stored]
    for pool, was, x, w, t, scale, what in ((keys, before[0], k, wk, table, ks, "keys"), (values, before[1], v, None, None, vs, "values")):
        want, bound = su.stored(*su.turned(x, w, t, positions, 1e-5, interleaved), cache, scale)
        got = pool.cpu().double()[at // page, :, at % page]
        su.assert_within(got, want[stored], bound[stored], what)
        rest = untouched(pool, slots, page)
        same = pool.cpu().view(torch.uint8).transpose(1, 2)[rest], was.cpu().view(torch.uint8).transpose(1, 2)[rest]
        assert torch.equal(*same), f"{what}: places that no token has were written"


def test_values_are_copied_bit_for_bit_and_specials_survive():
    keys, values, *_ = su.pool(2, 2, 16, 64, BF16, 1, device="cuda")
    kv = PagedKV(keys, values)
    _, k, v = tokens(4, 1, 2, 64, BF16, 2)
    k, v = k.contiguous(), v.contiguous()
    v[1, 0, 3], v[2, 1, 5], k[3, 0, 0] = float("inf"), float("nan"), float("-inf")
    kv.append(k, v, None, torch.arange(4, device="cuda"))
    assert torch.equal(values[0, :, :4].transpose(0, 1).view(torch.int16), v.view(torch.int16))
    assert torch.equal(keys[0, :, :4].transpose(0, 1).view(torch.int16), k.view(torch.int16))


def test_fp8_saturates_and_keeps_nan():
    keys, values, ks, vs = su.pool(1, 1, 16, 64, E4M3, 1, device="cuda")
    kv = PagedKV(keys, values, ks, vs)
    k = torch.zeros(1, 1, 64, device="cuda", dtype=BF16)
    k[0, 0, :4] = torch.tensor([1e5, -1e5, float("inf"), float("nan")])
    kv.append(k, k, None, torch.zeros(1, device="cuda", dtype=torch.int64))
    got = keys[0, 0, 0, :4].float().cpu()
    assert got[:3].tolist() == [448.0, -448.0, 448.0] and got[3].isnan()


def test_queries_in_place_and_without_queries():
    keys, values, *_ = su.pool(2, 2, 16, 128, BF16, 1, device="cuda")
    q, k, v = tokens(5, 4, 2, 128, BF16, 2)
    table, positions = rotary_table(128, 64, device="cuda"), torch.arange(5, device="cuda").int()
    slots = torch.arange(5, device="cuda")
    kv = PagedKV(keys, values)
    want = kv.append(k, v, positions, slots, table, q=q)
    first = keys.clone()
    assert kv.append(k, v, positions, slots, table) is None
    assert torch.equal(keys, first)
    assert kv.append(k, v, positions, slots, table, q=q, q_out=q) is q
    assert torch.equal(q, want)


def test_indices_outside_their_tables_touch_nothing_and_are_reported():
    keys, values, *_ = su.pool(2, 1, 16, 64, BF16, 1, device="cuda")
    kv = PagedKV(keys, values)
    q, k, v = tokens(3, 1, 1, 64, BF16, 2)
    table = rotary_table(64, 10, device="cuda")
    for slots, positions, row, what in (([0, 32, 1], [0, 1, 2], 1, "slot 2"), ([0, 1, 2], [0, 1, 10], 2, "position 10"),
                                        ([0, 1, 2], [-1, 1, 3], 0, "position -1"), ([0, 1 << 50, 2], [0, 1, 2], 1, "slot")):
        before = keys.clone()
        out = torch.full_like(q, 7.0)
        kv.append(k, v, torch.tensor(positions).int().cuda(), torch.tensor(slots).cuda(), table, q=q, q_out=out)
        assert bool((out[row] == 7).all()) and not bool((out == 7).all())
        good = [i for i in range(3) if i != row]
        assert not torch.equal(keys[0, 0, [slots[i] for i in good]], before[0, 0, [slots[i] for i in good]]) or what != "slot 2"
        with pytest.raises(IndexError, match=f"row {row}: {what}"):
            kv.check()
        kv.check()  # read and cleared


def test_no_tokens_is_no_launch():
    keys, values, *_ = su.pool(1, 1, 16, 64, BF16, 1, device="cuda")
    kv = PagedKV(keys, values)
    q, k, v = (t[:0] for t in tokens(1, 2, 1, 64, BF16, 2))
    none = torch.empty(0, device="cuda", dtype=torch.int64)
    assert kv.append(k, v, none.int(), none, rotary_table(64, 4, device="cuda"), q=q).shape == (0, 2, 64)


def test_captured_and_replayed():
    keys, values, *_ = su.pool(4, 2, 16, 128, BF16, 1, device="cuda")
    q, k, v = tokens(6, 4, 2, 128, BF16, 2)
    table, positions, slots = rotary_table(128, 64, device="cuda"), torch.arange(6, device="cuda").int(), torch.arange(6, device="cuda")
    kv = PagedKV(keys, values)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv.append(k, v, positions, slots, table, q=q)
    slots += 20
    positions += 3
    graph.replay()
    other = PagedKV(keys.clone(), values.clone())
    want = other.append(k, v, positions, slots, table, q=q)
    assert torch.equal(out, want) and torch.equal(other.keys, keys) and torch.equal(other.values, values)
