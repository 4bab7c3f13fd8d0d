"""Infinities and NaN in the values of long sequences: in steps of keys that only some rows of a tile see, when earlier steps have
results already, which the same step rescales. Rows that do not see them keep their bits."""

import math

import pytest
import torch

import serving_util as su
from dlmrt_b200.ops.paged_kv import PagedKV
from test_paged_attend_gpu import setup

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
N, PAGE, STEP = 330, 16, 64


def growing(batch, t, hq, hk, d, dtype, cache):
    """Sequences of N keys whose scores grow by 7.5 from a step of 64 keys to the next (more than 2^15 in two of them)."""
    kv, q, table, lengths = setup([N] * batch, t, hq, hk, d, PAGE, dtype, cache)
    q /= 4
    q[..., 0] = 10 * d ** 0.5
    rise = 0.75 * (torch.arange(-(-N // PAGE) * PAGE, device="cuda") // STEP).view(-1, 1, PAGE).float()
    if cache == E4M3:
        rise = rise / kv.k_scale.view(1, -1, 1)
    for row in table[:, :-(-N // PAGE)]:
        kv.keys[row.long(), :, :, 0] = rise.expand(-1, hk, -1).to(cache)
    return kv, q, table, lengths


def put(kv, table, key, element, special):
    """Sets an element of the values of a key of every sequence."""
    values = kv.values.view(torch.uint8) if kv.dtype == E4M3 else kv.values
    values[table[:, key // PAGE].long(), :, key % PAGE, element] = 0x7F if kv.dtype == E4M3 else special


@pytest.mark.parametrize("cache, special", [(BF16, math.inf), (BF16, math.nan), (F16, -math.inf), (F16, math.nan), (E4M3, math.nan)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t, hq, hk, batch", [(100, 1, 1, 2), (100, 1, 4, 40), (8, 2, 1, 2), (4, 8, 4, 40)])
def test_specials_behind_steps_that_count(t, hq, hk, batch, d, cache, special):
    """100 rows (tiles of 128: the first visible key of tokens 230 and on) and 16 rows; whole, and 40 sequences in a wider table
    over runs of about a dozen steps that begin and end anywhere."""
    kv, q, table, lengths = growing(batch, t, hq * hk if batch == 40 and t == 100 else hq, hk, d, F16 if cache == F16 else BF16, cache)
    if batch == 40:
        table = torch.cat((table, table.new_full((batch, 64 - table.shape[1]), -1)), 1)
    call = lambda **kw: kv.attend(q, table, lengths, causal=True, **kw)
    first = N - t
    clean = call()
    rows = [0, t // 2, t - 1]
    for i in rows:
        see = lengths[:2] - (t - 1 - i)
        want, bound, _ = su.attend(q[:2, i:i + 1], kv.keys, kv.values, kv.k_scale, kv.v_scale, table[:2], see.tolist(), d ** -0.5)
        su.assert_within(clean[:2, i:i + 1], want, bound)
    # behind the end: in the last step's last page
    for key in range(N, -(-N // PAGE) * PAGE):
        put(kv, table, key, slice(None), special)
    assert torch.equal(call(), clean)
    # in two steps of the same item that some rows see: tokens from those keys on
    places = [(first + t // 5, 5), (N - 1 - t // 20, 37)]
    for key, element in places:
        put(kv, table, key, element, special)
    got = call()
    for key, element in places:
        assert bool((~got[:, key - first:, :, element].isfinite()).all())
        got[:, key - first:, :, element] = clean[:, key - first:, :, element]
    assert torch.equal(got, clean)
    # with a window that leaves the first of them behind
    window = call(window=places[1][0] - places[0][0])
    assert bool(window[:, places[1][0] - first:, :, places[0][1]].isfinite().all())
    kv.check()


@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("t, hq", [(1, 8), (40, 2)])
@pytest.mark.parametrize("sign", [1, -1])
def test_a_visible_infinity_stays_one(sign, t, hq, cache):
    """In a step that all rows see in full an infinite value is part of the products: of its weight's high part, which may be a
    whole weight, and of its low part."""
    kv, q, table, lengths = setup([256, 200], t, hq, 1, 64, PAGE, cache, cache)
    kv.keys.zero_()  # all weights are the same power of two
    kv.values[table[0, 3], :, 5, 11] = sign * math.inf
    kv.values[table[1, 0], :, 0, 2] = sign * math.inf
    got = kv.attend(q, table, lengths)
    assert bool((got[0, ..., 11] == sign * math.inf).all()) and bool((got[1, ..., 2] == sign * math.inf).all())
    got[0, ..., 11] = got[1, ..., 2] = 0
    assert bool(got.isfinite().all())
    q = q / 8  # all kinds of weights
    kv.keys.normal_(generator=torch.Generator("cuda").manual_seed(4))
    got = kv.attend(q, table, lengths)
    assert bool((got[0, ..., 11] == sign * math.inf).all()) and bool((got[1, ..., 2] == sign * math.inf).all())
