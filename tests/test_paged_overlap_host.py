"""Which results may lie beside their inputs, on the host: the entry points refuse exactly those that share elements, as far as the
tensors step alike. Nothing here needs a GPU; where there is one, calls that would not be refused are left out."""

import random

import pytest
import torch

from dlmrt_b200 import _lib
from test_paged_kv_host import adapters, append, attend, pages

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused would run on addresses that are not")
BASE = 1 << 20


def elements(at, extents, strides, inner):
    """The 2-byte elements that a tensor takes."""
    starts = [at // 2]
    for extent, stride in zip(extents, strides):
        starts = [s + i * stride for s in starts for i in range(extent)]
    return {s + i for s in starts for i in range(inner)}


def refused(code):
    return code == _lib.ERR_OVERLAP


def test_a_projection_with_its_heads_in_turn_takes_rotated_queries_in_place():
    """[n, heads, (q, k, v), head dim] and [n, groups, (queries, key, value), head dim]: nothing is shared."""
    d = 64
    for n in (1, 3):
        call = append(n=n, q=BASE, q_out=BASE, q_heads=2, k=BASE + d * 2, v=BASE + 4 * d)
        for strides in (call.q_strides, call.out_strides, call.k_strides, call.v_strides):
            strides[:] = 6 * d, 3 * d
        assert not refused(_lib.lib().dlm_paged_append(call, None))
        call.k = BASE + 3 * d * 2  # the second head of q
        assert refused(_lib.lib().dlm_paged_append(call, None))


def test_rows_side_by_side_may_space_their_heads_otherwise():
    """Halves of the same longer rows: 4 heads of queries 64 apart, results 128 apart behind them; and keys 72 apart in front."""
    d, row = 64, 4 * 64 + 4 * 128 + 2 * 72
    call = append(n=3, q=BASE, q_out=BASE + 2 * 4 * d, q_heads=4, k=BASE + 2 * (4 * 64 + 4 * 128), v=BASE + (1 << 18), q_strides=(row, 64),
                  out_strides=(row, 128), k_strides=(row, 72))
    assert not refused(_lib.lib().dlm_paged_append(call, None))
    call.q_out = BASE + 2 * 4 * d - 16
    assert refused(_lib.lib().dlm_paged_append(call, None))
    two = attend(cache=pages(heads=4), q=BASE, out=BASE + 2 * 4 * d, q_heads=4, batch=3, q_strides=(row, row, 64), out_strides=(row, row, 128))
    assert not refused(_lib.lib().dlm_paged_attend(two, None))


@pytest.mark.parametrize("seed", range(10))
def test_append_refuses_what_shares_elements(seed):
    rng = random.Random(seed)
    for turn in range(30):
        n, hq, hk, d = rng.randint(1, 5), rng.randint(1, 5), rng.randint(1, 4), 64
        step = (rng.choice([64, 128, 192, 72, 320]), rng.choice([64, 128, 192, 256, 512, 72]))
        q, k, out = (BASE + 16 * rng.randint(-80, 80) for _ in range(3))
        v = BASE + (1 << 18)
        code = _lib.lib().dlm_paged_append(append(cache=pages(heads=hk), n=n, q=q, q_out=out, q_heads=hq, k=k, v=v, q_strides=step,
                                                  out_strides=step, k_strides=step, v_strides=(hk * 64, 64)), None)
        mine = elements(out, (n, hq), step, d)
        shares = mine & elements(k, (n, hk), step, d) or (q != out and mine & elements(q, (n, hq), step, d))
        assert refused(code) == bool(shares)


@pytest.mark.parametrize("seed", range(10))
def test_attend_refuses_what_shares_elements(seed):
    rng = random.Random(seed)
    for turn in range(30):
        b, t, hk, group, d = rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 3), rng.randint(1, 2), 64
        steps = [rng.choice([64, 128, 192, 256, 576, 1024, 2048, 72]) for _ in range(3)]
        other = list(steps)
        if turn % 3 == 0:
            other[rng.randrange(3)] += 64
        q, out = (BASE + 16 * rng.randint(-150, 150) for _ in range(2))
        extents = (b, t, hk * group)
        code = _lib.lib().dlm_paged_attend(attend(cache=pages(heads=hk), q=q, out=out, q_heads=hk * group, batch=b, tokens=t, q_strides=steps,
                                                  out_strides=other), None)
        alike = all(e == 1 or x == y for e, x, y in zip(extents, steps, other))
        shares = bool(elements(q, extents, steps, d) & elements(out, extents, other, d)) and not (q == out and alike)
        assert refused(code) == shares if alike else refused(code) or not shares


@pytest.mark.parametrize("seed", range(10))
def test_adapters_refuse_what_shares_elements(seed):
    rng = random.Random(seed)
    for turn in range(30):
        m, n, k, ld = rng.randint(1, 6), 8 * rng.randint(1, 12), 8 * rng.randint(1, 12), 8 * rng.randint(12, 40)
        x, out = (BASE + 16 * rng.randint(-60, 60) for _ in range(2))
        base = rng.choice([out, BASE + (1 << 18)])
        code = _lib.lib().dlm_adapters_bf16(adapters(x=x, base=base, out=out, m=m, n=n, k=k, ldx=ld, ldb=ld, ldo=ld), None)
        assert refused(code) == bool(elements(x, (m,), (ld,), k) & elements(out, (m,), (ld,), n))


def test_a_great_many_rows_are_looked_at_quickly():
    """2^16 tokens of 2^9 heads in turn, in three batches."""
    d = 64
    steps = ((1 << 16) * (1 << 9) * 2 * d, (1 << 9) * 2 * d, 2 * d)
    call = attend(cache=pages(heads=512), q=BASE, out=BASE + 2 * d, q_heads=512, batch=3, tokens=1 << 16, q_strides=steps, out_strides=steps)
    assert not refused(_lib.lib().dlm_paged_attend(call, None))
    call.out = BASE + 2 * d - 16
    assert refused(_lib.lib().dlm_paged_attend(call, None))
