"""Low-rank values of adapters at the end of the range: infinite ones, and finite ones that BF16 would round to infinity."""

import math

import pytest
import torch

import serving_util as su
from dlmrt_b200.layers.adapters import Adapters
from test_adapters_gpu import setup

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("rank", [8, 16, 24, 64, 128])
def test_infinite_rows_are_infinite_where_the_definition_says_so(rank):
    layer, x, base, g = setup(20, 2, rank, 64, 72)
    layer.a[:, :, 3] = layer.a[:, :, 3].abs() + 0.1
    layer.b[:, :40] = layer.b[:, :40].abs() + 0.1  # columns whose sum has one sign; the others are inf - inf
    layer.b[:, 60:] = -layer.b[:, 60:].abs() - 0.1
    ids = (torch.arange(20) % 3 - 1).int().cuda()
    clean = layer(x, ids, base)
    x[4, 3], x[8, 3], x[9, 3] = math.inf, -math.inf, math.inf  # adapters 0 and 1, and a row without one
    got = layer(x, ids, base)
    assert bool((got[4, :40] == math.inf).all()) and bool((got[4, 60:] == -math.inf).all())
    assert bool((got[8, :40] == -math.inf).all()) and bool((got[8, 60:] == math.inf).all())
    for row in (4, 8):
        low = layer.a[ids[row]].double() @ x[row].double()
        want = base[row].double() + layer.scales[ids[row]].double() * (layer.b[ids[row]].double() @ low)
        assert torch.equal(got[row].double().isnan(), want.isnan()) and torch.equal(got[row].isinf(), want.isinf())
    rest = [i for i in range(20) if i not in (4, 8)]
    assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("sign", [1, -1])
def test_values_past_the_largest_bf16_stay_finite(sign):
    """x A^T = 255.75 * 2^120: between the largest BF16 (255 * 2^120) and the largest FP32."""
    a = torch.zeros(1, 8, 16, dtype=BF16)
    a[0, 1, 0] = a[0, 1, 1] = sign
    b = torch.zeros(1, 24, 8, dtype=BF16)
    b[0, :, 1] = 2.0 ** -120
    x = torch.zeros(2, 16, dtype=BF16)
    x[0, 0], x[0, 1], x[1, 0] = 255 * 2.0 ** 120, 0.75 * 2.0 ** 120, 1
    layer = Adapters(a.cuda(), b.cuda(), torch.ones(1).cuda())
    base = torch.full((2, 24), -sign * 255.0, dtype=BF16).cuda()
    got = layer(x.cuda(), torch.zeros(2, dtype=torch.int32).cuda(), base)
    su.assert_within(got, *su.adapters(x, torch.zeros(2, dtype=torch.int32), base, a, b, layer.scales))
    assert bool((got[0] == sign * 0.75).all())
