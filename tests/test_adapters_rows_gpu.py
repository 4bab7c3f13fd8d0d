"""Adapters of a single row, as decoding has it, out of buffers of any width."""

import pytest
import torch

import serving_util as su
from test_adapters_gpu import setup

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("ids", [1, -1])
def test_a_row_of_odd_buffers(ids):
    layer, x, base, _ = setup(1, 2, 16, 64, 72)
    ids = torch.tensor([ids]).int().cuda()
    want = layer(x, ids, base)
    su.assert_within(want, *su.adapters(x, ids, base, layer.a, layer.b, layer.scales))
    wide = [torch.full((1, 64 + 72 + 5), 3.0, device="cuda", dtype=BF16) for _ in range(2)]
    wide[0][:, :64], wide[0][:, 64:136] = x, base
    view = wide[1][:, 8:80]
    assert layer(wide[0][:, :64], ids, wide[0][:, 64:136], out=view) is view
    assert torch.equal(view, want) and bool((wide[1][:, :8] == 3).all()) and bool((wide[1][:, 80:] == 3).all())
    assert torch.equal(layer(x.t().contiguous().t(), ids, base.t().contiguous().t()), want)  # rows 1 apart
