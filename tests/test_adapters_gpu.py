"""Low-rank adapters beside a projection on the GPU against 64 bits."""

import pytest
import torch

import serving_util as su
from dlmrt_b200.layers.adapters import Adapters

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def setup(m, count, rank, k, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = (torch.randn(count, rank, k, generator=g) * k ** -0.5).to(BF16).cuda()
    b = (torch.randn(count, n, rank, generator=g) * rank ** -0.5).to(BF16).cuda()
    scales = (torch.rand(count, generator=g) + 0.5).cuda()
    x, base = torch.randn(m, k, generator=g).to(BF16).cuda(), torch.randn(m, n, generator=g).to(BF16).cuda()
    return Adapters(a, b, scales), x, base, g


def check(layer, x, ids, base):
    out = layer(x, ids, base)
    su.assert_within(out, *su.adapters(x, ids, base, layer.a, layer.b, layer.scales))
    layer.check()
    return out


@pytest.mark.parametrize("m", [1, 2, 16, 17, 61, 255, 256])
@pytest.mark.parametrize("count", [1, 3, 40])
def test_rows_and_adapters(m, count):
    layer, x, base, g = setup(m, count, 16, 320, 200)
    ids = torch.randint(-1, count, (m,), generator=g).int().cuda()
    check(layer, x, ids, base)


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128])
def test_ranks(rank):
    layer, x, base, g = setup(20, 3, rank, 264, 136)
    check(layer, x, torch.randint(0, 3, (20,), generator=g).int().cuda(), base)


@pytest.mark.parametrize("k, n", [(8, 8), (16, 40), (4096, 32), (40, 2568), (2560, 2560)])
def test_sizes(k, n):
    layer, x, base, g = setup(5, 2, 16, k, n)
    check(layer, x, torch.tensor([1, 0, -1, 1, 1]).int().cuda(), base)


def test_every_row_of_one_adapter_and_rows_of_none():
    layer, x, base, _ = setup(100, 4, 16, 128, 128)
    check(layer, x, torch.full((100,), 3).int().cuda(), base)
    out = check(layer, x, torch.full((100,), -1).int().cuda(), base)
    assert torch.equal(out, base)


def test_in_place_and_strided():
    layer, x, base, g = setup(33, 4, 32, 256, 264)
    ids = torch.randint(-1, 4, (33,), generator=g).int().cuda()
    want = layer(x, ids, base)
    wide_x, wide = torch.zeros(33, 300 - 4, device="cuda", dtype=BF16), torch.full((33, 400), 5.0, device="cuda", dtype=BF16)
    wide_x[:, 8:264] = x
    wide[:, 16:280] = base
    view = wide[:, 16:280]
    assert layer(wide_x[:, 8:264], ids, view, out=view) is view
    assert torch.equal(view, want) and bool((wide[:, :16] == 5).all()) and bool((wide[:, 280:] == 5).all())
    one = base[:1].expand(33, -1)
    assert torch.equal(layer(x, ids, one)[ids.cpu().lt(0).cuda()], one[ids.cpu().lt(0).cuda()])


def test_an_id_past_the_last_adapter_counts_as_none_and_is_reported():
    layer, x, base, _ = setup(4, 2, 16, 64, 64)
    ids = torch.tensor([0, 2, 1, -5]).int().cuda()
    out = layer(x, ids, base)
    su.assert_within(out, *su.adapters(x, ids, base, layer.a, layer.b, layer.scales))
    assert torch.equal(out[1], base[1])
    with pytest.raises(IndexError, match="row 1: adapter 2"):
        layer.check()
    layer.check()


def test_one_rows_nan_stays_in_its_row():
    layer, x, base, _ = setup(12, 2, 16, 64, 64)
    ids = torch.tensor([0, 1] * 6).int().cuda()
    want = layer(x, ids, base)
    x[4, 3] = float("nan")
    base[7, 2] = float("inf")
    got = layer(x, ids, base)
    rows = [i for i in range(12) if i not in (4, 7)]
    assert torch.equal(got[rows], want[rows]) and bool(got[4].isnan().all()) and got[7, 2].isinf()


def test_captured_replayed_and_the_same_bits():
    layer, x, base, g = setup(50, 5, 16, 512, 512)
    ids = torch.randint(-1, 5, (50,), generator=g).int().cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, ids, base)
    ids.copy_(ids.flip(0))
    graph.replay()
    want = layer(x, ids, base)
    assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [layer(x, ids, base) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)
