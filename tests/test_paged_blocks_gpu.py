"""Attention of blocks of tokens over a paged cache: enough rows for the 128-row tiles of tensor memory. Against 64 bits."""

import math

import pytest
import torch

import serving_util as su
from test_paged_attend_gpu import check, setup

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t, hq, hk", [(17, 1, 1), (33, 1, 1), (32, 8, 2), (43, 3, 1)])
def test_one_tile_of_rows(t, hq, hk, d, dtype):
    """Rows just above 16 and 32, exactly 128, and one row more; lengths around the step of 64 keys, whole and split."""
    check(*setup([t, 64, 65, 128, 300], t, hq, hk, d, 16, dtype, dtype))
    check(*setup([0, t, 640, 1029], t, hq, hk, d, 32, dtype, dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t, hq, hk", [(32, 1, 1), (33, 1, 1), (32, 8, 2), (43, 3, 1)])
def test_one_tile_of_rows_over_codes(t, hq, hk, d, dtype):
    check(*setup([t, 64, 65, 128, 300], t, hq, hk, d, 16, dtype, E4M3))
    check(*setup([0, t, 640, 1029], t, hq, hk, d, 32, dtype, E4M3))


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [0, 40, 600])
def test_several_tiles_of_rows(d, causal, window, cache):
    check(*setup([200, 150, 700, 256], 150, 4, 2, d, 64, BF16, cache), causal=causal, window=window)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages_of_codes(page, layout, d):
    check(*setup([70, 257], 40, 2, 1, d, page, BF16, E4M3, layout=layout))


def test_queries_beyond_halves_over_codes():
    """BF16 queries whose products with codes are taken in halves: rows of 1e5, of 1e-7, and one of zeros."""
    kv, q, table, lengths = setup([300, 130], 40, 2, 1, 128, 16, BF16, E4M3)
    q[:, 3] *= 1e5
    q[:, 5] *= 1e-7
    q[:, 7] = 0
    for scale in (1e-6, 0.05):
        check(kv, q[:, 4:], table, lengths, scale=scale)
    check(kv, q, table, lengths, scale=1e-7)


def test_codes_that_are_not_numbers():
    """NaN codes behind the end, in front of the window and in later tokens' places stay out; a visible one reaches its rows."""
    kv, q, table, lengths = setup([100, 53], 40, 2, 1, 64, 16, BF16, E4M3)
    clean = kv.attend(q, table, lengths, causal=True, window=30)
    used = torch.zeros(kv.keys.shape[0], 16, dtype=torch.bool)
    for i, n in enumerate(lengths.tolist()):
        for j in range(max(0, n - 40 - 30 + 1), n):
            used[table[i, j // 16], j % 16] = True
    for t in (kv.keys, kv.values):
        t.view(torch.uint8).transpose(1, 2)[~used.cuda()] = 0x7F
    assert torch.equal(kv.attend(q, table, lengths, causal=True, window=30), clean)
    at = 100 - 40 + 35
    kv.values.view(torch.uint8)[table[0, at // 16], :, at % 16, 5] = 0xFF
    got = kv.attend(q, table, lengths, causal=True, window=30)
    assert bool(got[0, 35:, :, 5].isnan().all())
    got[0, 35:, :, 5] = clean[0, 35:, :, 5]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages(page, layout):
    check(*setup([70, 257], 40, 2, 1, 128, page, BF16, BF16, layout=layout))


def test_tokens_in_front_of_the_first_key():
    got = check(*setup([0, 10, 41], 40, 2, 1, 64, 16, BF16, BF16), causal=True)
    assert not got[0].any() and not got[1, :30].any() and bool(got[1, 30:].any())
    check(*setup([0, 10, 41], 40, 2, 1, 64, 16, BF16, BF16), causal=True, window=5)


@pytest.mark.parametrize("special", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_what_the_mask_hides(special, dtype):
    """As for single tokens: what lies behind the end, in front of the window or in later tokens' places stays out; in keys that
    a row does see it reaches that row."""
    kv, q, table, lengths = setup([100, 53], 40, 2, 1, 64, 16, dtype, dtype)
    clean = kv.attend(q, table, lengths, causal=True, window=30)
    used = torch.zeros(kv.keys.shape[0], 16, dtype=torch.bool)
    for i, n in enumerate(lengths.tolist()):
        for j in range(max(0, n - 40 - 30 + 1), n):
            used[table[i, j // 16], j % 16] = True
    for t in (kv.keys, kv.values):
        t.transpose(1, 2)[~used.cuda()] = special
    assert torch.equal(kv.attend(q, table, lengths, causal=True, window=30), clean)
    # the key of token 35 of sequence 0: rows 0..34 do not see it, later ones do
    at = 100 - 40 + 35
    kv.values[table[0, at // 16], :, at % 16, 5] = special
    kv.keys[table[0, at // 16], :, at % 16] = 0
    got = kv.attend(q, table, lengths, causal=True, window=30)
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :35], clean[0, :35])
    assert not bool(got[0, 35:, :, 5].isfinite().any())
    rest = torch.cat((got[0, 35:, :, :5], got[0, 35:, :, 6:]), -1)
    assert bool(rest.isfinite().all())


def test_maxima_that_grow_rescale_what_is_there():
    """Keys whose scores rise by far more than the threshold from step to step, and rows that rise at different steps."""
    kv, q, table, lengths = setup([640], 64, 2, 1, 64, 64, BF16, BF16)
    for j in range(10):
        kv.keys[table[0, j]] *= (j + 1) * 2
    check(kv, q, table, lengths)
    check(kv, q, table, lengths, scale=-1.0)
    check(kv, q, table, lengths, scale=0.0)


def test_the_same_bits_and_graphs():
    kv, q, table, lengths = setup([900, 300, 2000], 64, 8, 2, 128, 16, BF16, BF16)
    first = kv.attend(q, table, lengths)
    assert all(torch.equal(kv.attend(q, table, lengths), first) for _ in range(5))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    other = q.flip(0).contiguous()
    want = kv.attend(other, table, lengths)
    for graph, x in zip(graphs, (q, other)):
        with torch.cuda.graph(graph):
            outs.append(kv.attend(x, table, lengths))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], want)


@pytest.mark.parametrize("t, hq, hk, d", [(1, 8, 2, 128), (64, 8, 2, 128), (64, 8, 2, 64), (48, 8, 2, 256)])
def test_the_same_bits_beside_another_call(t, hq, hk, d):
    """Two calls at once share the SMs: what a CTA computes does not depend on when or where it runs."""
    kv, q, table, lengths = setup([900, 300, 2000], t, hq, hk, d, 16, BF16, BF16)
    queries = (q, q.flip(0).contiguous())
    want = [kv.attend(x, table, lengths) for x in queries]
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, x in zip(graphs, queries):
        with torch.cuda.graph(graph):
            outs.append(kv.attend(x, table, lengths))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(100):
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    kv.check()


@pytest.mark.parametrize("t, hq, hk, d", [(1, 8, 2, 128), (40, 2, 1, 64), (64, 8, 2, 128), (70, 4, 2, 256)])
def test_calls_in_turn_do_not_see_each_others_scratch(t, hq, hk, d):
    """Two calls on other inputs in turn, whose scratch torch's allocator puts in the same place: a result that was joined too
    early would be the other call's."""
    kv, q, table, lengths = setup([900, 300, t, 2000, 640], t, hq, hk, d, 16, BF16, BF16)
    other = (q.flip(0) * -1).contiguous()
    want = {}
    for x in (q, other):
        out, bound, _ = su.attend(x[:, :1], kv.keys, kv.values, None, None, table, lengths.tolist(), d ** -0.5)
        want[x is q] = kv.attend(x, table, lengths).clone()
        su.assert_within(want[x is q][:, :1], out, bound)
    for _ in range(60):
        assert torch.equal(kv.attend(q, table, lengths), want[True])
        assert torch.equal(kv.attend(other, table, lengths), want[False])


def test_strided_queries_in_place():
    kv, q, table, lengths = setup([100, 70], 40, 4, 2, 64, 16, BF16, BF16)
    want = kv.attend(q, table, lengths)
    wide = torch.zeros(2, 40, 6, 80, device="cuda", dtype=BF16)
    view = wide[:, :, 1:5, 8:72]
    view.copy_(q)
    assert kv.attend(view, table, lengths, out=view) is view
    assert torch.equal(view, want) and not wide[:, :, 0].any() and not wide[:, :, :, :8].any()


def test_a_page_outside_the_pool():
    kv, q, table, lengths = setup([100, 200], 40, 4, 2, 64, 16, BF16, BF16)
    table[1, 3] = kv.keys.shape[0]
    got = kv.attend(q, table, lengths)
    want, bound, _ = su.attend(q, kv.keys, kv.values, None, None, table, lengths.tolist(), 64 ** -0.5)
    su.assert_within(got, want, bound)
    with pytest.raises(IndexError, match="row 1: page"):
        kv.check()
