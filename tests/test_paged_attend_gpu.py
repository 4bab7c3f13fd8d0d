"""Attention over a paged cache on the GPU against 64 bits, at the lengths, masks and layouts where it can go wrong."""

import math

import pytest
import torch

import serving_util as su
from dlmrt_b200.ops.paged_kv import PagedKV

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def setup(lengths, t, hq, hk, d, page, dtype, cache, seed=0, layout="hnd", spare=2):
    pages = sum(-(-n // page) for n in lengths) + spare
    keys, values, ks, vs = su.pool(pages, hk, page, d, cache, seed, layout, "cuda")
    table = su.page_table(lengths, page, pages, seed + 1)
    q = (torch.randn(len(lengths), t, hq, d, generator=torch.Generator().manual_seed(seed + 2)) * 2).to(dtype).cuda()
    return PagedKV(keys, values, ks, vs), q, table.cuda(), torch.tensor(lengths).int().cuda()


def check(kv, q, table, lengths, window=0, causal=False, scale=None, out=None):
    b, t, hq, d = q.shape
    lse = torch.zeros(b, t, hq, device="cuda")
    got = kv.attend(q, table, lengths, out=out, lse=lse, window=window, causal=causal, scale=scale)
    want, bound, want_lse = su.attend(q, kv.keys, kv.values, kv.k_scale, kv.v_scale, table, lengths.tolist(),
                                      d ** -0.5 if scale is None else scale, window, causal)
    su.assert_within(got, want, bound, "out")
    assert torch.equal(lse.cpu() == -math.inf, want_lse == -math.inf)
    fine = want_lse > -math.inf
    # a score's error (2 d roundings of its products' magnitudes, at most |q||k|) plus the sum's and the logarithm's
    size = float(q.float().norm(dim=-1).max() * kv.keys.float().norm(dim=-1).max() * (1 if kv.k_scale is None else kv.k_scale.max())) * d ** -0.5
    off = (lse.cpu().double() - want_lse)[fine].abs()
    assert not len(off) or float(off.max()) <= 2 * d * su.U * size + 64 * su.U * (1 + float(want_lse[fine].abs().max()))
    kv.check()
    return got


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_single_tokens_of_ragged_lengths(d, dtype, cache):
    """Lengths around the tile (16 keys), the page, the warps of a CTA (64 keys) and the chunk (128 keys); 0 and 1."""
    args = setup([0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300], 1, 8, 2, d, 16, dtype, E4M3 if cache == "e4m3" else dtype)
    check(*args)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_sequences_that_are_split(d, dtype, cache):
    """More than 512 keys: work is cut into units of 64 keys, over as many CTAs as the GPU holds; items begin and end in the
    middle of a CTA's share, empty ones and ones of a single key among them."""
    args = setup([700, 0, 1, 1500, 64, 129, 0, 2000], 1, 8, 2, d, 16, dtype, E4M3 if cache == "e4m3" else dtype)
    check(*args)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [0, 500, 700])
@pytest.mark.parametrize("t, hq, hk", [(1, 40, 2), (7, 4, 2), (19, 4, 1)])
def test_split_sequences_with_masks_and_several_row_tiles(t, hq, hk, window, causal):
    check(*setup([1100, 19, 640, 1], t, hq, hk, 64, 32, BF16, BF16), window=window, causal=causal)


def test_many_sequences():
    """More items than CTAs, and more sequences than a CTA has threads."""
    lengths = [(i * 37) % 90 for i in range(700)]
    check(*setup(lengths, 1, 2, 1, 64, 16, BF16, BF16))
    lengths[350] = 3000
    check(*setup(lengths, 1, 2, 1, 64, 16, BF16, BF16))


def test_units_outnumber_what_fits():
    """One long sequence over every CTA, and a table much wider than any sequence needs."""
    kv, q, table, lengths = setup([9000], 1, 4, 2, 128, 64, BF16, BF16)
    check(kv, q, table, lengths)
    wide = torch.full((1, 100000), -1, device="cuda", dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    check(kv, q, wide, lengths)


@pytest.mark.parametrize("page", [8, 16, 32, 128, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_page_sizes_and_layouts(page, layout):
    check(*setup([5, 130, 257], 1, 4, 2, 64, page, BF16, BF16, layout=layout))
    check(*setup([5, 130, 257], 1, 4, 2, 64, page, BF16, E4M3, layout=layout))


@pytest.mark.parametrize("hq, hk", [(1, 1), (7, 7), (16, 1), (17, 1), (14, 2), (40, 5), (64, 1)])
def test_head_groups(hq, hk):
    check(*setup([33, 140], 1, hq, hk, 64, 16, F16, F16))


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("t, hq, hk, d", [(2, 4, 2, 128), (5, 14, 2, 64), (16, 4, 4, 256), (32, 8, 2, 128), (33, 3, 1, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_blocks_of_tokens(t, hq, hk, d, cache, causal):
    check(*setup([t, t + 1, 150, 290], t, hq, hk, d, 32, BF16, cache), causal=causal)


@pytest.mark.parametrize("window", [1, 2, 16, 37, 100, 4096])
@pytest.mark.parametrize("causal", [False, True])
def test_sliding_window(window, causal):
    check(*setup([6, 20, 150, 333], 6, 4, 2, 64, 16, BF16, BF16), window=window, causal=causal)
    check(*setup([1, 20, 150, 333], 1, 4, 2, 128, 16, F16, E4M3), window=window, causal=causal)


def test_tokens_in_front_of_the_first_key_see_nothing():
    """A sequence shorter than its block of tokens (a padded batch): causal rows in front of key 0 are empty."""
    got = check(*setup([0, 1, 3, 40], 5, 4, 2, 64, 16, BF16, BF16), causal=True)
    assert not got[0].any() and not got[1, :4].any() and not got[2, :2].any() and bool(got[2, 2].any())
    check(*setup([0, 2, 40], 5, 4, 2, 64, 16, BF16, BF16), causal=True, window=3)
    check(*setup([0, 2, 40], 5, 4, 2, 64, 16, BF16, BF16), window=3)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("special", [math.inf, -math.inf, math.nan])
def test_what_the_mask_hides_never_reaches_the_result(special, cache):
    """Infinities and NaN behind the end of a sequence, in pages it does not list, in front of the window, and in later
    tokens' keys and values, which other rows of the same tile do see."""
    if cache == E4M3 and not math.isnan(special):
        special = math.nan  # E4M3 has no infinity
    kv, q, table, lengths = setup([37, 53], 4, 4, 2, 64, 16, BF16, cache)
    clean = kv.attend(q, table, lengths, causal=True, window=20)
    used = torch.zeros(kv.keys.shape[0], 16, dtype=torch.bool)
    for i, n in enumerate(lengths.tolist()):
        for j in range(max(0, n - 4 - 20 + 1), n):
            used[table[i, j // 16], j % 16] = True
    for t in (kv.keys, kv.values):
        raw = t.transpose(1, 2)
        raw[~used.cuda()] = torch.tensor(special).to(t.dtype).cuda()
    assert torch.equal(kv.attend(q, table, lengths, causal=True, window=20), clean)
    # the last token of sequence 0: only row 3 sees it
    kv.keys[table[0, 2], :, 36 % 16] = torch.tensor(special).to(kv.keys.dtype).cuda()
    kv.values[table[0, 2], :, 36 % 16] = torch.tensor(special).to(kv.keys.dtype).cuda()
    got = kv.attend(q, table, lengths, causal=True, window=20)
    assert torch.equal(got[1], clean[1])
    want, bound, _ = su.attend(q, kv.keys[:, :, :, :].nan_to_num(0, 0, 0) if cache == BF16 else kv.keys.float().nan_to_num(0).to(E4M3),
                               kv.values.nan_to_num(0, 0, 0) if cache == BF16 else kv.values.float().nan_to_num(0).to(E4M3),
                               kv.k_scale, kv.v_scale, table, lengths.tolist(), 64 ** -0.5, 20, True)
    su.assert_within(got[0, :3], want[0, :3], bound[0, :3])
    assert not bool(got[0, 3].isfinite().all())


def test_large_scores_do_not_overflow():
    kv, q, table, lengths = setup([200], 1, 4, 2, 64, 16, BF16, BF16)
    check(kv, q * 64, table, lengths)
    check(kv, q, table, lengths, scale=0.0)
    check(kv, q, table, lengths, scale=-0.5)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4, 1e30])
def test_fp8_cache_takes_queries_of_any_size(size):
    """Products of an FP8 cache are of halves: BF16 queries are brought into their range row by row."""
    kv, q, table, lengths = setup([90], 1, 4, 2, 64, 16, BF16, E4M3)
    q[0, 0, 1] = 0
    check(kv, (q * size).to(BF16), table, lengths, scale=0.1 / size)


def test_pages_outside_the_pool_count_as_absent_and_are_reported():
    kv, q, table, lengths = setup([40, 70], 1, 4, 2, 64, 16, BF16, BF16)
    for bad in (-1, kv.keys.shape[0], 1 << 30):
        t = table.clone()
        t[1, 2] = bad
        got = kv.attend(q, t, lengths)
        want, bound, _ = su.attend(q, kv.keys, kv.values, None, None, t, lengths.tolist(), 64 ** -0.5)
        su.assert_within(got, want, bound)
        with pytest.raises(IndexError, match=f"row 1: page {bad}"):
            kv.check()


def test_lengths_outside_the_table_are_cut_and_reported():
    kv, q, table, lengths = setup([40, 70], 1, 4, 2, 64, 16, BF16, BF16)
    table = table[:, :5].contiguous()
    long = torch.tensor([40, 81]).int().cuda()
    table[1, 4] = 0
    got = kv.attend(q, table, long)
    want, bound, _ = su.attend(q, kv.keys, kv.values, None, None, table, [40, 80], 64 ** -0.5)
    su.assert_within(got, want, bound)
    with pytest.raises(IndexError, match="row 1: length 81"):
        kv.check()
    assert not kv.attend(q, table, torch.tensor([-3, 0]).int().cuda()).any()
    with pytest.raises(IndexError, match="row 0: length -3"):
        kv.check()


def test_strided_queries_in_place_and_three_dimensions():
    kv, q, table, lengths = setup([40, 70], 3, 4, 2, 64, 16, BF16, BF16)
    want = kv.attend(q, table, lengths)
    wide = torch.zeros(2, 3, 6, 80, device="cuda", dtype=BF16)
    view = wide[:, :, 1:5, 8:72]
    view.copy_(q)
    assert torch.equal(kv.attend(view, table, lengths), want)
    assert kv.attend(view, table, lengths, out=view) is view
    assert torch.equal(view, want) and not wide[:, :, 0].any() and not wide[:, :, :, :8].any() and not wide[:, :, :, 72:].any()
    one = q[:, 2].contiguous()
    assert torch.equal(kv.attend(one, table, lengths), kv.attend(one.unsqueeze(1), table, lengths).squeeze(1))
    assert torch.equal(kv.attend(q, table[:, :5], lengths), want)  # rows of a wider table


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("t", [1, 40])
def test_keys_and_values_in_one_pool(t, cache):
    """[pages, slot, keys or values, head, head dim], some heads and pages of a larger pool: any strides."""
    kv, q, table, lengths = setup([150, 70], t, 4, 2, 128, 16, BF16, cache)
    pages = kv.keys.shape[0]
    raw = torch.full((2 * pages, 16, 2, 5, 128), 0x7F, device="cuda", dtype=torch.uint8).repeat_interleave(kv.keys.element_size(), -1)
    both = raw.view(cache)[::2].transpose(1, 3)[:, 1:3]  # [pages, head, keys or values, slot, head dim]
    for i, pool in enumerate((kv.keys, kv.values)):
        both[:, :, i].view(torch.uint8).copy_(pool.view(torch.uint8)) if cache == E4M3 else both[:, :, i].copy_(pool)
    other = PagedKV(both[:, :, 0], both[:, :, 1], kv.k_scale, kv.v_scale)
    assert torch.equal(other.attend(q, table, lengths), kv.attend(q, table, lengths))
    k, v = (torch.randn(3, 2, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(2))
    slots = torch.tensor([int(table[0, 0]) * 16 + 3, int(table[1, 1]) * 16, -1], device="cuda")
    for pool in (kv, other):
        pool.append(k, v, None, slots)
        pool.check()
    assert torch.equal(other.attend(q, table, lengths), kv.attend(q, table, lengths))
    assert bool((raw.view(2 * pages, 16, 2, 5, -1)[1::2] == 0x7F).all()) and bool((raw[:, :, :, [0, 3, 4]] == 0x7F).all())


def test_no_pages_and_no_sequences():
    kv, q, table, lengths = setup([4], 1, 4, 2, 64, 16, BF16, BF16)
    none = torch.empty(1, 0, device="cuda", dtype=torch.int32)
    assert not kv.attend(q, none, torch.zeros(1, device="cuda", dtype=torch.int32)).any()
    assert kv.attend(q[:0], table[:0], lengths[:0]).shape == (0, 1, 4, 64)


def test_two_calls_at_once_and_captured_graphs_do_not_share_scratch():
    """Split sequences keep partial results in scratch: two streams, and two graphs replayed in turn, each have their own."""
    kv, q, table, lengths = setup([3000, 2000], 1, 8, 2, 64, 16, BF16, BF16)
    q2 = q.flip(0).contiguous()
    want, want2 = kv.attend(q, table, lengths), kv.attend(q2, table, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, got2 = [], []
    for _ in range(20):
        got.append(kv.attend(q, table, lengths))
        with torch.cuda.stream(side):
            got2.append(kv.attend(q2, table, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got) and all(torch.equal(x, want2) for x in got2)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph, x in zip(graphs, (q, q2)):
        with torch.cuda.graph(graph):
            outs.append(kv.attend(x, table, lengths))
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(main):
            graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)
    lengths -= 1000
    graphs[0].replay()
    assert torch.equal(outs[0], kv.attend(q, table, lengths))


def test_the_same_call_gives_the_same_bits():
    kv, q, table, lengths = setup([2500, 7, 900], 3, 8, 2, 128, 16, BF16, BF16)
    first = kv.attend(q, table, lengths, causal=True)
    assert all(torch.equal(kv.attend(q, table, lengths, causal=True), first) for _ in range(5))


def test_the_join_of_two_halves_is_the_whole():
    """lse is what a caller needs to join attention over two sets of keys."""
    kv, q, table, lengths = setup([640], 1, 4, 2, 64, 16, F16, F16)
    want, bound, _ = su.attend(q, kv.keys, kv.values, None, None, table, [640], 64 ** -0.5)
    parts = []
    for lo in (0, 320):
        lse = torch.empty(1, 1, 4, device="cuda")
        parts.append((kv.attend(q, table[:, lo // 16:lo // 16 + 20], torch.tensor([320]).int().cuda(), lse=lse).double(), lse.double()))
    w = torch.softmax(torch.stack([p[1] for p in parts]), 0).unsqueeze(-1)
    su.assert_within((parts[0][0] * w[0] + parts[1][0] * w[1]), want, 2 * bound)


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("cache", [F16, E4M3, BF16])
def test_many_keys_of_small_weight(cache, t):
    """One key outweighs each of the others by e^18, about 2^26. Weights are taken as halves (BF16 without FP8 or FP16), at
    least 2^7 for the heaviest key: half a step of the smallest is 2^-25, that of a light weight 2^7 e^-18 within 1 / 64 of it."""
    n, d, b = 8000, 64, 40
    kv, q, table, lengths = setup([n], t, 8, 8, d, 64, BF16 if cache == BF16 else F16, cache)
    q, table, lengths = q.repeat(b, 1, 1, 1), table.repeat(b, 1), lengths.repeat(b)  # more heads than CTAs: each meets all keys
    kv.keys.zero_(), kv.values.fill_(8), q.zero_()
    if cache == E4M3:
        kv.k_scale.fill_(1), kv.v_scale.fill_(1)
    q[..., 0] = 1
    first = table[0, 0]
    kv.keys[first, :, 0, 0] = 18
    kv.values[first, :, 0] = 0
    light = (n - 1) * math.exp(-18)
    want = 8 * light / (1 + light)
    got = kv.attend(q, table, lengths, scale=1.0).double()
    assert float((got / want - 1).abs().max()) <= 1 / 64 + 2 * su.HALF[q.dtype]
    kv.check()


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements, read at its end."""
    pages, page, hk, d = 33000, 128, 4, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free memory")
    keys = torch.zeros(pages, hk, page, d, device="cuda", dtype=BF16)
    values = torch.zeros_like(keys)
    small = su.pool(3, hk, page, d, BF16, 3, device="cuda")
    ids = torch.tensor([[pages - 1, 0, pages - 2]], device="cuda", dtype=torch.int32)
    kv = PagedKV(keys, values)
    for t, s in zip((keys, values), small):
        t[ids[0].long()] = s
    q = torch.randn(1, 1, 8, d, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    lengths = torch.tensor([300], device="cuda", dtype=torch.int32)
    other = PagedKV(*small[:2])
    want = other.attend(q, torch.tensor([[0, 1, 2]], device="cuda", dtype=torch.int32), lengths)
    assert torch.equal(kv.attend(q, ids, lengths), want)
    k = torch.ones(1, hk, d, device="cuda", dtype=BF16)
    kv.append(k, k * 2, None, torch.tensor([pages * page - 1], device="cuda"))
    assert bool((keys[-1, :, -1] == 1).all()) and bool((values[-1, :, -1] == 2).all()) and not bool((keys[-2, :, -1] == 1).all())
    kv.check()
