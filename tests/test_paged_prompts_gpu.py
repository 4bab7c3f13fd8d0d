"""Attention of whole prompts (many tiles of rows, each of which sees another part of the keys), and of tables around the width up
to which nothing is split. Sampled tokens against 64 bits."""

import pytest
import torch

import serving_util as su
from test_paged_attend_gpu import check, setup
from test_paged_append_gpu import norm, tokens
from dlmrt_b200.ops.paged_kv import PagedKV, rotary_table

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def check_tokens(args, sampled, window=0):
    """Causal tokens one by one: token i sees what a single one would at the end of lengths - tokens + i + 1 keys."""
    kv, q, table, lengths = args
    got = kv.attend(q, table, lengths, causal=True, window=window)
    d = q.shape[3]
    for i in sampled:
        seen = (lengths - q.shape[1] + i + 1).clamp_min(0)
        want, bound, _ = su.attend(q[:, i:i + 1], kv.keys, kv.values, kv.k_scale, kv.v_scale, table, seen.tolist(), d ** -0.5, window, True)
        su.assert_within(got[:, i:i + 1], want, bound, f"token {i}")
    kv.check()
    return got


@pytest.mark.parametrize("window", [0, 1024])
@pytest.mark.parametrize("d, cache", [(64, F16), (128, BF16), (128, E4M3), (256, BF16), (256, E4M3)])
def test_a_prompt_of_some_hundred_tiles(d, cache, window):
    """4096 tokens of 8 query heads are 256 tiles of 128 rows over one key head."""
    args = setup([4096], 4096, 8, 1, d, 64, F16 if cache == F16 else BF16, cache)
    check_tokens(args, [0, 1, 15, 16, 63, 64, 1023, 1024, 1025, 2047, 3000, 4095], window)


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("d, cache", [(64, BF16), (128, BF16), (128, E4M3), (256, F16)])
def test_prompts_of_a_padded_batch_behind_prefixes(d, cache, window):
    """Shorter and longer than the batch's 700 tokens: tokens in front of the first key see nothing, others a prefix, too."""
    args = setup([700, 0, 500, 1999, 1, 701], 700, 4, 2, d, 16, F16 if cache == F16 else BF16, cache)
    got = check_tokens(args, [0, 1, 199, 200, 201, 350, 698, 699], window)
    assert not got[1].any() and not got[2, :200].any() and not got[4, :699].any()


def test_the_longest_block_of_tokens():
    args = setup([65536], 65536, 1, 1, 64, 256, BF16, BF16)
    check_tokens(args, [0, 63, 64, 127, 128, 40000, 65535])


@pytest.mark.parametrize("t, hq, hk", [(1, 8, 2), (4, 8, 2), (33, 2, 1)])
@pytest.mark.parametrize("d, cache", [(64, BF16), (128, F16), (128, E4M3), (256, BF16)])
@pytest.mark.parametrize("page", [16, 128])
def test_tables_around_the_width_up_to_which_nothing_is_split(page, d, cache, t, hq, hk):
    """384 keys and a page more, the lengths themselves around 384 and 64, with windows that make a wide table a short one."""
    kv, q, table, lengths = setup([384, 383, 321, t, 65, 384], t, hq, hk, d, page, F16 if cache == F16 else BF16, cache)
    table = table[:, :384 // page].contiguous()
    for extra in (0, 1):
        wide = torch.cat((table, table.new_full((6, extra), -1)), 1)
        check(kv, q, wide, lengths, causal=True)
        check(kv, q, wide, lengths)
    wide = torch.cat((table, table.new_full((6, 4096), -1)), 1)
    for window in (320 - t, 321 - t, 319 - t):  # window + tokens + 64 is 384, and one more and less
        check(kv, q, wide, lengths, window=window, causal=True)


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_a_prompt_enters_the_cache(cache):
    """3001 tokens, rows that are not stored behind the last one; every stored row against 64 bits."""
    n, hq, hk, d, page = 3001, 4, 2, 128, 32
    kv = PagedKV(*su.pool(100, hk, page, d, cache, 1, device="cuda"))
    q, k, v = tokens(n, hq, hk, d, BF16, 2)
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(100 * page, generator=g)[:n].cuda()
    slots[-5:] = -1
    positions, table, wk = torch.randint(0, 4096, (n,), generator=g).int().cuda(), rotary_table(d, 4096, device="cuda"), norm(d, BF16, 5)
    out = kv.append(k, v, positions, slots, table, q=q, k_norm=wk)
    kv.check()
    su.assert_within(out, *su.stored(*su.turned(q, None, table, positions, 1e-6, False), BF16), "queries")
    at = slots[:-5].cpu()
    for pool, x, w, t, scale in ((kv.keys, k, wk, table, kv.k_scale), (kv.values, v, None, None, kv.v_scale)):
        want, bound = su.stored(*su.turned(x, w, t, positions, 1e-6, False), cache, scale)
        su.assert_within(pool.cpu().double()[at // page, :, at % page], want[:-5], bound[:-5])


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("t, hq, hk", [(1, 8, 2), (6, 4, 2), (50, 2, 1)])
@pytest.mark.parametrize("page", [8, 64, 128])
def test_pages_in_front_of_the_window_may_be_gone(page, t, hq, hk, cache):
    """A sliding window gives pages back: entries that no token's window reaches are not looked at, whatever they say."""
    kv, q, table, lengths = setup([900, 300, 1 + t, 2000], t, hq, hk, 64, page, BF16, cache)
    window = 200
    want = kv.attend(q, table, lengths, window=window)
    gone = table.clone()
    for i, n in enumerate(lengths.tolist()):
        first = max(0, n - t - window + 1) // page  # the page of the first token's oldest key
        gone[i, :first] = torch.tensor([-1, 1 << 30, kv.keys.shape[0]], dtype=torch.int32, device="cuda").repeat(first)[:first]
    assert torch.equal(kv.attend(q, gone, lengths, window=window), want)
    kv.check()


@pytest.mark.parametrize("t", [1, 40])
def test_sequences_share_the_pages_of_a_prefix(t):
    kv, q, table, lengths = setup([640, 700, 655], t, 4, 2, 64, 16, BF16, BF16)
    shared = table.clone()
    shared[1:, :37] = table[0, :37]
    check(kv, q, shared, lengths, causal=True)
    lengths[2] = lengths[0]
    shared[2] = shared[0]
    q[2] = q[0]
    got = kv.attend(q, shared, lengths, causal=True)
    # cut into other runs: two roundings of sums whose weights (2^-15) and values (below 8) are the same
    su.assert_within(got[2], got[0].cpu().double(), 2 * su.HALF[BF16] * got[0].cpu().double().abs() + 2.0 ** -12)
