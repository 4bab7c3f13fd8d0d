"""How exactly attention over the paged cache holds the weights of the softmax: results whose keys' values partly cancel are as
near to 64 bits as one rounding of the result allows, which weights of one 16-bit value each are not."""

import math

import pytest
import torch

import serving_util as su
from test_paged_attend_gpu import check as check_against_64_bits, setup

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn

# A weight is a high and a low value of the products' type. What is left of it after the high one (towards zero: less than a step,
# and what the low one is made larger by) is rounded once: relative to the weight half a step of that. Halves also end at 2^-24.
SPLIT = {BF16: 2.0 ** -8 * (2.0 ** -7 + 2.0 ** -20) + 2.0 ** -20, F16: 2.0 ** -11 * (2.0 ** -10 + 2.0 ** -12) + 2.0 ** -22}
NONZERO = 8  # elements of a query that are not zero


def expect(kv, q, table, lengths, scale, causal, window):
    """(out, bound) in 64 bits, as serving_util.attend, for queries of NONZERO elements."""
    keys, values, table = kv.keys.cpu().double(), kv.values.cpu().double(), table.cpu()
    if kv.k_scale is not None:
        keys, values = (x * s.cpu().double().view(1, -1, 1, 1) for x, s in ((keys, kv.k_scale), (values, kv.v_scale)))
    b, t, hq, d = q.shape
    hk, page = keys.shape[1], keys.shape[2]
    dtype, q = q.dtype, q.cpu().double().view(b, t, hk, hq // hk, d)
    products = F16 if kv.dtype == E4M3 else kv.dtype
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i, n in enumerate(lengths.tolist()):
        if n == 0:
            continue
        k, v = (x[table[i, :-(-n // page)].long()].transpose(0, 1).reshape(hk, -1, d)[:, :n] for x in (keys, values))
        s = torch.einsum("thgd,hnd->htgn", q[i], k) * scale
        size = torch.einsum("thgd,hnd->htgn", q[i].abs(), k.abs()) * scale
        at, place = torch.arange(n), n - t + torch.arange(t).view(-1, 1)
        see = (at <= place if causal else at >= 0) & (at > place - window if window else at >= 0)
        see = see.expand(t, n).view(1, t, 1, n)
        p = torch.softmax(s.masked_fill(~see, -math.inf), -1).nan_to_num(0)
        # a score's error, absolute, is the relative error of its weight; a cancelled sum of weights has theirs
        off = torch.where(see, 2 * NONZERO * su.U * size + 8 * su.U * s.abs(), 0.0).amax(-1, keepdim=True)
        weight = SPLIT[products] + 2 * off + 2 * n * su.U + 16 * su.U
        mean, most = (torch.einsum("htgn,hnd->thgd", p, x) for x in (v, v.abs()))
        off = weight.permute(1, 0, 2, 3) * most
        if products == F16:  # the heaviest weight is at least 2^7, steps are 2^-24 and rounded once in the low part
            off = off + n * 2.0 ** -32 * v.abs().amax(1).view(1, hk, 1, d)
        out[i], bound[i] = mean, off + su.HALF[dtype] * (mean.abs() + off) + su.TINY[dtype]
    return out.view(b, t, hq, d), bound.view(b, t, hq, d)


def sparse(q, seed):
    """q with NONZERO elements of each row left: scores whose own rounding is far below that of a 16-bit weight."""
    g = torch.Generator().manual_seed(seed)
    keep = torch.rand(q.shape, generator=g).argsort(-1) < NONZERO
    return torch.where(keep.cuda(), q, 0).contiguous()


def check(args, causal=False, window=0):
    kv, q, table, lengths = args
    q = sparse(q, 9)
    want, bound = expect(kv, q, table, lengths, 0.5, causal, window)
    su.assert_within(kv.attend(q, table, lengths, scale=0.5, causal=causal, window=window), want, bound)
    kv.check()


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t, hq", [(1, 8), (2, 16)])
def test_few_rows(t, hq, d, dtype, cache):
    """4 and 16 rows a key head, whole (tables of 300 keys) and split."""
    cache = E4M3 if cache == "e4m3" else dtype
    check(setup([0, 5, 63, 300], t, hq, 2, d, 16, dtype, cache), causal=t > 1)
    check(setup([700, 2, 1500, 64], t, hq, 2, d, 32, dtype, cache), window=900)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_blocks_of_tokens(d, dtype, cache):
    """The kernel for more rows than two tiles hold, whole and split."""
    cache = E4M3 if cache == "e4m3" else dtype
    check(setup([40, 63, 300], 40, 4, 2, d, 16, dtype, cache), causal=True)
    check(setup([700, 41, 1500], 33, 2, 1, d, 32, dtype, cache), window=900)


@pytest.mark.parametrize("size", [1e-35, 1e-36, 1e-37, 3e36])
@pytest.mark.parametrize("t, hq", [(1, 4), (40, 4)])
def test_queries_at_both_ends_of_bf16_over_codes(t, hq, size):
    """Rows whose largest element is near 2^-126 or 2^126 are brought into the range of halves as any others."""
    kv, q, table, lengths = setup([90, 333], t, hq, 2, 64, 16, BF16, E4M3)
    q[:, 0, 1] = 0
    check_against_64_bits(kv, (q * size).to(BF16), table, lengths, scale=0.1 / size)
