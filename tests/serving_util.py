"""Plain 64-bit implementations of the paged cache's operators and of low-rank adapters, for the parity tests, with how far
a correct kernel may be off: counts of roundings, in the terms of each formula.

U is the relative error of one FP32 rounding. A matrix instruction may drop low bits when it aligns its addends, so a sum of
n products counts 2 n U of the sum of magnitudes. HALF[t] is half a step of an output type."""

import math

import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float8_e4m3fn: 2.0 ** -10}  # half the smallest step
E4M3_MAX = 448.0


def pool(pages, heads, page, dim, dtype, seed, layout="hnd", device="cpu"):
    """(keys, values, k_scale, v_scale) with random contents. `layout`: order of heads and slots in memory."""
    g = torch.Generator().manual_seed(seed)
    out, scales = [], [None, None]
    for i in range(2):
        t = torch.randn(pages, heads, page, dim, generator=g)
        if dtype == torch.float8_e4m3fn:
            scales[i] = (torch.rand(heads, generator=g) * 0.03 + 0.01).to(device)
            t = (t / scales[i].cpu().view(1, -1, 1, 1)).clamp(-E4M3_MAX, E4M3_MAX)
        t = t.to(dtype)
        if layout == "nhd":
            t = t.transpose(1, 2).contiguous().transpose(1, 2)
        out.append(t.to(device))
    return *out, *scales


def page_table(lengths, page, pages, seed, extra=1):
    """Random distinct pages for sequences of these lengths, -1 behind the last one."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    width = max(-(-n // page) for n in lengths) + extra
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for i, n in enumerate(lengths):
        for j in range(-(-n // page)):
            table[i, j] = order.pop()
    return table


def attend(q, keys, values, k_scale, v_scale, table, lengths, scale, window=0, causal=False):
    """(out, bound, lse) in 64 bits. `bound`: |error| of a kernel that forms scores and sums in FP32, rounds each weight of
    the softmax once to the type its products are of (halves for an FP8 cache) and the result once to q's type."""
    q, keys, values, table = (t.cpu() for t in (q, keys, values, table))
    b, t, hq, d = q.shape
    hk, page = keys.shape[1], keys.shape[2]
    out, bound = torch.zeros(b, t, hq, d, dtype=torch.float64), torch.zeros(b, t, hq, d, dtype=torch.float64)
    lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64)
    narrow = torch.float16 if keys.dtype == torch.float8_e4m3fn else q.dtype
    for i in range(b):
        n = int(lengths[i])
        ids = table[i, :-(-n // page)].long()
        there = ((ids >= 0) & (ids < len(keys))).repeat_interleave(page)[:n]
        ids = ids.clamp(0, len(keys) - 1)
        k, v = (x[ids].double().transpose(1, 2).reshape(-1, hk, d)[:n] for x in (keys, values))
        if k_scale is not None:
            k, v = k * k_scale.cpu().double().view(1, -1, 1), v * v_scale.cpu().double().view(1, -1, 1)
        for j in range(t):
            at = n - t + j
            see = there & (torch.arange(n) < (at + 1 if causal else n))
            if window:
                see &= torch.arange(n) > at - window
            see = see.nonzero().squeeze(1)
            if not len(see):
                continue
            for h in range(hq):
                kk, vv, qq = k[see, h // (hq // hk)], v[see, h // (hq // hk)], q[i, j, h].double()
                s = kk @ qq * scale
                p = torch.softmax(s, 0)
                out[i, j, h] = p @ vv
                lse[i, j, h] = torch.logsumexp(s, 0)
                # a score's error, absolute: it is the relative error of its weight, and of the sum of weights
                off = float((2 * d * U * (kk.abs() @ qq.abs()) * abs(scale) + 8 * U * s.abs()).max())
                weight = HALF[narrow] + 2 * off + 2 * len(see) * U + 16 * U
                size = p @ vv.abs()
                lost = len(see) * TINY[torch.float16] * vv.abs().max(0).values if narrow == torch.float16 else 0.0
                bound[i, j, h] = weight * size + lost + HALF[q.dtype] * (out[i, j, h].abs() + weight * size) + TINY[q.dtype]
    return out, bound, lse


def turned(x, weight, table, positions, eps, interleaved):
    """(values, bound before the store's rounding) of norm and rotation in 64 bits; x [n, heads, d]."""
    x, d = x.cpu().double(), x.shape[-1]
    error = torch.zeros_like(x)
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.cpu().double()
        error = (d / 2 + 12) * U * x.abs()  # sum of d squares, reciprocal root (2 steps), two products
    if table is None:
        return x, error
    table = table.cpu().double()[positions.cpu().long()]
    half = table.shape[1] // 2
    c, s = table[:, None, :half], table[:, None, half:]
    y, bound = x.clone(), error.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size = x[..., a].abs() + x[..., b].abs()
    bound[..., a] = bound[..., b] = error[..., a] + error[..., b] + 3 * U * size
    return y, bound


def stored(x, bound, dtype, scale=None):
    """(values, bound) as the cache holds them, from turned()'s: rounded once, FP8 after division by the head's scale."""
    if scale is not None:
        s = scale.cpu().double().view(1, -1, 1)
        x, bound = (x / s).clamp(-E4M3_MAX, E4M3_MAX), bound / s + 2 * U * (x / s).abs()
    return x, bound + HALF[dtype] * (x.abs() + bound) + TINY[dtype]


def adapters(x, ids, base, a, b, scales):
    """(out, bound): FP32 sums over k, the low-rank vector split into two BF16 words (16 bits), one rounding at the end."""
    x, ids, base, a, b, scales = (t.cpu() for t in (x, ids, base, a, b, scales))
    out = base.double().clone()
    bound = torch.zeros_like(out)
    for i, e in enumerate(ids.tolist()):
        if 0 <= e < len(a):
            k, rank = a.shape[2], a.shape[1]
            low = a[e].double() @ x[i].double()
            off = (2 * k + 16) * U * (a[e].double().abs() @ x[i].double().abs()) + 2.0 ** -16 * low.abs()
            out[i] += float(scales[e]) * (b[e].double() @ low)
            bound[i] = float(scales[e]) * (b[e].double().abs() @ (off + (4 * rank + 4) * U * low.abs()))
        bound[i] += (HALF[torch.bfloat16] + 2 * U) * (out[i].abs() + bound[i]) * (0 <= e < len(a)) + TINY[torch.bfloat16]
    return out, bound


def assert_within(got, want, bound, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)  # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).nan_to_num(float('inf')).max()):.3g} " \
                          f"times the bound, first at {tuple(bad.nonzero()[0].tolist())}"
