"""The operators around a denoise round's projections as cases that can be timed and compared: appending rotated keys and
values to a paged cache, attention of new tokens over that cache, and low-rank adapters beside a shared projection.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare(case, seed)` makes what a program
holds before the call, `run(state)` is one pass (in elementary torch operations, or where `own` is true through this
package's entry points), `work(case)` what the pass cannot do without, and `exact(case, seed)` the same outputs in 64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
THETA = 1e6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "f16": 2, "e4m3": 1}
E4M3_MAX = 448.0


def listed():
    return [
        # One new token of one conversation enters the cache: the smallest call, latency only. Heads of a dense 4B model.
        dict(name="append_token", kind="append", tokens=1, sequences=1, q_heads=32, kv_heads=8, head_dim=128, page=16,
             dtype="bf16", cache="bf16", rotated=128, interleaved=False, norm=True, pad=0, positions=32768),
        # A denoise round's 256-token block, cache in FP8, two padded rows behind the last token.
        dict(name="append_block", kind="append", tokens=256, sequences=1, q_heads=32, kv_heads=8, head_dim=128, page=64,
             dtype="bf16", cache="e4m3", rotated=128, interleaved=False, norm=True, pad=2, positions=32768),
        # A prompt of several requests in one pass: heads of 256, half of each rotated, neighbouring pairs, odd token count.
        dict(name="append_prompt", kind="append", tokens=8189, sequences=5, q_heads=16, kv_heads=8, head_dim=256, page=32,
             dtype="bf16", cache="bf16", rotated=128, interleaved=True, norm=False, pad=0, positions=16384),
        # One new token over a short context: latency, from Python.
        dict(name="attend_token", kind="attend", batch=1, tokens=1, shortest=257, longest=257, q_heads=32, kv_heads=8,
             head_dim=128, page=16, dtype="bf16", cache="bf16", window=0, causal=False),
        # A serving batch of single tokens, ragged contexts from a few tokens to 8192: the largest.
        dict(name="attend_batch", kind="attend", batch=64, tokens=1, shortest=129, longest=8192, q_heads=32, kv_heads=8,
             head_dim=128, page=16, dtype="bf16", cache="bf16", window=0, causal=False),
        # One request with a long context and few heads: parallel only along the cache.
        dict(name="attend_long", kind="attend", batch=1, tokens=1, shortest=131071, longest=131071, q_heads=16, kv_heads=4,
             head_dim=128, page=64, dtype="bf16", cache="bf16", window=0, causal=False),
        # FP8 cache, heads of 256, two query heads for each key head.
        dict(name="attend_fp8", kind="attend", batch=24, tokens=1, shortest=1000, longest=12000, q_heads=16, kv_heads=8,
             head_dim=256, page=32, dtype="bf16", cache="e4m3", window=0, causal=False),
        # Sixteen requests' 32-token blocks over their prefixes: every token of a block sees the whole block.
        dict(name="attend_block", kind="attend", batch=16, tokens=32, shortest=1056, longest=8224, q_heads=32, kv_heads=8,
             head_dim=128, page=64, dtype="bf16", cache="bf16", window=0, causal=False),
        # Five drafted tokens checked at once, causal among themselves, sliding window, a head count of seven per key head.
        dict(name="attend_draft", kind="attend", batch=9, tokens=5, shortest=40, longest=6001, q_heads=14, kv_heads=2,
             head_dim=64, page=16, dtype="f16", cache="f16", window=2048, causal=True),
        # One row with an adapter beside a 4B model's output projection: latency.
        dict(name="adapters_row", kind="adapters", rows=1, adapters=4, rank=16, k=4096, n=2560, idle=0.0),
        # A serving batch in which most rows have an adapter of their own; some rows have none.
        dict(name="adapters_mixed", kind="adapters", rows=61, adapters=48, rank=16, k=2560, n=9728, idle=0.15),
        # Full block of rows over a few adapters of a high rank beside the down-projection.
        dict(name="adapters_block", kind="adapters", rows=256, adapters=8, rank=64, k=9728, n=2560, idle=0.0),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "adapters"])
    if kind == "adapters":
        return dict(kind=kind, rows=_log(rng, 1, 256), adapters=_log(rng, 1, 64), rank=rng.choice([8, 16, 24, 32, 64]),
                    k=_log(rng, 256, 9728, 8), n=_log(rng, 256, 9728, 8), idle=rng.choice([0.0, 0.0, 0.3]))
    kv_heads, head_dim = rng.randint(1, 8), rng.choice([64, 128, 128, 256])
    heads = dict(q_heads=kv_heads * rng.randint(1, 8), kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([16, 32, 64, 128]))
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads |= dict(dtype=dtype, cache=rng.choice([dtype, dtype, "e4m3"]))
    if kind == "append":
        tokens = _log(rng, 1, 4096)
        return dict(kind=kind, tokens=tokens, sequences=rng.randint(1, min(tokens, 64)), **heads,
                    rotated=rng.choice([head_dim, head_dim, head_dim // 2]), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.5, pad=rng.choice([0, 0, 3]) if tokens > 3 else 0, positions=16384)
    tokens = rng.choice([1, 1, 1, rng.randint(2, 32)])
    batch = _log(rng, 1, 64)
    longest = _log(rng, 64, min(65536, 196608 // batch))
    return dict(kind=kind, batch=batch, tokens=tokens, shortest=_log(rng, min(tokens, longest), longest), longest=longest, **heads,
                window=rng.choice([0, 0, 1024]), causal=rng.random() < 0.5)


# -- inputs --------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Context lengths from the shortest to the longest, evenly on a logarithmic scale (they follow from the case alone, the
    order from the seed)."""
    steps = max(case["batch"] - 1, 1)
    ratio = case["longest"] / case["shortest"]
    return [int(round(case["shortest"] * ratio ** (i / steps))) for i in range(case["batch"])]


def _pool(g, case, pages):
    """Pages of keys and values as earlier tokens left them: values of order one, in FP8 as codes of a scale per head."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    scales = None
    pool = []
    if case["cache"] == "e4m3":
        scales = [torch.rand(case["kv_heads"], generator=g, device=DEVICE) * 0.02 + 0.01 for _ in range(2)]
    for i in range(2):
        t = torch.empty(shape, device=DEVICE, dtype=TYPES[case["dtype"]]).normal_(generator=g)
        if scales is not None:
            t = (t / scales[i].view(1, -1, 1, 1).to(t.dtype)).clamp_(-E4M3_MAX, E4M3_MAX).to(TYPES["e4m3"])
        pool.append(t)
    return pool, scales


def _prepare_append(case, g):
    n, sequences, page, d = case["tokens"], case["sequences"], case["page"], case["head_dim"]
    hq, hk = case["q_heads"], case["kv_heads"]
    most = -(-n // sequences)                       # tokens of the longest sequence
    per_sequence = -(-(most + page - 1) // page)    # pages that they can touch
    pages = sequences * per_sequence + 64
    pool, scales = _pool(g, case, pages)
    qkv = torch.empty(n, (hq + 2 * hk) * d, device=DEVICE, dtype=TYPES[case["dtype"]]).normal_(generator=g)
    q, k, v = (t.view(n, -1, d) for t in qkv.split((hq * d, hk * d, hk * d), 1))
    token = torch.arange(n, device=DEVICE)
    sequence = token * sequences // n
    within = token - (sequence * n + sequences - 1) // sequences
    start = torch.randint(0, case["positions"] - most, (sequences,), generator=g, device=DEVICE)
    positions = start[sequence] + within
    logical = start[sequence] % page + within
    order = torch.randperm(pages, generator=g, device=DEVICE)
    slots = order[sequence * per_sequence + logical // page] * page + logical % page
    if case["pad"]:
        slots[n - case["pad"]:] = -1
    half = case["rotated"] // 2
    angle = torch.arange(case["positions"], device=DEVICE, dtype=torch.float64).view(-1, 1) \
        * THETA ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    table = torch.cat((angle.cos(), angle.sin()), 1).float()
    norms = [torch.empty(d, device=DEVICE, dtype=q.dtype).normal_(1.0, 0.1, generator=g) for _ in range(2)]
    return dict(q=q, k=k, v=v, positions=positions.int(), slots=slots, table=table, pool=pool, scales=scales,
                norms=norms if case["norm"] else (None, None))


def _prepare_attend(case, g):
    b, t, page = case["batch"], case["tokens"], case["page"]
    lengths = torch.tensor(_lengths(case), device=DEVICE)[torch.randperm(b, generator=g, device=DEVICE)]
    held = -(-case["longest"] // page)
    used = sum(-(-n // page) for n in _lengths(case))
    pool, scales = _pool(g, case, used + 16)
    need = (lengths + page - 1) // page
    column = torch.arange(held, device=DEVICE)
    order = torch.randperm(used + 16, generator=g, device=DEVICE)
    at = (need.cumsum(0) - need).view(-1, 1) + column
    table = torch.where(column < need.view(-1, 1), order[at.clamp_max(used + 15)], -1).int()
    q = torch.empty(b, t, case["q_heads"], case["head_dim"], device=DEVICE, dtype=TYPES[case["dtype"]]).normal_(0, 2, generator=g)
    return dict(q=q, pages=table, lengths=lengths.int(), pool=pool, scales=scales)


def _prepare_adapters(case, g):
    m, count, r, k, n = case["rows"], case["adapters"], case["rank"], case["k"], case["n"]
    bf16 = dict(device=DEVICE, dtype=torch.bfloat16)
    ids = torch.arange(m, device=DEVICE) % count  # every adapter that the rows can reach is reached
    ids[: _idle(case)] = -1
    return dict(a=torch.empty(count, r, k, **bf16).normal_(0, k ** -0.5, generator=g),
                b=torch.empty(count, n, r, **bf16).normal_(0, 0.5 * r ** -0.5, generator=g),
                scales=torch.rand(count, generator=g, device=DEVICE) * 2 + 0.5,
                x=torch.empty(m, k, **bf16).normal_(generator=g), base=torch.empty(m, n, **bf16).normal_(generator=g),
                ids=ids[torch.randperm(m, generator=g, device=DEVICE)].int())


def _idle(case):
    """Rows without an adapter: the first so many before the rows are mixed."""
    return int(case["rows"] * case["idle"])


def prepare(case, seed):
    torch.cuda.set_device(DEVICE)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"append": _prepare_append, "attend": _prepare_attend, "adapters": _prepare_adapters}[case["kind"]](case, g)
    state["case"] = case
    if own:  # the objects that a program makes once, when it allocates its cache and loads its adapters
        if case["kind"] == "adapters":
            from dlmrt_b200.layers.adapters import Adapters

            state["adapters"] = Adapters(state["a"], state["b"], state["scales"])
        else:
            from dlmrt_b200.ops.paged_kv import PagedKV

            state["cache"] = PagedKV(*state["pool"], *(state["scales"] or ()))
    return state


# -- one pass ------------------------------------------------------------------------------------------------------------
def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _rotated(x, cos, sin, interleaved):
    """The first 2 * half elements of each head turned by the angles of its token; the rest as it is."""
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _append(state):
    case, table = state["case"], state["table"]
    half = table.shape[1] // 2
    rows = table[state["positions"].long()].unsqueeze(1)
    cos, sin = rows[..., :half], rows[..., half:]
    weights = [w if w is None else w.float() for w in state["norms"]]
    q = _rotated(_normed(state["q"].float(), weights[0]), cos, sin, case["interleaved"]).to(state["q"].dtype)
    k = _rotated(_normed(state["k"].float(), weights[1]), cos, sin, case["interleaved"])
    # A padded row writes once more what the first real one writes: no row has to be looked for on the host.
    real = state["slots"] >= 0
    source = torch.where(real, torch.arange(len(real), device=DEVICE), real.int().argmax())
    slots = state["slots"][source]
    page, offset = slots // case["page"], slots % case["page"]
    keys, values = state["pool"]
    keys[page, :, offset] = _held(k[source], state["scales"], 0, keys.dtype)
    values[page, :, offset] = _held(state["v"].float()[source], state["scales"], 1, values.dtype)
    return q, keys, values


def _held(x, scales, which, dtype):
    """x as the cache holds it: rounded, in FP8 after division by the head's scale, at most the largest code."""
    return x.to(dtype) if scales is None else (x / scales[which].view(1, -1, 1)).clamp(-E4M3_MAX, E4M3_MAX).to(dtype)


def _context(state, which):
    """Keys or values of every sequence, gathered from its pages: [batch, kv heads, slots of the table, head dim] FP32."""
    x = state["pool"][which][state["pages"].clamp_min(0).long()].float()
    if state["scales"] is not None:
        x = x * state["scales"][which].view(1, 1, -1, 1, 1)
    b, pages, heads, page, d = x.shape
    return x.transpose(1, 2).reshape(b, heads, pages * page, d)


def _attend(state):
    case, q, lengths = state["case"], state["q"], state["lengths"].long()
    b, t, hq, d = q.shape
    hk = case["kv_heads"]
    keys = _context(state, 0)
    rows = q.float().view(b, t, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, t * (hq // hk), d)
    scores = (rows @ keys.transpose(-1, -2) * d ** -0.5).view(b, hk, t, hq // hk, -1)
    del keys
    at = torch.arange(scores.shape[-1], device=DEVICE).view(1, 1, 1, 1, -1)
    end = lengths.view(-1, 1, 1, 1, 1)
    position = end - t + torch.arange(t, device=DEVICE).view(1, 1, -1, 1, 1)
    seen = at < end
    if case["causal"]:
        seen = seen & (at <= position)
    if case["window"]:
        seen = seen & (at > position - case["window"])
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))  # a row that sees nothing: zeros
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(b, hk, t * (hq // hk), -1)
    out = p @ _context(state, 1)
    return out.view(b, hk, t, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype)


def _adapters(state):
    ids = state["ids"].long()
    has = ids.clamp_min(0)
    low = state["a"][has].float() @ state["x"].float().unsqueeze(-1)
    delta = (state["b"][has].float() @ low).squeeze(-1) * state["scales"][has].unsqueeze(-1)
    base = state["base"].float()
    return torch.where(ids.unsqueeze(-1) < 0, base, base + delta).to(state["base"].dtype)


def run(state):
    kind, case = state["case"]["kind"], state["case"]
    if not own:
        return {"append": _append, "attend": _attend, "adapters": _adapters}[kind](state)
    if kind == "append":
        q = state["cache"].append(state["k"], state["v"], state["positions"], state["slots"], state["table"], q=state["q"],
                                  q_norm=state["norms"][0], k_norm=state["norms"][1], eps=EPS, interleaved=case["interleaved"])
        return q, *state["pool"]
    if kind == "attend":
        return state["cache"].attend(state["q"], state["pages"], state["lengths"], window=case["window"], causal=case["causal"])
    return state["adapters"](state["x"], state["ids"], state["base"])


# -- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "adapters":
        m, r, k, n = case["rows"], case["rank"], case["k"], case["n"]
        active = m - _idle(case)
        distinct = min(active, case["adapters"])
        return {"bytes": distinct * r * (k + n) * 2 + active * k * 2 + 2 * m * n * 2 + m * 4,
                "flops": 2 * active * r * (k + n)}
    hq, hk, d, size = case["q_heads"], case["kv_heads"], case["head_dim"], SIZE[case["cache"]]
    if case["kind"] == "append":
        n, held = case["tokens"], case["tokens"] - case["pad"]
        moved = 2 * n * hq * d * 2 + held * 2 * hk * d * (2 + size)
        return {"bytes": moved + n * (case["rotated"] * 4 + 12), "flops": n * (hq + hk) * (3 * case["rotated"] + 4 * d * case["norm"])}
    t, w = case["tokens"], case["window"]
    read = pairs = 0
    for n in _lengths(case):
        first = max(0, n - t - w + 1) if w else 0   # the oldest key that the first token's window holds
        read += n - first
        if not w and not case["causal"]:
            pairs += t * n
        else:
            pairs += sum(max(0, (n - t + i + 1 if case["causal"] else n) - max(0, n - t + i - w + 1 if w else 0)) for i in range(t))
    return {"bytes": read * 2 * hk * d * size + 2 * case["batch"] * t * hq * d * 2 + 4 * case["batch"] + 4 * (read // case["page"]),
            "flops": 4 * pairs * hq * d}


# -- the same in 64 bits, from the definitions ---------------------------------------------------------------------------
def _exact_append(case, s):
    half = case["rotated"] // 2
    keys, values = (t.double() for t in s["pool"])
    written = (s["slots"] >= 0).nonzero().squeeze(1)
    slots = s["slots"][written]
    turned = []
    for x, weight in zip((s["q"], s["k"]), s["norms"]):
        x = x.double()
        if weight is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / case["head_dim"] + EPS).sqrt() * weight.double()
        angle = s["table"].double().index_select(0, s["positions"].long())
        z = torch.complex(angle[:, :half], angle[:, half:]).unsqueeze(1)
        if case["interleaved"]:
            pairs = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:2], half, 2).contiguous())
            x = torch.cat((torch.view_as_real(pairs * z).reshape(*x.shape[:2], 2 * half), x[..., 2 * half:]), -1)
        else:
            pairs = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z
            x = torch.cat((pairs.real, pairs.imag, x[..., 2 * half:]), -1)
        turned.append(x)
    for pool, new, i in ((keys, turned[1], 0), (values, s["v"].double(), 1)):
        if s["scales"] is not None:
            new = (new / s["scales"][i].double().view(1, -1, 1)).clamp(-E4M3_MAX, E4M3_MAX)
        flat = pool.transpose(1, 2).reshape(-1, case["kv_heads"], case["head_dim"])
        flat[slots] = new[written]
        pool.copy_(flat.view(-1, case["page"], case["kv_heads"], case["head_dim"]).transpose(1, 2))
    return turned[0], keys, values


def _exact_attend(case, s):
    b, t, hq, d = s["q"].shape
    hk, page = case["kv_heads"], case["page"]
    out = torch.zeros(b, t, hq, d, device=DEVICE, dtype=torch.float64)
    for i, n in enumerate(s["lengths"].tolist()):
        ids = s["pages"][i, :-(-n // page)].long()
        keys, values = (pool[ids].double().transpose(1, 2).reshape(-1, hk, d)[:n] for pool in s["pool"])
        if s["scales"] is not None:
            keys, values = (x * c.double().view(1, -1, 1) for x, c in zip((keys, values), s["scales"]))
        where = torch.arange(n, device=DEVICE)
        for j in range(t):
            at = n - t + j
            lo = max(0, at - case["window"] + 1) if case["window"] else 0
            hi = at + 1 if case["causal"] else n
            if hi <= lo:
                continue
            span = where[lo:hi]
            q = s["q"][i, j].double().view(hk, hq // hk, d)
            score = torch.einsum("hgd,nhd->hgn", q, keys[span]) / math.sqrt(d)
            out[i, j] = torch.einsum("hgn,nhd->hgd", torch.softmax(score, -1), values[span]).reshape(hq, d)
    return out


def _exact_adapters(case, s):
    out = s["base"].double()
    for adapter in s["ids"].unique().tolist():
        if adapter >= 0:
            rows = (s["ids"] == adapter).nonzero().squeeze(1)
            low = s["x"][rows].double() @ s["a"][adapter].double().t()
            out[rows] += float(s["scales"][adapter]) * (low @ s["b"][adapter].double().t())
    return out


def exact(case, seed):
    """From the definitions, token by token and adapter by adapter. FP8 entries are given unrounded, as their codes."""
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "adapters": _exact_adapters}[case["kind"]](case, s)
