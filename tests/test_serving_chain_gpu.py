"""A layer's attention half as a program runs it: qkv projection with adapters, append, attention over the pages, o_proj with
adapters into the reduction with residual and norm. Each stage is held to 64 bits on what the stage before it gave; the
whole in a graph, and in the device loop, gives the bits of the calls made one by one."""

import pytest
import torch

import serving_util as su
from dlmrt_b200.distributed.parallel import Group
from dlmrt_b200.layers.adapters import Adapters
from dlmrt_b200.layers.linear import Linear
from dlmrt_b200.ops.block_graph import BlockGraph
from dlmrt_b200.ops.paged_kv import PagedKV, rotary_table

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HIDDEN, HQ, HK, D, PAGE, EPS = 512, 8, 2, 64, 16, 1e-6


class Layer:
    def __init__(self, seed, rows, cache=BF16):
        g = torch.Generator().manual_seed(seed)

        def randn(*shape, std=1.0, mean=0.0):
            return (torch.randn(*shape, generator=g) * std + mean).to(BF16).cuda()

        def adapters(n, k):
            return Adapters(randn(3, 16, k, std=k ** -0.5), randn(3, n, 16, std=0.25), torch.tensor([0.5, 1.0, 2.0]).cuda())

        self.group = Group.local("cuda:0")
        n = (HQ + 2 * HK) * D
        self.qkv = Linear(randn(n, HIDDEN, std=HIDDEN ** -0.5), adapters=adapters(n, HIDDEN))
        self.o = Linear(randn(HIDDEN, HQ * D, std=(HQ * D) ** -0.5), group=self.group, adapters=adapters(HIDDEN, HQ * D))
        self.norm, self.q_norm, self.k_norm = randn(HIDDEN, std=0.1, mean=1), randn(D, std=0.1, mean=1), randn(D, std=0.1, mean=1)
        self.kv = PagedKV(*su.pool(80, HK, PAGE, D, cache, seed, device="cuda"))
        self.table = rotary_table(D, 1024, 1e6, "cuda")
        self.rows = rows

    def step(self, x, h, ids, batch, positions, slots, pages, lengths, site="o", causal=False):
        qkv = self.qkv(x, ids=ids)
        q, k, v = (t.view(self.rows, -1, D) for t in qkv.split((HQ * D, HK * D, HK * D), 1))
        q = self.kv.append(k, v, positions, slots, self.table, q=q, q_norm=self.q_norm, k_norm=self.k_norm, eps=EPS)
        a = self.kv.attend(q.view(batch, -1, HQ, D), pages, lengths, causal=causal)
        p = self.o(a.view(self.rows, HQ * D), out=self.group.partial("o", (self.rows, HIDDEN)), ids=ids)
        return qkv, q, a, p.clone(), self.group.reduce_norm(p, h, self.norm, EPS, site=site)


def batch_of(lengths, tokens):
    """What a scheduler hands over for `tokens` new tokens of sequences that have `lengths` keys with them."""
    table = su.page_table(lengths, PAGE, 80, 3)
    positions = torch.tensor([n - tokens + i for n in lengths for i in range(tokens)])
    which = torch.tensor([b for b in range(len(lengths)) for _ in range(tokens)])
    slots = table[which, positions // PAGE].long() * PAGE + positions % PAGE
    return positions.int().cuda(), slots.cuda(), table.cuda(), torch.tensor(lengths).int().cuda()


def linear64(x, weight):
    """(x W^T, bound): FP32 sums in any split of K, one rounding."""
    want = x.cpu().double() @ weight.cpu().double().t()
    size = x.cpu().double().abs() @ weight.cpu().double().abs().t()
    return want, 2 * x.shape[1] * su.U * size + su.HALF[BF16] * (want.abs() + 2 * x.shape[1] * su.U * size)


@pytest.mark.parametrize("cache", [BF16, torch.float8_e4m3fn])
@pytest.mark.parametrize("lengths, tokens, causal", [([1, 17, 33, 40, 64, 100, 5, 16, 2, 3, 90, 31, 32, 80, 7, 9], 1, False),
                                                     ([40, 96], 16, False), ([16, 50, 130], 16, True)])
def test_every_stage_and_the_whole(lengths, tokens, causal, cache):
    rows = len(lengths) * tokens
    g = torch.Generator().manual_seed(1)
    x, h = (torch.randn(rows, HIDDEN, generator=g).to(BF16).cuda() for _ in range(2))
    ids = torch.randint(-1, 3, (rows,), generator=g).int().cuda()
    positions, slots, pages, lens = batch_of(lengths, tokens)
    layer = Layer(0, rows, cache)
    h0, before = h.clone(), h.clone()
    qkv, q, a, partial, out = layer.step(x, h0, ids, len(lengths), positions, slots, pages, lens, causal=causal)
    out = out.clone()
    layer.kv.check()
    layer.qkv.adapters.check()
    # qkv: the projection's rounding, then the adapters' on top of it
    base, base_bound = linear64(x, layer.qkv.weight)
    ad = layer.qkv.adapters
    want, bound = su.adapters(x, ids, base, ad.a, ad.b, ad.scales)
    su.assert_within(qkv, want, bound + base_bound * (1 + 2.0 ** -7), "qkv")
    # append, on the qkv that was computed
    parts = [t.view(rows, -1, D) for t in qkv.split((HQ * D, HK * D, HK * D), 1)]
    su.assert_within(q, *su.stored(*su.turned(parts[0], layer.q_norm, layer.table, positions, EPS, False), BF16), "q")
    page, at = slots.cpu() // PAGE, slots.cpu() % PAGE
    want, bound = su.stored(*su.turned(parts[1], layer.k_norm, layer.table, positions, EPS, False), cache, layer.kv.k_scale)
    su.assert_within(layer.kv.keys.cpu().double()[page, :, at], want, bound, "keys")
    # attention, on the pages as they are
    want, bound, _ = su.attend(q.view(len(lengths), tokens, HQ, D), layer.kv.keys, layer.kv.values, layer.kv.k_scale,
                               layer.kv.v_scale, pages, lengths, D ** -0.5, 0, causal)
    su.assert_within(a, want, bound, "attention")
    # o_proj with adapters, not deferred
    base, base_bound = linear64(a.view(rows, -1), layer.o.weight)
    ad = layer.o.adapters
    want, bound = su.adapters(a.view(rows, -1), ids, base, ad.a, ad.b, ad.scales)
    su.assert_within(partial, want, bound + base_bound * (1 + 2.0 ** -7), "partial")
    # residual: exactly one BF16 addition
    assert torch.equal(h0, (partial.float() + before.float()).to(BF16))

    # the same in a graph
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    h1 = before.clone()
    with torch.cuda.stream(stream):
        layer.step(x, h1, ids, len(lengths), positions, slots, pages, lens, site="warm", causal=causal)
        layer.group.reduce(partial, site="between")
        h1.copy_(before)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = layer.step(x, h1, ids, len(lengths), positions, slots, pages, lens, site="graph", causal=causal)
    torch.cuda.current_stream().wait_stream(stream)
    graph.replay()
    for name, mine, want in zip(("qkv", "q", "a", "partial", "out"), got, (qkv, q, a, partial, out)):
        assert torch.equal(mine, want), name
    assert torch.equal(h1, h0)
    layer.group.check()
    layer.kv.check()


def test_decoding_in_the_device_loop():
    """Tokens decoded one after the other by the conditional WHILE node, the lengths, positions and slots advancing on the
    device, equal the same steps launched from the host."""
    lengths, rows, steps = [1, 30, 47, 64] * 4, 16, 5
    g = torch.Generator().manual_seed(1)
    x = torch.randn(rows, HIDDEN, generator=g).to(BF16).cuda()
    ids = torch.randint(-1, 3, (rows,), generator=g).int().cuda()
    room = [n + steps for n in lengths]
    table = su.page_table(room, PAGE, 120, 3).cuda()

    def program(layer):
        h = x.clone()
        now, positions, slots = (torch.zeros(rows, device="cuda", dtype=t) for t in (torch.int32, torch.int32, torch.int64))
        remaining, step = (torch.zeros(1, device="cuda", dtype=torch.int32) for _ in range(2))
        first = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        which = torch.arange(rows, device="cuda")
        normed = x.clone()

        def begin():
            now.copy_(first)
            h.copy_(x)
            normed.copy_(x)
            remaining.fill_(steps)
            step.zero_()

        def round_():
            positions.copy_(now - 1)
            slots.copy_(table[which, positions.long() // PAGE].long() * PAGE + positions % PAGE)
            # two call sites: a site may not run twice in a row
            out = layer.step(normed, h, ids, rows, positions, slots, table, now, site="a")[-1]
            out = layer.step(out, h, ids, rows, positions, slots, table, now, site="b")[-1]
            normed.copy_(out)
            now.add_(1)
            remaining.sub_(1)
            step.add_(1)

        return begin, round_, remaining, step, (h, normed, now, layer.kv.keys, layer.kv.values)

    def layer():
        made = Layer(0, rows)
        made.kv = PagedKV(*su.pool(120, HK, PAGE, D, BF16, 5, device="cuda"))
        return made

    begin, round_, *_, want = program(layer())
    begin()
    for _ in range(steps):
        round_()
    made = layer()
    begin, round_, remaining, step, got = program(made)
    keys = made.kv.keys.clone(), made.kv.values.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        for fn in (begin, round_, lambda: step.add_(0)):
            fn()
            graphs.append(torch.cuda.CUDAGraph(keep_graph=True))
            with torch.cuda.graph(graphs[-1], stream=stream):
                fn()
        made.kv.keys.copy_(keys[0])
        made.kv.values.copy_(keys[1])
    torch.cuda.current_stream().wait_stream(stream)
    loop = BlockGraph(*(graph.raw_cuda_graph() for graph in graphs), remaining.data_ptr(), step.data_ptr(), steps)
    loop.replay(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert int(step) == steps
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    made.kv.check()
    made.group.check()


def test_ids_drop_a_projection_that_was_put_off():
    """A partial for which a deferred GEMM is on record and that a call with ids then writes: the later call counts."""
    layer = Layer(0, 16)
    a = torch.randn(16, HQ * D, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    ids = torch.zeros(16, device="cuda", dtype=torch.int32)
    p = layer.group.partial("o", (16, HIDDEN))
    layer.o(a * 3, out=p)
    want = layer.o(a, ids=ids)
    layer.o(a, out=p, ids=ids)
    assert torch.equal(layer.group.reduce(p, site="x"), want)
