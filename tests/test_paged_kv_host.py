"""What the paged cache and the adapters refuse, on the host: nothing here needs a GPU."""

import ctypes as C

import pytest
import torch

from dlmrt_b200 import _lib
from dlmrt_b200._lib import DlmAdapters, DlmAppend, DlmAttend, DlmPages
from dlmrt_b200.layers.adapters import Adapters
from dlmrt_b200.layers.linear import Linear
from dlmrt_b200.ops.paged_kv import PagedKV, rotary_table

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def pages(**kw):
    p = DlmPages()
    p.keys, p.values, p.pages, p.page_size, p.heads, p.head_dim, p.type = 0x1000, 0x2000, 4, 16, 2, 64, _lib.BF16
    p.k_strides[:] = p.v_strides[:] = (2048, 1024, 64)
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


PAGES = [
    (dict(keys=None), _lib.ERR_NULL), (dict(values=None), _lib.ERR_NULL), (dict(type=3), _lib.ERR_SHAPE),
    (dict(type=_lib.E4M3), _lib.ERR_NULL), (dict(head_dim=96), _lib.ERR_SHAPE), (dict(page_size=24), _lib.ERR_SHAPE),
    (dict(page_size=8192), _lib.ERR_SHAPE), (dict(page_size=0), _lib.ERR_SHAPE), (dict(page_size=4), _lib.ERR_SHAPE), (dict(pages=0), _lib.ERR_SHAPE),
    (dict(heads=0), _lib.ERR_SHAPE), (dict(k_strides=(2048, 1024, 68)), _lib.ERR_ALIGN), (dict(v_strides=(-8, 8, 8)), _lib.ERR_ALIGN),
    (dict(keys=0x1008), _lib.ERR_ALIGN),
    (dict(type=_lib.E4M3, k_scale=0x10, v_scale=0x10, k_strides=(2048, 1024, 72)), _lib.ERR_ALIGN),
]


def append(cache=None, **kw):
    a = DlmAppend()
    a.cache = cache or pages()
    a.k, a.v, a.slots, a.n, a.eps = 0x3000, 0x4000, 0x5000, 3, 1e-6
    a.k_strides[:] = a.v_strides[:] = a.q_strides[:] = a.out_strides[:] = (128, 64)
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


def attend(cache=None, **kw):
    a = DlmAttend()
    a.cache = cache or pages()
    a.q, a.out, a.page_table, a.lengths = 0x3000, 0x4000, 0x5000, 0x6000
    a.batch, a.tokens, a.q_heads, a.table_pages, a.table_stride, a.scale = 2, 1, 4, 8, 8, 0.125
    a.q_strides[:] = a.out_strides[:] = (256, 256, 64)
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, code", PAGES)
def test_pages_are_checked_by_both_entry_points(kw, code):
    assert _lib.lib().dlm_paged_append(append(pages(**kw)), None) == code
    assert _lib.lib().dlm_paged_attend(attend(pages(**kw)), None) == code


@pytest.mark.parametrize("kw, code", [
    (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL), (dict(slots=None), _lib.ERR_NULL),
    (dict(q=0x7000, q_heads=2), _lib.ERR_NULL), (dict(q=0x7000, q_out=0x8000, q_heads=0), _lib.ERR_SHAPE),
    (dict(rotated=32), _lib.ERR_NULL), (dict(rotated=32, positions=0x10, table=0x20, table_rows=0), _lib.ERR_SHAPE),
    (dict(rotated=24, positions=0x10, table=0x20, table_rows=4), _lib.ERR_SHAPE),
    (dict(rotated=80, positions=0x10, table=0x20, table_rows=4), _lib.ERR_SHAPE), (dict(type=_lib.E4M3), _lib.ERR_SHAPE),
    (dict(type=_lib.F16), _lib.ERR_SHAPE), (dict(n=-1), _lib.ERR_SHAPE), (dict(interleaved=2), _lib.ERR_SHAPE),
    (dict(k=0x3008), _lib.ERR_ALIGN), (dict(k_strides=(128, 60)), _lib.ERR_ALIGN), (dict(k_norm=0x18), _lib.ERR_ALIGN),
    (dict(n=0, k=None), _lib.OK),
])
def test_append_refuses(kw, code):
    assert _lib.lib().dlm_paged_append(append(**kw), None) == code


@pytest.mark.parametrize("kw, code", [
    (dict(q=None), _lib.ERR_NULL), (dict(out=None), _lib.ERR_NULL), (dict(lengths=None), _lib.ERR_NULL),
    (dict(page_table=None), _lib.ERR_NULL), (dict(q_heads=3), _lib.ERR_SHAPE), (dict(q_heads=0), _lib.ERR_SHAPE),
    (dict(tokens=0), _lib.ERR_SHAPE), (dict(batch=-1), _lib.ERR_SHAPE), (dict(batch=65536), _lib.ERR_SHAPE),
    (dict(table_pages=1 << 27), _lib.ERR_SHAPE), (dict(window=-1), _lib.ERR_SHAPE), (dict(causal=2), _lib.ERR_SHAPE),
    (dict(type=_lib.F16), _lib.ERR_SHAPE), (dict(q=0x3004), _lib.ERR_ALIGN), (dict(q_strides=(256, 256, 68)), _lib.ERR_ALIGN),
    (dict(cache=pages(heads=1024), q_heads=1024, batch=65535, table_pages=1 << 20), _lib.ERR_SHAPE),  # more than 2^31 units of work
    (dict(tokens=1 << 17), _lib.ERR_SHAPE),
    (dict(out_strides=(256, 256, -64)), _lib.ERR_ALIGN), (dict(q_strides=(-3, 256, 64)), _lib.ERR_ALIGN), (dict(batch=0, q=None), _lib.OK),
])
def test_attend_refuses(kw, code):
    assert _lib.lib().dlm_paged_attend(attend(**kw), None) == code


@pytest.mark.parametrize("q, q_strides, out, out_strides, batch, tokens, refused", [
    (0x3000, (256, 256, 64), 0x3000, (256, 256, 64), 2, 1, False),                 # in place
    (0x3000, (256, 256, 64), 0x3100, (256, 256, 64), 2, 1, True),                  # shifted by two heads
    (0x3000, (256, 256, 64), 0x3000, (512, 256, 64), 2, 1, True),                  # the same beginning, other rows
    (0x3000, (512, 256, 64), 0x3200, (512, 256, 64), 4, 1, False),                 # halves of the same longer rows
    (0x3200, (512, 256, 64), 0x3000, (512, 256, 64), 4, 1, False),
    (0x3000, (512, 256, 64), 0x3180, (512, 256, 64), 4, 1, True),                  # halves that meet
    (0x3000, (2048, 512, 64), 0x3200, (2048, 512, 64), 2, 4, False),
    (0x3000, (2048, 512, 64), 0x3200, (2048, 256, 64), 2, 4, True),                # steps differ: cannot be told
    (0x3000, (64, 128, 256), 0x3000, (64, 128, 256), 2, 2, False),                 # heads outermost, in place
])
def test_attend_results_overlap_no_queries_but_their_own(q, q_strides, out, out_strides, batch, tokens, refused):
    call = attend(q=q, q_strides=q_strides, out=out, out_strides=out_strides, batch=batch, tokens=tokens, cache=pages(heads=4))
    code = _lib.lib().dlm_paged_attend(call, None) if refused or not torch.cuda.is_available() else _lib.OK  # never on addresses that are not
    assert (code == _lib.ERR_OVERLAP) == refused


def test_append_results_overlap_no_input_but_their_own():
    code = lambda **kw: _lib.lib().dlm_paged_append(append(q=0x7000, q_heads=4, **kw), None)
    rows = dict(n=3, q_strides=(512, 64), out_strides=(512, 64), k_strides=(512, 64), v_strides=(512, 64))
    assert code(**rows, q_out=0x7040) == _lib.ERR_OVERLAP and code(**rows, q_out=0x6FF0) == _lib.ERR_OVERLAP
    assert code(**rows, q_out=0x7000, k=0x7100, v=0x7300) == _lib.ERR_OVERLAP  # k inside the row of q that is written
    if not torch.cuda.is_available():
        assert code(**rows, q_out=0x7000, k=0x7200, v=0x7300) != _lib.ERR_OVERLAP  # slices of one projection, in place
        assert code(**rows, q_out=0x9000) != _lib.ERR_OVERLAP


def test_attend_workspace_grows_with_what_is_split():
    size = lambda **kw: _lib.lib().dlm_paged_attend_workspace_bytes(attend(**kw))
    assert size(table_pages=1) == 0
    assert size(table_pages=4096) > 0 and size(table_pages=4096, batch=4) >= size(table_pages=4096)
    assert size(table_pages=4096, window=64) < size(table_pages=4096)
    assert size(tokens=0) == 0


def adapters(**kw):
    a = DlmAdapters()
    a.x, a.base, a.out, a.a, a.b, a.scales, a.ids = 0x100000, 0x200000, 0x300000, 0x4000, 0x5000, 0x6000, 0x7000
    a.ldx, a.ldb, a.ldo, a.m, a.n, a.k, a.rank, a.count = 64, 64, 64, 4, 64, 64, 16, 2
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, code", [
    (dict(x=None), _lib.ERR_NULL), (dict(ids=None), _lib.ERR_NULL), (dict(scales=None), _lib.ERR_NULL), (dict(m=257), _lib.ERR_SHAPE),
    (dict(m=-1), _lib.ERR_SHAPE), (dict(n=60), _lib.ERR_SHAPE), (dict(k=4), _lib.ERR_SHAPE), (dict(rank=12), _lib.ERR_SHAPE),
    (dict(rank=136), _lib.ERR_SHAPE), (dict(count=0), _lib.ERR_SHAPE), (dict(x=0x100008), _lib.ERR_ALIGN), (dict(ldo=56), _lib.ERR_ALIGN),
    (dict(ldb=60), _lib.ERR_ALIGN), (dict(m=0, x=None), _lib.OK),
])
def test_adapters_refuse(kw, code):
    assert _lib.lib().dlm_adapters_bf16(adapters(**kw), None) == code


def test_adapters_results_overlap_no_input_but_base():
    code = lambda **kw: _lib.lib().dlm_adapters_bf16(adapters(**kw), None)
    assert code(out=0x100000) == _lib.ERR_OVERLAP and code(out=0x200010) == _lib.ERR_OVERLAP
    assert code(out=0x200000, ldo=128) == _lib.ERR_OVERLAP and code(out=0x200000, ldb=0) == _lib.ERR_OVERLAP
    if not torch.cuda.is_available():
        assert code(out=0x200000) != _lib.ERR_OVERLAP and code(x=0x100000, out=0x100080, ldx=128, ldo=128) != _lib.ERR_OVERLAP


def test_windows_longer_than_any_cache():
    assert _lib.lib().dlm_paged_attend(attend(window=(1 << 30) + 1), None) == _lib.ERR_SHAPE
    keys = torch.zeros(2, 2, 16, 64, dtype=BF16)
    plan = PagedKV(keys, keys.clone())._plan_attend(torch.zeros(1, 2, 64, dtype=BF16), torch.zeros(1, 2, dtype=torch.int32),
                                                    torch.zeros(1, dtype=torch.int32), None, None, None, 1 << 33, False)
    assert plan.window == 1 << 30


def test_struct_layouts_match():
    sizes = [C.sizeof(s) for s in (DlmAppend, DlmAttend, DlmAdapters)]
    assert _lib.lib().dlm_abi_check_serving(*sizes) == _lib.OK
    assert _lib.lib().dlm_abi_check_serving(sizes[0] + 8, *sizes[1:]) == _lib.ERR_SHAPE
    assert b"outside" in _lib.lib().dlm_strerror(_lib.ERR_INDEX)


def cache(dtype=BF16, shape=(4, 2, 16, 64), **kw):
    return PagedKV(torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype), **kw)


@pytest.mark.parametrize("make", [
    lambda: PagedKV(torch.zeros(4, 2, 16, 64, dtype=BF16), torch.zeros(4, 2, 16, 64, dtype=F16)),
    lambda: PagedKV(torch.zeros(4, 2, 16, 64, dtype=BF16), torch.zeros(4, 2, 8, 64, dtype=BF16)),
    lambda: cache(shape=(2, 16, 64)), lambda: cache(torch.float32), lambda: cache(shape=(4, 2, 16, 80)),
    lambda: cache(shape=(4, 2, 12, 64)), lambda: cache(E4M3), lambda: cache(k_scale=torch.ones(2), v_scale=torch.ones(2)),
    lambda: cache(E4M3, k_scale=torch.ones(3), v_scale=torch.ones(2)),
    lambda: cache(E4M3, k_scale=torch.ones(2).half(), v_scale=torch.ones(2)),
    lambda: PagedKV(*[torch.zeros(4, 2, 64, 16, dtype=BF16).transpose(2, 3) for _ in range(2)]),
])
def test_caches_that_cannot_be(make):
    with pytest.raises(ValueError):
        make()


def test_calls_that_cannot_be():
    kv = cache()
    k = torch.zeros(3, 2, 64, dtype=BF16)
    q = torch.zeros(3, 4, 64, dtype=BF16)
    slots, positions, table = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(5, 64)
    for args, kw in [((k.half(), k.half(), positions, slots), {}), ((k[:, :1], k, positions, slots), {}),
                     ((k, k[:2], positions, slots), {}), ((k, k, positions, slots.int()), {}),
                     ((k, k, positions.long(), slots, table), {}), ((k, k, positions, slots, table.half()), {}),
                     ((k, k, positions, slots, table.t()), {}), ((k, k, positions, slots, table[0]), {}),
                     ((k, k, positions, slots), dict(q=q[:2])), ((k, k, positions, slots), dict(q=q[0])),
                     ((k, k, positions, slots), dict(q=q, q_out=q[:, :2])), ((k, k, positions, slots), dict(q_out=q)),
                     ((k, k, positions, slots), dict(q=q, q_norm=torch.ones(32, dtype=BF16))),
                     ((k, k, positions, slots), dict(k_norm=torch.ones(64))),
                     ((k, k, positions, slots), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)))]:
        with pytest.raises(ValueError):
            kv.append(*args, **kw)
    q, pages_, lengths = torch.zeros(2, 1, 4, 64, dtype=BF16), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args, kw in [((q.half(), pages_, lengths), {}), ((q[:, :, :3], pages_, lengths), {}), ((q[..., :32], pages_, lengths), {}),
                     ((q, pages_.long(), lengths), {}), ((q, pages_[:1], lengths), {}), ((q, pages_, lengths[:1]), {}),
                     ((q, pages_, lengths.long()), {}), ((q, pages_, lengths), dict(out=q.half())), ((q, pages_, lengths), dict(window=-1)),
                     ((q, pages_, lengths), dict(lse=torch.zeros(2, 4))), ((q, torch.zeros(3, 2, dtype=torch.int32).t(), lengths), {})]:
        with pytest.raises(ValueError):
            kv.attend(*args, **kw)


def test_adapters_that_cannot_be():
    a, b, s = torch.zeros(2, 8, 64, dtype=BF16), torch.zeros(2, 128, 8, dtype=BF16), torch.ones(2)
    for args in [(a, b[:1], s), (a[:, :4], b, s), (a[0], b, s), (a.float(), b, s), (a, b, s.half()), (a, b, torch.ones(3)),
                 (a[:, :4].contiguous(), b[..., :4].contiguous(), s), (a[..., :60].contiguous(), b, s), (a[:, :, ::2], b, s)]:
        with pytest.raises(ValueError):
            Adapters(*args)
    layer = Adapters(a, b, s)
    x, base, ids = torch.zeros(3, 64, dtype=BF16), torch.zeros(3, 128, dtype=BF16), torch.zeros(3, dtype=torch.int32)
    for args, kw in [((x[:, :32], ids, base), {}), ((x, ids, base[:2]), {}), ((x, ids.long(), base), {}), ((x, ids[:2], base), {}),
                     ((x.float(), ids, base), {}), ((x, ids, base), dict(out=base[:, :64])), ((x, ids, base.float()), {})]:
        with pytest.raises(ValueError):
            layer(*args, **kw)
    weight = torch.zeros(128, 64, dtype=BF16)
    with pytest.raises(ValueError):
        Linear(weight[:, :32], adapters=layer)
    with pytest.raises(ValueError):
        Linear(weight)(x, ids=ids)


def test_rotary_table_holds_64_bit_angles():
    table = rotary_table(64, 1 << 17, 10000.0, "cpu")
    assert table.shape == (1 << 17, 64) and table.dtype == torch.float32
    import math

    for pos, i in [(0, 0), (131071, 0), (131071, 31), (77777, 7)]:
        angle = pos * 10000.0 ** (-i / 32)
        assert abs(float(table[pos, i]) - math.cos(angle)) <= 2.0 ** -24 + 1e-9
        assert abs(float(table[pos, 32 + i]) - math.sin(angle)) <= 2.0 ** -24 + 1e-9
    given = rotary_table(16, 10, device="cpu", inverse_frequencies=torch.ones(8))
    assert torch.equal(given[3], torch.tensor([math.cos(3)] * 8 + [math.sin(3)] * 8))
    with pytest.raises(ValueError):
        rotary_table(16, 10, device="cpu", inverse_frequencies=torch.ones(4))
