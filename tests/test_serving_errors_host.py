"""What the refusals of the paged cache and of adapters say, and calls of a single row. Nothing here needs a GPU."""

import pytest
import torch

from dlmrt_b200 import _lib
from dlmrt_b200.ops.paged_kv import PagedKV
from test_paged_kv_host import adapters, append, attend

BF16 = torch.bfloat16


def test_texts_name_no_other_operator():
    """One text for each code: it does not speak of a fused GEMM to a caller of attention."""
    for code in (_lib.ERR_SHAPE, _lib.ERR_ALIGN, _lib.ERR_OVERLAP, _lib.ERR_NULL, _lib.ERR_WORKSPACE, _lib.ERR_INDEX):
        assert b"GEMM" not in _lib.lib().dlm_strerror(code)
    assert _lib.lib().dlm_strerror(_lib.ERR_SHAPE).startswith(b"a size that this entry point does not take")


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused would run on addresses that are not")
def test_the_distance_of_a_single_row_to_the_next_is_nobodys_business():
    call = lambda **kw: _lib.lib().dlm_adapters_bf16(adapters(**kw), None)
    odd = dict(ldx=61, ldb=-3, ldo=1)
    assert call(m=1, **odd) != _lib.ERR_ALIGN
    assert all(call(m=2, **{name: value}) == _lib.ERR_ALIGN for name, value in odd.items())


def test_the_status_of_another_device_is_read_on_that_device(monkeypatch):
    """A default stream's handle is 0 on every device: what it means is the current device's."""
    kv = PagedKV(torch.zeros(2, 1, 16, 64, dtype=BF16), torch.zeros(2, 1, 16, 64, dtype=BF16))
    current, read = [0], []

    class Current:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Status:
        device = torch.device("cuda:1")
        get_device = staticmethod(lambda: 1)
        data_ptr = staticmethod(lambda: 0x1000)

    class Library:
        @staticmethod
        def dlm_status_read(address, out, stream):
            read.append((address, stream, current[0]))
            return _lib.OK

    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(_lib, "lib", lambda: Library)
    kv.status = Status()
    kv.check()
    assert read == [(0x1000, 0, 1)] and current == [0]


def test_a_rotation_needs_positions():
    kv = PagedKV(torch.zeros(2, 1, 16, 64, dtype=BF16), torch.zeros(2, 1, 16, 64, dtype=BF16))
    k, slots = torch.zeros(3, 1, 64, dtype=BF16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="positions"):
        kv.append(k, k, None, slots, torch.zeros(5, 64))
