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
