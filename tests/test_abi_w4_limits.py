"""Sizes next to 32 bits are refused, and refused calls are not counted (CPU only)."""
import ctypes

import pytest

F32, BF16, SHAPE = 0, 2, 2


@pytest.fixture()
def lib(qm):
    from quadmul_b200 import _lib

    return _lib.LIB


@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(256)
    p.keep = buf
    return (ctypes.addressof(buf) + 15) & ~15


def test_sizes_next_to_32_bits(lib, p):
    """Sizes that an int holds, but not together with the tile or the turn that a kernel adds to them, are refused."""
    top, wide = 2**31 - 1, 2**31
    for rows in (top, top - 511):
        assert lib.qm_gemm_w4(p, BF16, 32, p, p, BF16, 32, p, 8, rows, 8, 32, None, 0, None) == SHAPE
        assert lib.qm_moe_gemm_w4(p, BF16, 32, p, p, BF16, 32, p, 2, p, 8, rows, 8, 32, None, 0, None) == SHAPE
    for hidden in (top, top - 4095):
        assert lib.qm_moe_sort(p, BF16, wide, p, 8, 4, p, wide, p, p, 2, 2, hidden, None, 0, None) == SHAPE
        assert lib.qm_moe_combine(p, BF16, wide, 4, p, p, F32, p, wide, 2, 2, hidden, None) == SHAPE
        assert lib.qm_moe_combine_grad(p, wide, p, wide, BF16, 4, p, p, F32, p, wide, p, 2, 2, hidden, None) == SHAPE
    # blocks of 8192 tokens, each with a count per expert, and the totals
    assert lib.qm_moe_sort_workspace_bytes(top, 1, 4) == (2**18 + 1) * 4 * 4


@pytest.mark.parametrize("binding", ["compiled", "ctypes"])
def test_refused_calls_are_not_counted(qm, monkeypatch, binding):
    import torch

    import quadmul_b200.moe
    import quadmul_b200.w4

    if binding == "ctypes":
        monkeypatch.setattr(quadmul_b200.w4, "_EXT", None)
        monkeypatch.setattr(quadmul_b200.moe, "_EXT", None)
    elif quadmul_b200.w4._EXT is None:
        pytest.skip("the compiled binding is not built")
    x, b, s = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8, 1, dtype=torch.bfloat16)
    ids, slots = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2, dtype=torch.int32)
    before = qm.launch_count()
    for call in (lambda: qm.gemm_w4(x, b, s), lambda: qm.moe_gemm_w4(x, b[None], s[None], torch.zeros(2, dtype=torch.int32)), lambda: qm.quantize_w4(x),
                 lambda: qm.moe_sort(x, ids, 4), lambda: qm.moe_combine(x, slots), lambda: qm.moe_combine_grad(x, x, slots, torch.zeros(4, 2))):
        with pytest.raises(ValueError):
            call()
    assert qm.launch_count() == before
