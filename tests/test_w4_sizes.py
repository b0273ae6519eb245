"""Sizes that the library's 32-bit ints do not hold are refused by the ctypes form too (CPU only: shapes, no tensors of that size)."""
import pytest

BIG = 2**32 + 8  # its low 32 bits are 8


class Shape:
    """What the checks look at: a CUDA tensor's shape and layout, without its memory."""

    is_cuda = True
    requires_grad = False

    def __init__(self, *shape, dtype=None):
        import torch

        self.shape, self.dtype, self.device = torch.Size(shape), dtype or torch.int32, torch.device("cuda", 0)

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return [self.shape[1], 1][i]

    def is_contiguous(self):
        return True

    def numel(self):
        return self.shape.numel()


def test_rows(qm):
    from quadmul_b200.w4 import check_rows

    check_rows("call", x=Shape(2**31 - 1, 8), y=Shape(8, 2**31 - 1))
    for shape in ((BIG, 8), (8, BIG), (2**31, 1), (1, 2**31)):
        with pytest.raises(ValueError, match="call: x is too large"):
            check_rows("call", x=Shape(*shape))


def test_slots(qm):
    from quadmul_b200.moe import _check_slots

    device = Shape(1).device
    _check_slots("call", Shape(2**31 - 1, 1), device)
    _check_slots("call", Shape(2**19 - 1, 4096), device)
    for shape in ((BIG, 1), (2**31, 1), (BIG, 0), (2, 4097), (2**19, 4096), (2**30, 2)):
        with pytest.raises(ValueError):
            _check_slots("call", Shape(*shape), device)


def test_weights_of_a_product(qm):
    import torch

    from quadmul_b200.w4 import _check_weights

    x = Shape(4, 64, dtype=torch.bfloat16)
    assert _check_weights("call", x, Shape(8, 32, dtype=torch.int8), Shape(8, 1, dtype=torch.bfloat16), 64, ())[2:] == (8, 64)
    for lead in ((), (2,), (BIG,)):
        n = 8 if lead == (BIG,) else BIG
        with pytest.raises(ValueError, match="call: b is too large"):
            _check_weights("call", x, Shape(*lead, n, 32, dtype=torch.int8), Shape(*lead, n, 1, dtype=torch.bfloat16), 64, lead)
