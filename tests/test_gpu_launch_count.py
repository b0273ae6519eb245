"""launch_count() counts the kernels of the 4-bit-weight and routing calls: copies too, empty calls not."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(params=["compiled", "ctypes"])
def binding(request, monkeypatch):
    import quadmul_b200.moe
    import quadmul_b200.w4

    if request.param == "ctypes":
        monkeypatch.setattr(quadmul_b200.w4, "_EXT", None)
        monkeypatch.setattr(quadmul_b200.moe, "_EXT", None)
    elif quadmul_b200.w4._EXT is None:
        pytest.skip("the compiled binding is not built")


def test_counts(qm, cuda_clean, binding):
    def zeros(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    def product(x, n, group=64):
        k = x.shape[1]
        return lambda: qm.gemm_w4(x, zeros(n, k // 2, dtype=torch.int8), zeros(n, -(-k // group)), group)

    def experts(rows, count, n=8, k=64):
        return lambda: qm.moe_gemm_w4(zeros(rows, k), zeros(count, n, k // 2, dtype=torch.int8), zeros(count, n, -(-k // 64)), zeros(count + 1, dtype=torch.int32), 64)

    slots, ids = zeros(4, 2, dtype=torch.int32), zeros(4, 2, dtype=torch.int64)
    off = zeros(8 * 32 + 1, dtype=torch.int8)[1:].view(8, 32)  # not on a 16-byte boundary
    wide = zeros(4, 72)
    cases = [
        (product(zeros(4, 64), 8), 1), (product(zeros(300, 64), 8), 1), (product(zeros(4, 62), 8), 3), (product(zeros(0, 64), 8), 0), (product(zeros(4, 64), 0), 0),
        (product(zeros(4, 0), 8), 1), (product(wide[:, 2:66], 8), 2), (product(wide[:, 8:72], 8), 1), (product(zeros(4, 68)[:, :64], 8), 2),
        (lambda: qm.gemm_w4(zeros(4, 64), off, zeros(8, 1), 64), 2),
        (experts(4, 2), 1), (experts(4, 0), 0), (experts(0, 2), 0), (experts(4, 2, n=0), 0), (experts(4, 2, k=30), 3), (experts(4, 2, k=0), 1),
        (lambda: qm.quantize_w4(zeros(4, 64)), 1), (lambda: qm.quantize_w4(zeros(0, 64)), 0), (lambda: qm.quantize_w4(zeros(4, 0)), 0),
        (lambda: qm.moe_sort(zeros(4, 8), ids, 3), 1), (lambda: qm.moe_sort(zeros(9000, 8), zeros(9000, 2, dtype=torch.int64), 3), 3),
        (lambda: qm.moe_sort(zeros(9000, 8), zeros(9000, 2, dtype=torch.int64), 0), 1), (lambda: qm.moe_sort(zeros(0, 8), ids[:0], 3), 1),
        (lambda: qm.moe_combine(zeros(8, 8), slots), 1), (lambda: qm.moe_combine(zeros(8, 0), slots), 0), (lambda: qm.moe_combine(zeros(8, 8), slots[:0]), 0),
        (lambda: qm.moe_combine_grad(zeros(4, 8), zeros(8, 8), slots, zeros(4, 2)), 1),
        (lambda: qm.moe_combine_grad(zeros(4, 8), zeros(8, 8), slots[:, :0].contiguous(), zeros(4, 0)), 0),
        (lambda: qm.moe_linear_w4(zeros(4, 64), ids, zeros(4, 2), zeros(3, 8, 32, dtype=torch.int8), zeros(3, 8, 1), 64), 3),
    ]
    for i, (call, want) in enumerate(cases):
        before = qm.launch_count()
        call()
        assert qm.launch_count() - before == want, i
