"""Products whose inputs the kernel before them has just written, launched one behind the other."""
import pytest
import torch

from _w4 import codes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 6, 40, 300])
@pytest.mark.parametrize("widths", [(512, 768, 640, 512), (512, 766, 642, 512)])  # the second: copies in front of the products
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_each_product_reads_the_one_before(qm, cuda_clean, m, widths, dtype):
    gen = torch.Generator().manual_seed(m)
    layers = []
    for k, n in zip(widths, widths[1:]):
        packed = codes((n, k), gen)[1].cuda()
        layers.append((packed, (0.2 * torch.rand(n, -(-k // 64), generator=gen) / k**0.5).to(dtype).cuda()))
    x = torch.randn(m, widths[0], generator=gen).to(dtype).cuda()
    held = [torch.empty(m, n, dtype=dtype, device="cuda") for n in widths[1:]]

    def chain(waits):
        y = x
        for (b, s), out in zip(layers, held):
            y = qm.gemm_w4(y, b, s, 64, out=out)
            if waits:
                torch.cuda.synchronize()
        return y.clone()

    want = chain(True)
    assert bool(torch.isfinite(want).all()) and bool((want != 0).any())
    for _ in range(20):
        for t in held:
            t.fill_(float("nan"))  # what is read too early shows
        got = [chain(False) for _ in range(3)]
        for y in got:
            assert torch.equal(y, want)


def test_offsets_of_the_sort_before(qm, cuda_clean):
    tokens, top_k, experts, k, n = 48, 4, 6, 256, 136
    gen = torch.Generator().manual_seed(2)
    b, s = codes((experts, n, k), gen)[1].cuda(), (0.01 * torch.rand(experts, n, k // 64, generator=gen)).bfloat16().cuda()
    x = torch.randn(tokens, k, generator=gen).bfloat16().cuda()
    ids = [torch.randint(-1, experts, (tokens, top_k), generator=gen).cuda() for _ in range(4)]
    w = torch.rand(tokens, top_k, generator=gen).cuda()

    def each(waits):
        out = []
        for i in ids:
            out.append(qm.moe_linear_w4(x, i, w, b, s, 64))
            if waits:
                torch.cuda.synchronize()
        return out

    want = each(True)
    for _ in range(20):
        assert all(torch.equal(a, c) for a, c in zip(each(False), want))
