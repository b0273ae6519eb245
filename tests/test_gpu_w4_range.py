"""gemm_w4 and moe_gemm_w4 where the elements of x differ by orders of magnitude and a weight of zero takes the largest out of the sum.

Held against the definition in 64 bits with the tolerance of `close_to`, whose S is the sum over an output's own products: a column
with code 0 on the outlier has to be right on the scale of what is left."""
import pytest
import torch

from _w4 import close_to, codes, dequantised

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def outlier_case(m, n, k, group, dtype, octaves, tiers=(1,), rows=None, seed=0):
    """Normal x times 2^low, with one element per 128 that is 2^octaves times as large (`tiers`: further ones, at shares of the way up), in `rows`.
    The first half of the columns has code 0 on all of these, and nowhere else."""
    gen = torch.Generator().manual_seed(seed + octaves)
    low = -2 if dtype == BF16 else max(-7, min(0, 13 - octaves))
    x = torch.randn(m, k, generator=gen)
    q, _ = codes((n, k), gen)
    q = torch.where(q == 0, 1, q)
    for i, share in enumerate(tiers):
        at = torch.arange(5 + 17 * i, k, 128)
        for r in range(m) if rows is None else rows:
            x[r, at] = 2.0 ** (share * octaves) * (1 + torch.rand(at.numel(), generator=gen))
        q[: n // 2, at] = 0
    packed = ((q[:, 0::2] & 15) | ((q[:, 1::2] & 15) << 4)).to(torch.uint8).view(torch.int8)
    scales = (0.01 * torch.exp(0.5 * torch.randn(n, -(-k // group), generator=gen))).to(dtype)
    x = (x.double() * 2.0**low).to(dtype)
    assert bool(torch.isfinite(x).all())
    return x, q, packed, scales


def check(got, x, q, scales, group):
    w = dequantised(q, scales, group)
    half = q.shape[0] // 2
    close_to(got[:, :half].contiguous(), x, w[:half])
    close_to(got[:, half:].contiguous(), x, w[half:])


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype,octaves", [(BF16, 8), (BF16, 11), (BF16, 12), (BF16, 15), (BF16, 20), (BF16, 30), (FP16, 6), (FP16, 9), (FP16, 12), (FP16, 16), (FP16, 20)])
def test_an_outlier(qm, cuda_clean, m, group, dtype, octaves):
    n, k = 96, 1056
    x, q, packed, scales = outlier_case(m, n, k, group, dtype, octaves)
    check(qm.gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), group), x, q, scales, group)


@pytest.mark.parametrize("m", [1, 7])
@pytest.mark.parametrize("dtype,octaves", [(BF16, 40), (FP16, 18)])
def test_outliers_of_several_sizes(qm, cuda_clean, m, dtype, octaves):
    n, k, group = 128, 2048, 128
    x, q, packed, scales = outlier_case(m, n, k, group, dtype, octaves, tiers=(1, 0.75, 0.5, 0.25))
    check(qm.gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), group), x, q, scales, group)


@pytest.mark.parametrize("m,n,k", [(8, 76000, 640), (6, 20100, 1024), (2, 20011, 2048), (1, 300, 16384)])
def test_some_rows_of_many_blocks(qm, cuda_clean, m, n, k):
    """Every warp goes through several blocks of weights; one row has outliers, the others do not."""
    x, q, packed, scales = outlier_case(m, n, k, 128, BF16, 24, rows=[m - 1])
    got = qm.gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), 128).cpu()
    pick = torch.cat([torch.arange(0, 60), torch.arange(n // 2 - 40, n // 2 + 40), torch.arange(n - 60, n)])
    w = dequantised(q[pick], scales[pick], 128)
    for part in (pick < n // 2, pick >= n // 2):
        close_to(got[:, pick[part]].contiguous(), x, w[part])


@pytest.mark.parametrize("dtype,octaves", [(BF16, 24), (FP16, 16)])
def test_rows_of_experts(qm, cuda_clean, dtype, octaves):
    offsets = [0, 1, 9, 9, 13, 20, 31]
    experts, n, k, group, rows = len(offsets) - 1, 72, 512, 64, offsets[-1]
    x, _, _, _ = outlier_case(rows, n, k, group, dtype, octaves, rows=[0, 4, 8, 12, 30])
    parts = [outlier_case(1, n, k, group, dtype, octaves, seed=e) for e in range(experts)]
    packed, scales = torch.stack([p[2] for p in parts]), torch.stack([p[3] for p in parts])
    got = qm.moe_gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), torch.tensor(offsets, dtype=torch.int32).cuda(), group).cpu()
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if b > a:
            check(got[a:b], x[a:b], parts[e][1], parts[e][3], group)


@pytest.mark.parametrize("m", [1, 8, 9])
def test_tiny_x(qm, cuda_clean, m):
    """bf16 values next to the smallest normal number, with scales that bring the result back: no digit is lost."""
    n, k, group = 64, 512, 64
    gen = torch.Generator().manual_seed(4)
    x = (torch.randn(m, k, generator=gen).clamp(-3, 3).bfloat16().double() * 2.0**-112).to(BF16)
    q, packed = codes((n, k), gen)
    scales = (2.0**95 * torch.rand(n, k // group, generator=gen)).to(FP32)
    close_to(qm.gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), group), x, dequantised(q, scales, group))


@pytest.mark.parametrize("m", [1, 2, 8])
def test_sparse_rows(qm, cuda_clean, m):
    """One element in nine is not zero; half the columns keep the largest of them, the others do not."""
    n, k, group = 96, 1152, 128
    x, q, packed, scales = outlier_case(m, n, k, group, BF16, 22)
    x[:, [i for i in range(k) if i % 9 and i % 128 != 5]] = 0
    check(qm.gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), group), x, q, scales, group)


@pytest.mark.parametrize("m", [1, 8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_equal_calls_give_equal_bits(qm, cuda_clean, m, dtype):
    x, q, packed, scales = outlier_case(m, 512, 4096, 128, dtype, 18)
    args = (x.cuda(), packed.cuda(), scales.cuda(), 128)
    first = qm.gemm_w4(*args)
    for _ in range(10):
        assert torch.equal(first, qm.gemm_w4(*args))


@pytest.mark.parametrize("m", [1, 2, 8])
@pytest.mark.parametrize("every", [2, 3, 4, 8, 16])
@pytest.mark.parametrize("dtype,octaves", [(BF16, 22), (FP16, 17)])
def test_large_elements_at_a_regular_distance(qm, cuda_clean, m, every, dtype, octaves):
    """One element in `every` is large, and half the columns have code 0 on all of these."""
    n, k, group = 96, 1024, 128
    gen = torch.Generator().manual_seed(every)
    x, q = torch.randn(m, k, generator=gen), codes((n, k), gen)[0]
    q = torch.where(q == 0, 1, q)
    x[:, ::every] = 2.0**octaves * (1 + torch.rand(m, x[:, ::every].shape[1], generator=gen))
    q[: n // 2, ::every] = 0
    x = (x.double() * 2.0 ** (-2 if dtype == BF16 else -5)).to(dtype)
    packed = ((q[:, 0::2] & 15) | ((q[:, 1::2] & 15) << 4)).to(torch.uint8).view(torch.int8)
    scales = (0.01 * torch.exp(0.5 * torch.randn(n, k // group, generator=gen))).to(dtype)
    assert bool(torch.isfinite(x).all())
    check(qm.gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), group), x, q, scales, group)
