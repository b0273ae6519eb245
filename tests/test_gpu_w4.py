"""gemm_w4, moe_gemm_w4 and quantize_w4 against their definitions in 64 bits."""
import pytest
import torch

from _w4 import close_to, codes, dequantised, normal_case, whole_case

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SENTINEL = -77.0

# (m, n, k, group): one token to many, sizes around every tile edge, k below, at and beside whole groups and chunks
SHAPES = [
    (1, 1, 2, 32), (1, 8, 32, 32), (1, 100, 30, 64), (2, 33, 34, 128), (3, 31, 96, 64), (5, 7, 130, 256), (7, 130, 160, 32), (8, 64, 128, 128),
    (9, 129, 256, 128), (15, 16, 4096, 128), (16, 257, 2208, 64), (17, 32, 1056, 32), (31, 100, 64, 256), (32, 256, 512, 64), (33, 1100, 2208, 64),
    (63, 65, 96, 32), (64, 128, 4128, 128), (65, 300, 1024, 256), (100, 40, 6, 32), (127, 127, 1022, 64), (128, 256, 256, 128), (129, 200, 320, 64),
    (255, 257, 512, 32), (256, 256, 384, 128), (257, 520, 64, 64), (300, 130, 4064, 256), (513, 384, 1024, 128), (1, 4096, 4096, 128),
    (4, 1024, 11008, 128), (16, 512, 11008, 64), (600, 72, 94, 128), (8, 300, 8192, 128), (8, 5000, 8192, 256), (3, 300, 8192, 64), (2, 300, 16384, 128),
    (1, 100, 30000, 32), (2, 64, 65536, 128),
]


def run(qm, x, packed, scales, group, **kw):
    return qm.gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), group, **kw)


@pytest.mark.parametrize("m,n,k,group", SHAPES)
@pytest.mark.parametrize("dtype,scale_dtype", [(BF16, BF16), (FP16, FP16), (BF16, FP32), (FP16, FP32)])
def test_exact_inputs_give_the_rounded_definition(qm, cuda_clean, m, n, k, group, dtype, scale_dtype):
    x, q, packed, scales = whole_case(m, n, k, group, dtype, scale_dtype, m * 7 + n + k)
    out = torch.full((m, n), SENTINEL, dtype=dtype, device="cuda")
    got = run(qm, x, packed, scales, group, out=out)
    assert got is out
    want = (x.double() @ dequantised(q, scales, group).T).to(dtype)
    assert torch.equal(got.cpu(), want), f"{int((got.cpu() != want).sum())} of {want.numel()} outputs differ"


@pytest.mark.parametrize("m,n,k,group", [(1, 4096, 4096, 128), (6, 512, 4096, 32), (16, 640, 11008, 64), (40, 300, 2208, 64), (200, 384, 4096, 128),
                                         (700, 512, 2048, 256)])
@pytest.mark.parametrize("dtype,scale_dtype", [(BF16, BF16), (FP16, FP16), (BF16, FP32), (FP16, FP32)])
def test_random_inputs(qm, cuda_clean, m, n, k, group, dtype, scale_dtype):
    x, q, packed, scales = normal_case(m, n, k, group, dtype, scale_dtype, 3)
    close_to(run(qm, x, packed, scales, group), x, dequantised(q, scales, group))


@pytest.mark.parametrize("m", [1, 12, 40, 300])
@pytest.mark.parametrize("pad_x,pad_out,shift", [(8, 8, 0), (2, 1, 1), (16, 3, 8)])
def test_column_slabs(qm, cuda_clean, m, pad_x, pad_out, shift):
    """x and out are slabs of wider tensors, on and off vector boundaries; what lies beside out stays."""
    n, k, group = 200, 320, 64
    x, q, packed, scales = whole_case(m, n, k, group, BF16, BF16, 5)
    wide = torch.zeros(m, k + pad_x + shift, dtype=BF16, device="cuda")
    wide[:, shift : shift + k] = x.cuda()
    out = torch.full((m, n + pad_out + shift), SENTINEL, dtype=BF16, device="cuda")
    qm.gemm_w4(wide[:, shift : shift + k], packed.cuda(), scales.cuda(), group, out=out[:, shift : shift + n])
    want = torch.full((m, n + pad_out + shift), SENTINEL, dtype=BF16)
    want[:, shift : shift + n] = (x.double() @ dequantised(q, scales, group).T).to(BF16)
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("m,n,k", [(0, 16, 64), (4, 0, 64), (4, 16, 0), (300, 16, 0)])
def test_empty_sizes(qm, cuda_clean, m, n, k):
    out = torch.full((m, n), SENTINEL, dtype=BF16, device="cuda")
    x, b = torch.zeros(m, k, dtype=BF16, device="cuda"), torch.zeros(n, k // 2, dtype=torch.int8, device="cuda")
    qm.gemm_w4(x, b, torch.zeros(n, (k + 127) // 128, dtype=BF16, device="cuda"), out=out)
    assert bool((out == 0).all())


@pytest.mark.parametrize("m", [3, 20, 200])
def test_values_that_are_not_finite_stay_in_their_row(qm, cuda_clean, m):
    n, k, group = 96, 256, 64
    x, q, packed, scales = whole_case(m, n, k, group, FP16, FP16, 6)
    x[1, 5], x[2, 9] = float("nan"), float("inf")
    got = run(qm, x, packed, scales, group).cpu()
    want = x.double() @ dequantised(q, scales, group).T
    assert bool(torch.isnan(got[1]).all())
    hit = q[:, 9] != 0  # infinity times a code of zero is no number
    assert bool(torch.isinf(got[2][hit]).all()) and bool((torch.sign(got[2][hit]) == torch.sign(q[:, 9][hit])).all()) and bool(torch.isnan(got[2][~hit]).all())
    rest = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(got[rest], want[rest].to(FP16))


@pytest.mark.parametrize("m,group", [(2, 32), (6, 128), (20, 64), (200, 128)])
@pytest.mark.parametrize("dtype,scale_dtype", [(BF16, BF16), (FP16, FP32)])
def test_scales_that_are_not_finite_stay_in_their_column(qm, cuda_clean, m, group, dtype, scale_dtype):
    n, k = 300, 416
    x, q, packed, scales = whole_case(m, n, k, group, dtype, scale_dtype, 7)
    scales[5, 1], scales[130, 0], scales[299, -1] = float("inf"), float("nan"), float("-inf")
    got = run(qm, x, packed, scales, group).cpu()
    odd = torch.zeros(n, dtype=torch.bool)
    odd[[5, 130, 299]] = True
    assert not bool(torch.isfinite(got[:, odd]).any())
    want = (x.double() @ dequantised(q, scales, group).T).to(dtype)
    assert torch.equal(got[:, ~odd], want[:, ~odd])


@pytest.mark.parametrize("m,n,k,group", [(8, 76000, 640, 128), (5, 20100, 1024, 32), (2, 20011, 2048, 64), (1, 9000, 4096, 256)])
def test_many_blocks_of_weights(qm, cuda_clean, m, n, k, group):
    """Few rows and so many of the weights that every warp goes through several blocks of them."""
    x, q, packed, scales = whole_case(m, n, k, group, BF16, BF16, 11)
    want = (x.double() @ dequantised(q, scales, group).T).to(BF16)
    assert torch.equal(run(qm, x, packed, scales, group).cpu(), want)


@pytest.mark.parametrize("m", [2, 20, 200])
@pytest.mark.parametrize("size,x_size", [(2.0**-20, 2.0**13), (2.0**-3, 1.0), (2.0**14, 2.0**-12)])
def test_fp16_with_small_and_large_scales(qm, cuda_clean, m, size, x_size):
    """Scales whose products with the codes fp16 could not hold: the sums are fp32, only x and the result have to fit."""
    n, k, group = 64, 512, 128
    x, q, packed, scales = whole_case(m, n, k, group, FP16, FP32, 8)
    x, scales = x * x_size, scales * size
    got = run(qm, x, packed, scales, group).cpu()
    want = (x.double() @ dequantised(q, scales, group).T).to(FP16)
    assert torch.equal(got, want)


@pytest.mark.parametrize("m", [2, 20, 200])
def test_fp16_scales_of_a_row_that_differ_by_orders(qm, cuda_clean, m):
    n, k, group = 64, 512, 64
    x, q, packed, _ = normal_case(m, n, k, group, FP16, FP32, 9)
    scales = torch.exp2(torch.randint(-24, 4, (n, k // group), generator=torch.Generator().manual_seed(1)).double()).float()
    close_to(run(qm, x, packed, scales, group), x, dequantised(q, scales, group))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_other_stream_and_graph(qm, cuda_clean, m):
    n, k, group = 384, 1024, 128
    x, q, packed, scales = whole_case(m, n, k, group, BF16, BF16, 10)
    want = (x.double() @ dequantised(q, scales, group).T).to(BF16)
    xd, bd, sd = torch.zeros_like(x).cuda(), packed.cuda(), scales.cuda()
    out = torch.zeros(m, n, dtype=BF16, device="cuda")
    qm.init()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qm.gemm_w4(x.cuda(), bd, sd, group, out=out)
    side.synchronize()
    assert torch.equal(out.cpu(), want)
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed one after the other and with other inputs
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = qm.gemm_w4(xd, bd, sd, group)
        graphs.append((g, held))
    xd.copy_(x.cuda())
    for g, held in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, held in graphs:
        assert torch.equal(held.cpu(), want)


def test_two_graphs_replayed_at_once(qm, cuda_clean):
    n, k, group = 512, 4096, 128
    cases = [whole_case(m, n, k, group, BF16, BF16, m) for m in (8, 64)]
    qm.init()
    graphs = []
    for x, q, packed, scales in cases:
        args = (x.cuda(), packed.cuda(), scales.cuda())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = qm.gemm_w4(*args, group)
        graphs.append((g, held, args))
    sides = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for side, (g, _, _) in zip(sides, graphs):
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for (x, q, packed, scales), (_, held, _) in zip(cases, graphs):
        assert torch.equal(held.cpu(), (x.double() @ dequantised(q, scales, group).T).to(BF16))


def test_equal_calls_give_equal_bits(qm, cuda_clean):
    for m in (5, 48, 260):
        x, q, packed, scales = normal_case(m, 512, 4096, 128, BF16, BF16, 12)
        args = (x.cuda(), packed.cuda(), scales.cuda(), 128)
        first = qm.gemm_w4(*args)
        for _ in range(20):
            assert torch.equal(first, qm.gemm_w4(*args))


@pytest.mark.parametrize("m,n,k,group", [(17, 20070, 4096, 128), (64, 40000, 1024, 64), (96, 20070, 4096, 128), (200, 20070, 2048, 32), (500, 19000, 1024, 128)])
@pytest.mark.parametrize("dtype,scale_dtype", [(BF16, BF16), (FP16, FP32)])
def test_many_tiles_of_many_steps(qm, cuda_clean, m, n, k, group, dtype, scale_dtype):
    """Every pair of SMs goes through several tiles, a few dozen steps each, and the rings between its warps wrap at any place."""
    gen = torch.Generator().manual_seed(14)
    x = torch.randint(-1, 2, (m, k), generator=gen).to(dtype)
    q, packed = codes((n, k), gen)
    scales = torch.exp2(torch.randint(-2, 2, (n, k // group), generator=gen).double()).to(scale_dtype)
    w = dequantised(q, scales, group).float()  # exact, as is the product: multiples of 1/4 below 2^19
    want = (x.float() @ w.T).to(dtype)
    args = (x.cuda(), packed.cuda(), scales.cuda(), group)
    for _ in range(5):
        assert torch.equal(qm.gemm_w4(*args).cpu(), want)


def test_many_tiles_of_experts(qm, cuda_clean):
    experts, n, k, group = 24, 2000, 1024, 128
    offsets = torch.cumsum(torch.randint(5, 70, (experts + 1,), generator=torch.Generator().manual_seed(3)), 0).int()
    rows = int(offsets[-1])
    x, q, packed, scales = whole_case(rows, n, k, group, BF16, BF16, 15, (experts,))
    args = (x.cuda(), packed.cuda(), scales.cuda(), offsets.cuda(), group)
    out = torch.full((rows, n), SENTINEL, dtype=BF16)
    want = expert_reference(x, q, scales, group, offsets.tolist(), out)
    for _ in range(5):
        assert torch.equal(qm.moe_gemm_w4(*args, out=out.cuda()).cpu(), want)


@pytest.mark.parametrize("m", [2, 40])
def test_weights_of_more_than_32_bits(qm, cuda_clean, m):
    """The packed matrix has more than 2^32 bytes, the output of the next test more than 2^31 elements."""
    n, k, group = (1 << 20) + 70, 8192 + 32, 128
    b = torch.randint(-128, 128, (n, k // 2), dtype=torch.int8, device="cuda")
    scales = torch.exp2(torch.randint(-2, 2, (n, -(-k // group)), device="cuda").float()).to(BF16)
    x = torch.randint(-1, 2, (m, k), generator=torch.Generator().manual_seed(1)).to(BF16)
    got = qm.gemm_w4(x.cuda(), b, scales, group)
    for first in (0, n // 2, n - 200):
        part = slice(first, first + 200)
        w = dequantised(qm.unpack(b[part].contiguous()).cpu(), scales[part].cpu(), group)
        assert torch.equal(got[:, part].cpu(), (x.double() @ w.T).to(BF16))


def test_output_of_more_than_32_bits(qm, cuda_clean):
    rows, n, k, group = 600_000, 4096, 64, 32
    _, q, packed, scales = whole_case(1, n, k, group, BF16, BF16, 13, (2,))
    x = torch.randint(-3, 4, (rows, k), generator=torch.Generator().manual_seed(2)).to(BF16)
    offsets = torch.tensor([0, 100, rows], dtype=torch.int32, device="cuda")
    got = qm.moe_gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), offsets, group)
    for first, e in ((0, 0), (rows // 2, 1), (rows - 100, 1)):
        part = slice(first, first + 100)
        assert torch.equal(got[part].cpu(), (x[part].double() @ dequantised(q[e], scales[e], group).T).to(BF16))
    weights = torch.ones(rows // 2, 2, dtype=BF16, device="cuda")
    slots = torch.arange(rows, dtype=torch.int32, device="cuda").view(-1, 2)
    y = qm.moe_combine(got, slots, weights)
    assert torch.equal(y[-5:], (got[-10::2].float() + got[-9::2].float()).to(BF16))
    dys, dw = qm.moe_combine_grad(y, got, slots, weights)
    assert torch.equal(dys[-10::2], y[-5:]) and torch.equal(dys[-9::2], y[-5:])
    ids = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    xs, _, slots = qm.moe_sort(got, ids, 1, out=dys)
    assert torch.equal(xs[-5:], got[-5:]) and slots[-1, 0] == rows - 1


# ---- experts ---------------------------------------------------------------------------------------------------------------


def expert_reference(x, q, scales, group, offsets, out):
    out = out.clone()
    for e in range(q.shape[0]):
        a, b = offsets[e], offsets[e + 1]
        out[a:b] = (x[a:b].double() @ dequantised(q[e], scales[e], group).T).to(out.dtype)
    return out


SEGMENTS = [
    [0, 3, 3, 10, 10],              # experts without rows, rows behind the last segment
    [0, 0, 0, 0, 17],
    [0, 1, 2, 3, 4],
    [0, 16, 33, 50, 130],
    [5, 70, 200, 200, 461],         # rows before the first segment
    [0, 600, 600, 601, 1200],
]


@pytest.mark.parametrize("offsets", SEGMENTS)
@pytest.mark.parametrize("n,k,group,dtype,scale_dtype", [(40, 64, 32, BF16, BF16), (130, 320, 64, FP16, FP32), (256, 1024, 128, BF16, FP32), (64, 94, 64, FP16, FP16)])
def test_experts(qm, cuda_clean, offsets, n, k, group, dtype, scale_dtype):
    rows, experts = offsets[-1] + 3, len(offsets) - 1
    x, q, packed, scales = whole_case(rows, n, k, group, dtype, scale_dtype, 20, (experts,))
    x[offsets[-1] :] = float("nan")  # what no expert has is not read into any result
    out = torch.full((rows, n), SENTINEL, dtype=dtype)
    got = qm.moe_gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), torch.tensor(offsets, dtype=torch.int32).cuda(), group, out=out.cuda())
    assert torch.equal(got.cpu(), expert_reference(x, q, scales, group, offsets, out))


@pytest.mark.parametrize("n,k,rows,longest", [(200, 320, 190, 150), (3300, 128, 190, 100), (130, 256, 1000, 700)])
def test_one_long_segment_among_short_ones(qm, cuda_clean, n, k, rows, longest):
    experts, group = 24, 64
    x, q, packed, scales = whole_case(rows, n, k, group, BF16, BF16, 24, (experts,))
    before = sorted(torch.randint(0, rows - longest + 1, (experts // 2,), generator=torch.Generator().manual_seed(4)).tolist())
    after = sorted(torch.randint(before[-1] + longest, rows + 1, (experts // 2,), generator=torch.Generator().manual_seed(5)).tolist())
    offsets = before + after + [rows]
    out = torch.full((rows, n), SENTINEL, dtype=BF16)
    got = qm.moe_gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), torch.tensor(offsets, dtype=torch.int32).cuda(), group, out=out.cuda())
    assert torch.equal(got.cpu(), expert_reference(x, q, scales, group, offsets, out))


@pytest.mark.parametrize("rows", [300, 2000])
def test_many_experts(qm, cuda_clean, rows):
    experts, n, k, group = 300, 72, 96, 32
    x, q, packed, scales = whole_case(rows, n, k, group, BF16, BF16, 21, (experts,))
    gen = torch.Generator().manual_seed(2)
    offsets = [0] + sorted(torch.randint(0, rows + 1, (experts - 1,), generator=gen).tolist()) + [rows]
    out = torch.full((rows, n), SENTINEL, dtype=BF16)
    got = qm.moe_gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), torch.tensor(offsets, dtype=torch.int32).cuda(), group, out=out.cuda())
    assert torch.equal(got.cpu(), expert_reference(x, q, scales, group, offsets, out))


@pytest.mark.parametrize("rows", [40, 700])
def test_offsets_outside_the_rows_are_clamped(qm, cuda_clean, rows):
    x, q, packed, scales = whole_case(rows, 64, 128, 128, BF16, BF16, 22, (3,))
    out = torch.full((rows, 64), SENTINEL, dtype=BF16)
    bad = torch.tensor([-9, 12, 5, rows + 1000], dtype=torch.int32)  # 5 < 12: the second expert has no rows, the third begins at 12
    got = qm.moe_gemm_w4(x.cuda(), packed.cuda(), scales.cuda(), bad.cuda(), 128, out=out.cuda())
    assert torch.equal(got.cpu(), expert_reference(x, q, scales, 128, [0, 12, 12, rows], out))


@pytest.mark.parametrize("rows", [64, 600])
def test_a_captured_launch_follows_new_offsets(qm, cuda_clean, rows):
    n, k, group = 136, 256, 64
    x, q, packed, scales = whole_case(rows, n, k, group, BF16, BF16, 23, (4,))
    args = (x.cuda(), packed.cuda(), scales.cuda())
    offsets = torch.tensor([0, rows, rows, rows, rows], dtype=torch.int32).cuda()
    out = torch.zeros(rows, n, dtype=BF16, device="cuda")
    qm.init()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        qm.moe_gemm_w4(*args, offsets, group, out=out)
    for new in ([0, 1, 20, 20, rows - 1], [0, 0, 0, 0, 0], [0, rows // 2, rows // 2 + 1, rows, rows]):
        offsets.copy_(torch.tensor(new, dtype=torch.int32))
        out.fill_(SENTINEL)
        g.replay()
        assert torch.equal(out.cpu(), expert_reference(x, q, scales, group, new, torch.full((rows, n), SENTINEL, dtype=BF16)))


def test_no_experts_and_no_rows(qm, cuda_clean):
    out = torch.full((4, 8), SENTINEL, dtype=BF16, device="cuda")
    x, b, s = torch.ones(4, 64, dtype=BF16, device="cuda"), torch.zeros(0, 8, 32, dtype=torch.int8, device="cuda"), torch.zeros(0, 8, 1, dtype=BF16, device="cuda")
    qm.moe_gemm_w4(x, b, s, torch.zeros(1, dtype=torch.int32, device="cuda"), out=out)
    assert bool((out == SENTINEL).all())
    b, s = torch.zeros(2, 8, 32, dtype=torch.int8, device="cuda"), torch.zeros(2, 8, 1, dtype=BF16, device="cuda")
    assert qm.moe_gemm_w4(x[:0], b, s, torch.zeros(3, dtype=torch.int32, device="cuda")).shape == (0, 8)


# ---- quantiser -------------------------------------------------------------------------------------------------------------


def quantiser_reference(w, group, scale_dtype):
    n, k = w.shape
    groups = -(-k // group)
    padded = torch.zeros(n, groups * group)
    padded[:, :k] = w.float()
    padded = padded.view(n, groups, group)
    scales = (padded.abs().amax(-1) * torch.tensor(1 / 7)).to(scale_dtype)  # amax hands a NaN on
    codes = torch.round(padded.double() / scales.double().unsqueeze(-1)).nan_to_num(0.0).clamp(-8, 7).to(torch.int8)
    codes[~torch.isfinite(scales)] = 0
    return codes.view(n, -1)[:, :k], scales


@pytest.mark.parametrize("n,k", [(1, 2), (3, 30), (5, 34), (7, 64), (4, 130), (33, 256), (9, 1000), (130, 2208), (64, 4096), (3, 11008)])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype,scale_dtype", [(BF16, BF16), (FP16, FP16), (FP32, FP32), (BF16, FP32), (FP16, FP32)])
def test_quantiser(qm, cuda_clean, n, k, group, dtype, scale_dtype):
    w = (0.02 * torch.randn(n, k, generator=torch.Generator().manual_seed(n + k))).to(dtype)
    codes_, scales = quantiser_reference(w, group, scale_dtype)
    packed, got = qm.quantize_w4(w.cuda(), group, scale_dtype=scale_dtype)
    assert got.dtype == scale_dtype and torch.equal(got.cpu(), scales)
    assert torch.equal(qm.unpack(packed).cpu(), codes_)


def test_quantiser_at_ties_and_borders(qm, cuda_clean):
    """Values at, and one place beside, the middle between two codes; the largest value is 7 * scale, so the scale is exact."""
    for dtype, scale in ((FP32, 0.3), (FP32, 1.0), (FP16, 0.25), (BF16, 2.0)):
        s = torch.tensor(scale, dtype=torch.float32)
        mid = (torch.arange(-7, 7) + 0.5).float() * s
        w = torch.stack([mid, torch.nextafter(mid, torch.tensor(9.0)), torch.nextafter(mid, torch.tensor(-9.0))]).to(dtype).flatten()
        w = torch.cat([w, torch.zeros(63 - w.numel(), dtype=dtype), (7 * s).to(dtype).view(1)]).view(1, 64)
        codes_, scales = quantiser_reference(w, 64, dtype)
        packed, got = qm.quantize_w4(w.cuda(), 64)
        assert torch.equal(got.cpu(), scales) and torch.equal(qm.unpack(packed).cpu(), codes_)


def test_quantiser_groups_of_zeros_infinities_and_nan(qm, cuda_clean):
    w = torch.randn(4, 256, generator=torch.Generator().manual_seed(3))
    w[0, :64] = 0
    w[1, 70] = float("inf")
    w[2, 3], w[2, 4] = float("nan"), float("-inf")
    w[3, 64:128] *= 1e-42  # subnormal values and scale
    codes_, scales = quantiser_reference(w, 64, FP32)
    packed, got = qm.quantize_w4(w.cuda(), 64)
    assert torch.equal(torch.nan_to_num(got.cpu(), nan=-1.0), torch.nan_to_num(scales, nan=-1.0))
    got_codes = qm.unpack(packed).cpu()
    assert torch.equal(got_codes[:3], codes_[:3]) and torch.equal(got_codes[3, :64], codes_[3, :64]) and torch.equal(got_codes[3, 128:], codes_[3, 128:])
    assert torch.equal(got_codes[3, 64:128], codes_[3, 64:128])
    assert got[0, 0] == 0 and torch.isinf(got[1, 1]) and torch.isnan(got[2, 0])


@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 1)])
def test_quantiser_of_a_column_slab(qm, cuda_clean, pad, shift):
    wide = torch.randn(40, 192 + pad + shift, generator=torch.Generator().manual_seed(4))
    w = wide[:, shift : shift + 192]
    codes_, scales = quantiser_reference(w, 64, FP32)
    packed, got = qm.quantize_w4(wide.cuda()[:, shift : shift + 192], 64)
    assert torch.equal(got.cpu(), scales) and torch.equal(qm.unpack(packed).cpu(), codes_)


def test_quantised_weights_in_a_product(qm, cuda_clean):
    """The two together: no weight is off by more than half its group's scale, and the product is that of the quantised weights."""
    w = 0.02 * torch.randn(300, 1024, generator=torch.Generator().manual_seed(5))
    for dtype in (BF16, FP16):
        packed, scales = qm.quantize_w4(w.to(dtype).cuda(), 128)
        back = dequantised(qm.unpack(packed).cpu(), scales.cpu(), 128)
        at = torch.arange(1024) // 128
        # the largest value's quotient exceeds 7 by the rounding of the scale at most, and is clamped to 7
        slack = 0.5 + 7 * torch.finfo(dtype).eps / 2
        assert bool(((back - w.to(dtype).double()).abs() <= slack * scales.cpu().double()[:, at]).all())
        x = torch.randn(20, 1024, generator=torch.Generator().manual_seed(6)).to(dtype)
        close_to(qm.gemm_w4(x.cuda(), packed, scales), x, back)


# ---- refusals --------------------------------------------------------------------------------------------------------------


@pytest.fixture(params=["compiled", "ctypes"])
def binding(request, monkeypatch):
    """Both ways into the library: the compiled binding, and the ctypes form that is used without it."""
    import quadmul_b200.moe
    import quadmul_b200.w4

    if request.param == "ctypes":
        monkeypatch.setattr(quadmul_b200.w4, "_EXT", None)
        monkeypatch.setattr(quadmul_b200.moe, "_EXT", None)
    elif quadmul_b200.w4._EXT is None:
        pytest.skip("the compiled binding is not built")


def test_both_bindings(qm, cuda_clean, binding):
    x, q, packed, scales = whole_case(9, 40, 128, 64, BF16, FP32, 30)
    want = (x.double() @ dequantised(q, scales, 64).T).to(BF16)
    assert torch.equal(run(qm, x, packed, scales, 64).cpu(), want)
    offsets = torch.tensor([0, 4, 9], dtype=torch.int32).cuda()
    two = (torch.stack([packed, packed]).cuda(), torch.stack([scales, scales]).cuda())
    assert torch.equal(qm.moe_gemm_w4(x.cuda(), *two, offsets, 64).cpu(), want)
    codes_, s = quantiser_reference(x.float(), 64, FP32)
    p, got = qm.quantize_w4(x.cuda(), 64, scale_dtype=FP32)
    assert torch.equal(got.cpu(), s) and torch.equal(qm.unpack(p).cpu(), codes_)


def test_refusals(qm, cuda_clean, binding):
    def make(m=4, n=8, k=64, dtype=BF16, group=64):
        return [torch.zeros(m, k, dtype=dtype, device="cuda"), torch.zeros(n, k // 2, dtype=torch.int8, device="cuda"),
                torch.zeros(n, -(-k // group), dtype=dtype, device="cuda"), group]

    x, b, s, g = make()
    assert qm.gemm_w4(x, b, s, g).shape == (4, 8)
    for args, error in [
        ((x.float(), b, s, g), TypeError), ((x, b.float(), s, g), TypeError), ((x, b, s.half(), g), TypeError), ((x, b, s.double(), g), TypeError),
        ((x, b, s, 48), ValueError), ((x, b, s, 0), ValueError), ((x[:, :62], b, s, g), ValueError), ((x[:, :63], b, s, g), ValueError),
        ((x, b, s, 32), ValueError), ((x[0], b, s, g), ValueError), ((x, b[None], s, g), ValueError), ((x.cpu(), b, s, g), ValueError),
        ((x, b.cpu(), s, g), ValueError), ((x, b, s.cpu(), g), ValueError), ((x, b.t().contiguous().t(), s, g), ValueError),
        ((x.t().contiguous().t(), b, s, g), ValueError), ((x[:1].expand(4, 64), b, s, g), ValueError), ((x.clone().requires_grad_(), b, s, g), ValueError),
    ]:
        with pytest.raises(error):
            qm.gemm_w4(*args)
    for out, error in [(torch.zeros(4, 9, dtype=BF16, device="cuda"), ValueError), (torch.zeros(4, 8, device="cuda"), TypeError),
                       (torch.zeros(8, 4, dtype=BF16, device="cuda").t(), ValueError), (torch.zeros(4, 8, dtype=BF16), ValueError)]:
        with pytest.raises(error):
            qm.gemm_w4(x, b, s, g, out=out)
    with torch.no_grad():
        qm.gemm_w4(x.clone().requires_grad_(), b, s, g)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    eb, es = torch.zeros(2, 8, 32, dtype=torch.int8, device="cuda"), torch.zeros(2, 8, 1, dtype=BF16, device="cuda")
    qm.moe_gemm_w4(x, eb, es, off, g)
    for args, error in [((x, eb, es, off.long(), g), ValueError), ((x, eb, es, off[:2], g), ValueError), ((x, eb, es, off.cpu(), g), ValueError),
                        ((x, eb[0], es, off, g), ValueError), ((x, eb, es[:1], off, g), ValueError)]:
        with pytest.raises(error):
            qm.moe_gemm_w4(*args)
    w = torch.zeros(4, 64, device="cuda")
    for args, kw, error in [((w.double(),), {}, TypeError), ((w.int(),), {}, TypeError), ((w, 48), {}, ValueError), ((w[:, :63], 64), {}, ValueError),
                            ((w,), {"scale_dtype": BF16}, TypeError), ((w.cpu(),), {}, ValueError), ((w[0],), {}, ValueError)]:
        with pytest.raises(error):
            qm.quantize_w4(*args, **kw)
    torch.cuda.synchronize()
