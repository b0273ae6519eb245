"""moe_sort, moe_combine, their gradients and moe_linear_w4 against their definitions in 64 bits."""
import pytest
import torch

from _w4 import HALF_STEP, codes, dequantised

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SENTINEL = -77.0

# (tokens, top_k, experts, hidden, share of dropped assignments)
CASES = [
    (1, 1, 1, 1, 0.0), (1, 8, 64, 64, 0.0), (2, 3, 4, 7, 0.5), (16, 8, 64, 128, 0.1), (33, 2, 8, 120, 0.0), (64, 6, 60, 1000, 0.2), (100, 4, 4096, 24, 0.1),
    (500, 1, 3, 257, 0.3), (1000, 2, 8, 512, 0.0), (2049, 8, 128, 72, 0.05), (3001, 6, 200, 40, 0.0), (9000, 4, 16, 8, 0.1), (20000, 2, 300, 4, 0.0),
    (5, 4, 8, 4096, 1.0),
]


def routing(tokens, top_k, experts, drop, seed):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen)  # the same expert may come twice for a token
    out = torch.rand(tokens, top_k, generator=gen) < drop
    # what is outside the range in any way is dropped
    ids[out] = torch.tensor([-1, -5, experts, experts + 3])[torch.randint(0, 4, (int(out.sum()),), generator=gen)]
    return ids


def order(ids, experts):
    flat = ids.flatten().tolist()
    places = [[i for i, e in enumerate(flat) if e == x] for x in range(experts)] if experts <= 64 else None
    if places is None:
        places = [[] for _ in range(experts)]
        for i, e in enumerate(flat):
            if 0 <= e < experts:
                places[e].append(i)
    offsets, slots, at = [0], [-1] * len(flat), 0
    for p in places:
        for i in p:
            slots[i] = at
            at += 1
        offsets.append(at)
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(slots, dtype=torch.int32).view(ids.shape)


@pytest.mark.parametrize("tokens,top_k,experts,hidden,drop", CASES)
@pytest.mark.parametrize("dtype,id_type", [(BF16, torch.int64), (FP32, torch.int32), (FP16, torch.int32)])
def test_sort(qm, cuda_clean, tokens, top_k, experts, hidden, drop, dtype, id_type):
    ids = routing(tokens, top_k, experts, drop, tokens)
    x = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(1)).to(dtype)
    offsets, slots = order(ids, experts)
    xs = torch.full((tokens * top_k, hidden), SENTINEL, dtype=dtype)
    live = slots >= 0
    xs[slots[live].long()] = x.unsqueeze(1).expand(-1, top_k, -1)[live]
    got_xs, got_offsets, got_slots = qm.moe_sort(x.cuda(), ids.to(id_type).cuda(), experts, out=torch.full_like(xs, SENTINEL).cuda())
    assert torch.equal(got_offsets.cpu(), offsets) and torch.equal(got_slots.cpu(), slots)
    assert torch.equal(got_xs.cpu(), xs)


def case(tokens, top_k, experts, hidden, drop, dtype, weight_dtype, extra=3):
    ids = routing(tokens, top_k, experts, drop, tokens)
    offsets, slots = order(ids, experts)
    gen = torch.Generator().manual_seed(2)
    rows = tokens * top_k + extra
    ys = torch.randn(rows, hidden, generator=gen).to(dtype)
    weights = torch.rand(tokens, top_k, generator=gen).to(weight_dtype)
    dy = torch.randn(tokens, hidden, generator=gen).to(dtype)
    return slots, ys, weights, dy


def gathered(ys, slots, rows):
    """float64 [tokens, top_k, hidden], zeros where the slot is none, and which slots are some."""
    live = (slots >= 0) & (slots < rows)
    return torch.where(live.unsqueeze(-1), ys.double()[slots.clamp(0, rows - 1).long()], 0.0), live


@pytest.mark.parametrize("tokens,top_k,experts,hidden,drop", CASES)
@pytest.mark.parametrize("dtype,weight_dtype", [(BF16, FP32), (FP16, FP16), (FP32, FP32), (BF16, BF16), (FP16, FP32)])
def test_combine(qm, cuda_clean, tokens, top_k, experts, hidden, drop, dtype, weight_dtype):
    slots, ys, weights, _ = case(tokens, top_k, experts, hidden, drop, dtype, weight_dtype)
    rows, live = gathered(ys, slots, ys.shape[0])
    for w in (weights, None):
        got = qm.moe_combine(ys.cuda(), slots.cuda(), None if w is None else w.cuda())
        part = rows if w is None else rows * w.double().unsqueeze(-1)
        # the result's rounding, and one fp32 rounding of a partial sum for each of the top_k products
        limit = HALF_STEP[dtype] * part.sum(1).abs() + (top_k + 1) * 2.0**-24 * part.abs().sum(1) + 2.0**-24 * torch.finfo(dtype).smallest_normal * 2.0**14
        assert got.dtype == dtype and bool(((got.cpu().double() - part.sum(1)).abs() <= limit).all())
        assert bool((got.cpu()[~live.any(1)] == 0).all())
        if w is None:
            assert torch.equal(qm.moe_sort_grad(ys.cuda(), slots.cuda()), got)


@pytest.mark.parametrize("tokens,top_k,experts,hidden,drop", CASES)
@pytest.mark.parametrize("dtype,weight_dtype", [(BF16, FP32), (FP16, FP16), (FP32, FP32), (BF16, BF16), (FP16, FP32)])
def test_combine_grad(qm, cuda_clean, tokens, top_k, experts, hidden, drop, dtype, weight_dtype):
    slots, ys, weights, dy = case(tokens, top_k, experts, hidden, drop, dtype, weight_dtype)
    rows, live = gathered(ys, slots, ys.shape[0])
    out = torch.full_like(ys, SENTINEL)
    dys, dweights = qm.moe_combine_grad(dy.cuda(), ys.cuda(), slots.cuda(), weights.cuda(), out=out.cuda())
    want = out.clone()
    # weight * dy is exact in 64 bits and, for 16-bit operands, in fp32 up to one rounding; the second is the type's
    back = (weights.float().unsqueeze(-1) * dy.float().unsqueeze(1)).to(dtype)
    want[slots[live].long()] = back[live]
    assert torch.equal(dys.cpu(), want)
    dots = rows * dy.double().unsqueeze(1)
    size = dots.abs().sum(-1)
    # a sum of `hidden` fp32 products: at most one rounding of a partial sum each
    limit = HALF_STEP[weight_dtype] * dots.sum(-1).abs() + (hidden + 1) * 2.0**-24 * size + 2.0**-24
    assert dweights.dtype == weight_dtype and bool(((dweights.cpu().double() - dots.sum(-1)).abs() <= limit).all())
    assert bool((dweights.cpu()[~live] == 0).all())


def test_gradients_against_differences(qm, cuda_clean):
    """sort, a scaling per row, combine: a change along a direction changes the result by the gradient's product with it."""
    tokens, top_k, experts, hidden = 7, 3, 5, 16
    ids = routing(tokens, top_k, experts, 0.2, 4).cuda()
    gen = torch.Generator().manual_seed(5)
    x, dx = (torch.randn(tokens, hidden, generator=gen).cuda() for _ in range(2))
    w, dw = (torch.rand(tokens, top_k, generator=gen).cuda() for _ in range(2))
    scale = torch.rand(tokens * top_k, 1, generator=gen).cuda() + 0.5
    probe = torch.randn(tokens, hidden, generator=gen).cuda()

    def loss(x, w):
        xs, _, slots = qm.moe_sort(x, ids, experts, out=torch.zeros(tokens * top_k, hidden, device="cuda"))
        return float((qm.moe_combine(xs * scale, slots, w).double() * probe.double()).sum())

    xs, _, slots = qm.moe_sort(x, ids, experts, out=torch.zeros(tokens * top_k, hidden, device="cuda"))
    dys, dweights = qm.moe_combine_grad(probe, xs * scale, slots, w, out=torch.zeros(tokens * top_k, hidden, device="cuda"))
    gx = qm.moe_sort_grad(dys * scale, slots)
    h = 2.0**-6
    # the loss is linear in x and in w, so the central difference has no error of its own: only fp32 roundings of sums of
    # tokens * hidden terms of size one, divided by h
    limit = 4 * tokens * hidden * 2.0**-24 / h
    assert abs((loss(x + h * dx, w) - loss(x - h * dx, w)) / (2 * h) - float((gx * dx).double().sum())) <= limit * 8
    assert abs((loss(x, w + h * dw) - loss(x, w - h * dw)) / (2 * h) - float((dweights * dw).double().sum())) <= limit * 8


@pytest.mark.parametrize("hidden,pad,shift", [(64, 8, 0), (64, 3, 1), (33, 2, 1)])
def test_column_slabs(qm, cuda_clean, hidden, pad, shift):
    tokens, top_k, experts = 50, 3, 6
    ids = routing(tokens, top_k, experts, 0.1, 6)
    offsets, slots = order(ids, experts)

    def slab(rows, fill=None):
        wide = torch.randn(rows, hidden + pad + shift, generator=torch.Generator().manual_seed(rows)).to(BF16) if fill is None else torch.full(
            (rows, hidden + pad + shift), fill, dtype=BF16)
        wide = wide.cuda()
        return wide, wide[:, shift : shift + hidden]

    _, x = slab(tokens)
    wide, out = slab(tokens * top_k, SENTINEL)
    qm.moe_sort(x, ids.cuda(), experts, out=out)
    want = torch.full((tokens * top_k, hidden + pad + shift), SENTINEL, dtype=BF16)
    live = slots >= 0
    want[slots[live].long(), shift : shift + hidden] = x.cpu().unsqueeze(1).expand(-1, top_k, -1)[live]
    assert torch.equal(wide.cpu(), want)
    _, ys = slab(tokens * top_k)
    wide, out = slab(tokens, SENTINEL)
    y = qm.moe_combine(ys, slots.cuda(), None, out=out)
    plain = qm.moe_combine(ys.contiguous(), slots.cuda())
    assert torch.equal(y, plain) and bool((wide[:, :shift] == SENTINEL).all()) and bool((wide[:, shift + hidden :] == SENTINEL).all())
    weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(1)).cuda()
    wide, out = slab(tokens * top_k, SENTINEL)
    dys, dweights = qm.moe_combine_grad(x, ys, slots.cuda(), weights, out=out)
    same, dsame = qm.moe_combine_grad(x.contiguous(), ys.contiguous(), slots.cuda(), weights, out=torch.full((tokens * top_k, hidden), SENTINEL, dtype=BF16).cuda())
    assert torch.equal(dys, same)
    assert bool((wide[:, :shift] == SENTINEL).all()) and bool((wide[:, shift + hidden :] == SENTINEL).all())
    assert bool(((dweights - dsame).abs() <= hidden * 2.0**-23 * 64).all())  # the order of the sum may differ


def test_slots_outside_the_rows_add_nothing(qm, cuda_clean):
    ys = torch.randn(6, 8, generator=torch.Generator().manual_seed(7)).cuda()
    slots = torch.tensor([[0, 6], [-1, 5], [2**31 - 1, -(2**31)]], dtype=torch.int32).cuda()
    w = torch.full((3, 2), 2.0).cuda()
    y = qm.moe_combine(ys, slots, w)
    assert torch.equal(y[0], 2 * ys[0]) and torch.equal(y[1], 2 * ys[5]) and bool((y[2] == 0).all())
    dys, dw = qm.moe_combine_grad(torch.ones(3, 8).cuda(), ys, slots, w, out=torch.full((6, 8), SENTINEL).cuda())
    assert bool((dys[0] == 2).all()) and bool((dys[5] == 2).all()) and bool((dys[1:5] == SENTINEL).all())
    assert bool((dw[2] == 0).all()) and dw[0, 1] == 0 and dw[1, 0] == 0


def test_empty_sizes(qm, cuda_clean):
    x = torch.zeros(0, 8, device="cuda")
    xs, offsets, slots = qm.moe_sort(x, torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 4)
    assert xs.shape == (0, 8) and offsets.tolist() == [0] * 5 and slots.shape == (0, 2)
    x = torch.ones(3, 8, device="cuda")
    xs, offsets, slots = qm.moe_sort(x, torch.zeros(3, 0, dtype=torch.int64, device="cuda"), 4)
    assert xs.shape == (0, 8) and offsets.tolist() == [0] * 5
    assert bool((qm.moe_combine(xs, slots) == 0).all())
    xs, offsets, slots = qm.moe_sort(x, torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 0)
    assert offsets.tolist() == [0] and slots.flatten().tolist() == [-1] * 6
    many = torch.ones(9000, 8, device="cuda")  # more ids than one launch sorts
    _, offsets, slots = qm.moe_sort(many, torch.zeros(9000, 2, dtype=torch.int32, device="cuda"), 0)
    assert offsets.tolist() == [0] and bool((slots == -1).all())
    y = qm.moe_linear_w4(many.bfloat16(), torch.zeros(9000, 2, dtype=torch.int32, device="cuda"), torch.ones(9000, 2, device="cuda"),
                         torch.zeros(0, 6, 4, dtype=torch.int8, device="cuda"), torch.zeros(0, 6, 1, dtype=BF16, device="cuda"))
    assert y.shape == (9000, 6) and bool((y == 0).all())
    xs, offsets, slots = qm.moe_sort(x[:, :0], torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 2)
    assert xs.shape == (6, 0) and offsets.tolist() == [0, 6, 6] and slots.flatten().tolist() == list(range(6))
    dys, dw = qm.moe_combine_grad(x[:, :0], xs, slots, torch.ones(3, 2, device="cuda"))
    assert dys.shape == (6, 0) and bool((dw == 0).all())


def test_captured_on_another_stream(qm, cuda_clean):
    """The steps of one projection in one graph, replayed with other tokens and another routing."""
    tokens, top_k, experts, k, n = 24, 4, 8, 128, 96
    q, packed = codes((experts, n, k), torch.Generator().manual_seed(8))
    scales = torch.exp2(torch.randint(-2, 2, (experts, n, 1), generator=torch.Generator().manual_seed(9)).float()).to(BF16)
    x = torch.zeros(tokens, k, dtype=BF16, device="cuda")
    ids = torch.zeros(tokens, top_k, dtype=torch.int64, device="cuda")
    w = torch.zeros(tokens, top_k, device="cuda")
    b, s = packed.cuda(), scales.cuda()
    qm.init()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = qm.moe_linear_w4(x, ids, w, b, s, 128)
    for seed in (1, 2, 3):
        gen = torch.Generator().manual_seed(seed)
        new_x = torch.randint(-2, 3, (tokens, k), generator=gen).to(BF16)
        new_ids = routing(tokens, top_k, experts, 0.2, seed)
        new_w = torch.exp2(torch.randint(-2, 1, (tokens, top_k), generator=gen).float())
        x.copy_(new_x), ids.copy_(new_ids), w.copy_(new_w)
        g.replay()
        assert_linear(y, new_x, new_ids, new_w, q, scales, 128)
        assert torch.equal(qm.moe_linear_w4(x, ids, w, b, s, 128), y)


def assert_linear(y, x, ids, w, q, scales, group):
    experts = q.shape[0]
    full = torch.stack([x.double() @ dequantised(q[e], scales[e], group).T for e in range(experts)])  # experts, tokens, n
    live = (ids >= 0) & (ids < experts)
    rows = full[ids.clamp(0, experts - 1), torch.arange(x.shape[0]).unsqueeze(1)]  # tokens, top_k, n
    part = torch.where(live.unsqueeze(-1), rows, 0.0) * w.double().unsqueeze(-1)
    # every product is rounded to the type once, and so is the sum
    u = HALF_STEP[y.dtype]
    limit = (1 + u) * u * part.abs().sum(1) + u * part.sum(1).abs() + 2.0**-20 * part.abs().sum(1)
    assert bool(((y.cpu().double() - part.sum(1)).abs() <= limit).all())


@pytest.mark.parametrize("tokens", [1, 16, 500])
def test_a_feed_forward_layer_of_experts(qm, cuda_clean, tokens):
    """As a program runs them: quantised weights, tokens sorted once, two products with an activation between them, combined."""
    top_k, experts, hidden, inner, group = 2, 6, 256, 384, 64
    gen = torch.Generator().manual_seed(11)
    up, down = (0.05 * torch.randn(experts, a, b, generator=gen) for a, b in ((2 * inner, hidden), (hidden, inner)))
    (ub, us), (db, ds) = ([t.view(experts, *shape) for t, shape in zip(qm.quantize_w4(w.to(BF16).view(-1, w.shape[-1]).cuda(), group), (
        (w.shape[1], w.shape[2] // 2), (w.shape[1], w.shape[2] // group)))] for w in (up, down))
    x = torch.randn(tokens, hidden, generator=gen).to(BF16)
    value, ids = torch.topk(torch.randn(tokens, experts, generator=gen), top_k, dim=1)
    w = torch.softmax(value, 1)
    xs, offsets, slots = qm.moe_sort(x.cuda(), ids.cuda(), experts)
    h = qm.moe_gemm_w4(xs, ub, us, offsets, group)
    gate, lin = h.chunk(2, dim=1)
    act = torch.nn.functional.silu(gate.float()).mul(lin.float()).to(BF16)
    y = qm.moe_combine(qm.moe_gemm_w4(act, db, ds, offsets, group), slots, w.cuda()).cpu()
    uw, dw = (dequantised(qm.unpack(b.view(-1, b.shape[-1])).cpu(), s.cpu().view(-1, s.shape[-1]), group).view(experts, b.shape[1], -1) for b, s in ((ub, us), (db, ds)))
    want = torch.zeros(tokens, hidden, dtype=torch.float64)
    for t in range(tokens):
        for j in range(top_k):
            h64 = uw[ids[t, j]] @ x[t].double()
            g64, l64 = h64.chunk(2)
            want[t] += w[t, j].double() * (dw[ids[t, j]] @ (torch.nn.functional.silu(g64) * l64))
    # the layer rounds to bf16 five times on the way (both products' weights and results, the activation) and once at the end:
    # six independent roundings of half a step, in 2-norm
    assert float((y.double() - want).norm() / want.norm()) <= 6 * HALF_STEP[BF16]


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


@pytest.mark.parametrize("tokens", [40, 5000])
def test_both_bindings(qm, cuda_clean, binding, tokens):
    top_k, experts, hidden = 4, 9, 24
    ids = routing(tokens, top_k, experts, 0.1, 1)
    offsets, slots = order(ids, experts)
    x = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(2))
    xs, got_offsets, got_slots = qm.moe_sort(x.cuda(), ids.cuda(), experts)
    assert torch.equal(got_offsets.cpu(), offsets) and torch.equal(got_slots.cpu(), slots)
    w = torch.ones(tokens, top_k).cuda()
    assert torch.equal(qm.moe_combine(xs, got_slots, w), qm.moe_sort_grad(xs, got_slots))
    dys, dw = qm.moe_combine_grad(x.cuda(), xs, got_slots, w)
    last = int(offsets[-1])
    assert torch.equal(dys[:last], xs[:last]) and dw.shape == w.shape


def test_refusals(qm, cuda_clean, binding):
    x, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    for args, error in [((x.double(), ids, 3), TypeError), ((x.int(), ids, 3), TypeError), ((x, ids.float(), 3), TypeError), ((x, ids[:3], 3), ValueError),
                        ((x, ids[:, 0], 3), ValueError), ((x, ids, -1), ValueError), ((x, ids, 4097), ValueError), ((x.cpu(), ids, 3), ValueError),
                        ((x, ids.cpu(), 3), ValueError), ((x.t(), ids, 3), ValueError), ((x, ids.t().contiguous().t(), 3), ValueError),
                        ((x[:1].expand(4, 8), ids, 3), ValueError), ((x.clone().requires_grad_(), ids, 3), ValueError)]:
        with pytest.raises(error):
            qm.moe_sort(*args)
    for out, error in [(torch.zeros(7, 8, device="cuda"), ValueError), (torch.zeros(8, 8, device="cuda").half(), TypeError), (torch.zeros(8, 8), ValueError)]:
        with pytest.raises(error):
            qm.moe_sort(x, ids, 3, out=out)
    ys, slots, w = torch.zeros(8, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    for args, error in [((ys.int(), slots, w), TypeError), ((ys, slots.long(), w), ValueError), ((ys, slots[0], w), ValueError), ((ys, slots, w[:3]), ValueError),
                        ((ys, slots, w.half()), TypeError), ((ys, slots, w.cpu()), ValueError), ((ys, slots.cpu(), w), ValueError), ((ys.t(), slots, w), ValueError),
                        ((ys, slots, w.clone().requires_grad_()), ValueError), ((ys.clone().requires_grad_(), slots, w), ValueError)]:
        with pytest.raises(error):
            qm.moe_combine(*args)
        with pytest.raises(error):
            qm.moe_combine_grad(x, *args)
    for args, error in [((x.half(), ys, slots, w), TypeError), ((x[:3], ys, slots, w), ValueError), ((x[:, :4], ys, slots, w), ValueError), ((x.cpu(), ys, slots, w), ValueError)]:
        with pytest.raises(error):
            qm.moe_combine_grad(*args)
    with pytest.raises(ValueError):
        qm.moe_linear_w4(x.half(), ids, w, torch.zeros(8, 4, dtype=torch.int8, device="cuda"), torch.zeros(8, 1, device="cuda"))
    torch.cuda.synchronize()
