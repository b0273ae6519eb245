"""moe_sort with as many experts as it takes and more assignments than fit one block, from one thread and from many; more than eight
experts per token."""
import threading

import pytest
import torch

from _w4 import HALF_STEP

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def order(ids, experts):
    """Offsets and slots of a stable sort by expert, -1 where an id is outside [0, experts)."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    place = torch.argsort(key, stable=True)
    slots = torch.empty_like(place)
    slots[place] = torch.arange(flat.numel())
    slots = torch.where(key < experts, slots, -1)
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    return torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).int(), slots.int().view(ids.shape)


@pytest.mark.parametrize("tokens,top_k,experts", [(330_000, 4, 4096), (500_000, 5, 4096), (130_000, 17, 3000), (700, 4096, 4096)])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_sort_of_many(qm, cuda_clean, tokens, top_k, experts, id_type):
    hidden = 2
    gen = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-2, experts + 2, (tokens, top_k), generator=gen)
    x = torch.randint(-100, 100, (tokens, hidden), generator=gen).to(BF16)
    offsets, slots = order(ids, experts)
    xs, got_offsets, got_slots = qm.moe_sort(x.cuda(), ids.to(id_type).cuda(), experts)
    assert torch.equal(got_offsets.cpu(), offsets) and torch.equal(got_slots.cpu(), slots)
    live = slots >= 0
    assert torch.equal(xs.cpu()[slots[live].long()], x.unsqueeze(1).expand(-1, top_k, -1)[live])


def test_threads_sort_different_sizes(qm, cuda_clean):
    """All need more shared memory than a launch has by default, some more than others: none may take it away from another."""
    from quadmul_b200._lib import LIB

    experts, top_k = 4096, 8
    failed = []
    sizes = 6 * (300_000, 160_000)
    start = threading.Barrier(len(sizes))

    def work(tokens):
        stream = torch.cuda.Stream()
        ids = torch.zeros(tokens, top_k, dtype=torch.int32, device="cuda")
        offsets, slots = torch.empty(experts + 1, dtype=torch.int32, device="cuda"), torch.empty_like(ids)
        need = LIB.qm_moe_sort_workspace_bytes(tokens, top_k, experts)
        space = torch.empty(need // 4, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        start.wait()
        for _ in range(400):
            st = LIB.qm_moe_sort(None, 2, 0, ids.data_ptr(), 4, experts, None, 0, offsets.data_ptr(), slots.data_ptr(), tokens, top_k, 0, space.data_ptr(),
                                 need, stream.cuda_stream)
            if st:
                failed.append((tokens, st))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, f"{len(failed)} calls refused, the first {failed[0]}"


@pytest.mark.parametrize("top_k", [9, 16, 23, 64])
@pytest.mark.parametrize("hidden", [7, 64, 2056])
@pytest.mark.parametrize("dtype,weight_dtype", [(BF16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
def test_more_than_eight_experts_per_token(qm, cuda_clean, top_k, hidden, dtype, weight_dtype):
    tokens, experts = 40, 70
    gen = torch.Generator().manual_seed(top_k)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=gen)
    _, slots = order(ids, experts)
    rows = tokens * top_k
    ys, dy = torch.randn(rows, hidden, generator=gen).to(dtype), torch.randn(tokens, hidden, generator=gen).to(dtype)
    weights = torch.rand(tokens, top_k, generator=gen).to(weight_dtype)
    live = slots >= 0
    part = torch.where(live.unsqueeze(-1), ys.double()[slots.clamp(min=0).long()], 0.0)
    weighted = part * weights.double().unsqueeze(-1)
    got = qm.moe_combine(ys.cuda(), slots.cuda(), weights.cuda()).cpu()
    # the result's rounding, and one fp32 rounding of a partial sum for each product
    limit = HALF_STEP[dtype] * weighted.sum(1).abs() + (top_k + 1) * 2.0**-24 * weighted.abs().sum(1) + 2.0**-24 * 2.0**-10
    assert bool(((got.double() - weighted.sum(1)).abs() <= limit).all())
    dys, dweights = qm.moe_combine_grad(dy.cuda(), ys.cuda(), slots.cuda(), weights.cuda(), out=torch.full_like(ys, -77.0).cuda())
    want = torch.full_like(ys, -77.0)
    want[slots[live].long()] = (weights.float().unsqueeze(-1) * dy.float().unsqueeze(1)).to(dtype)[live]
    assert torch.equal(dys.cpu(), want)
    dots = part * dy.double().unsqueeze(1)
    limit = HALF_STEP[weight_dtype] * dots.sum(-1).abs() + (hidden + 1) * 2.0**-24 * dots.abs().sum(-1) + 2.0**-24
    assert bool(((dweights.cpu().double() - dots.sum(-1)).abs() <= limit).all())
