"""Tokens to experts and back, with gradients, around the experts' products (w4.moe_gemm_w4).

  moe_sort(x, ids, experts)            rows of x in expert order, the experts' offsets, every assignment's slot
  moe_combine(ys, slots, weights)      y[t] = sum_j weights[t, j] * ys[slots[t, j]]
  moe_sort_grad, moe_combine_grad      their gradients, as calls of their own (nothing here is recorded by autograd)
  moe_linear_w4(...)                   the three steps of one 4-bit expert projection

The reference has no counterpart.  Everything is deterministic: there are no floating-point atomics.  An `out` must not share
elements with the inputs.
"""
from __future__ import annotations

from . import _EXT, _count, _on_device, _stream_of, _torch
from ._lib import LIB, check
from .w4 import check_out, check_rows, check_sizes, check_whole, compiled, moe_gemm_w4, pitch, type_of

MAX_EXPERTS = 4096


def check_assignments(what, tokens, top_k):
    check_sizes(what, "the number of tokens", (tokens,))
    if top_k > MAX_EXPERTS or tokens * top_k >= 1 << 31:
        raise ValueError(f"{what}: too many assignments")


def _check_slots(what, slots, device):
    if slots.dim() != 2 or slots.dtype != _torch().int32:
        raise ValueError(f"{what}: slots must be int32 [tokens, top_k]")
    check_whole(what, device, slots=slots)
    check_assignments(what, *slots.shape)


def _check_weights(what, weights, slots, like):
    check_whole(what, like.device, weights=weights)
    if tuple(weights.shape) != tuple(slots.shape):
        raise ValueError(f"{what}: weights have shape {tuple(weights.shape)}, slots {tuple(slots.shape)}")
    torch = _torch()
    if weights.dtype not in (like.dtype, torch.float32):
        raise TypeError(f"{what}: weights must be {like.dtype} or torch.float32")
    return type_of(what, "weights", weights)


def moe_sort(x, expert_ids, num_experts: int, out=None):
    """x [tokens, hidden], expert_ids [tokens, top_k] (int32 or int64) -> (xs, offsets, slots).

    xs [tokens * top_k, hidden] holds x[t] at row slots[t, j] for every assignment; rows are grouped by expert and in the order of
    (t, j) within one.  offsets (int32, num_experts + 1) are the groups' bounds, slots (int32, [tokens, top_k]) is -1 for an
    assignment whose id is outside [0, num_experts): it is dropped.  Rows of xs from offsets[-1] on are left as they were in
    `out` (and undefined in an xs that is allocated here)."""
    what = "moe_sort"
    torch = _torch()
    if _EXT is not None:
        return compiled(_EXT.moe_sort, x, expert_ids, num_experts, out)
    code = type_of(what, "x", x)
    check_rows(what, x=x)
    check_whole(what, x.device, expert_ids=expert_ids)
    if expert_ids.dim() != 2 or expert_ids.shape[0] != x.shape[0]:
        raise ValueError(f"{what}: expert_ids must be [tokens, top_k]")
    if expert_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: expert_ids must be int32 or int64")
    if not 0 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"{what}: num_experts must be within [0, {MAX_EXPERTS}]")
    (tokens, hidden), top_k = x.shape, expert_ids.shape[1]
    check_assignments(what, tokens, top_k)
    xs = check_out(what, "out", out, (tokens * top_k, hidden), x)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=x.device)
    slots = torch.empty((tokens, top_k), dtype=torch.int32, device=x.device)
    need = LIB.qm_moe_sort_workspace_bytes(tokens, top_k, num_experts)
    workspace = torch.empty(need // 4, dtype=torch.int32, device=x.device) if need else None
    with _on_device(x):
        st = LIB.qm_moe_sort(x.data_ptr(), code, pitch(x), expert_ids.data_ptr(), expert_ids.element_size(), num_experts, xs.data_ptr(), pitch(xs),
                             offsets.data_ptr(), slots.data_ptr(), tokens, top_k, hidden, None if workspace is None else workspace.data_ptr(),
                             need, _stream_of(x))
    check(st, f"{what}(tokens={tokens}, top_k={top_k}, hidden={hidden}, experts={num_experts})")
    _count(3 if need else 1)
    return xs, offsets, slots


def moe_combine(ys, slots, weights=None, out=None):
    """y[t] = sum over j of weights[t, j] * ys[slots[t, j]], summed in fp32 in the order of j.

    ys [rows, hidden]; slots int32 [tokens, top_k] as `moe_sort` returns them (a slot outside [0, rows) adds nothing, a token
    without any gets zeros); weights [tokens, top_k] of ys's type or float32, None for all ones."""
    what = "moe_combine"
    if _EXT is not None:
        return compiled(_EXT.moe_combine, ys, slots, weights, out)
    code = type_of(what, "ys", ys)
    check_rows(what, ys=ys)
    _check_slots(what, slots, ys.device)
    wcode = code if weights is None else _check_weights(what, weights, slots, ys)
    (rows, hidden), (tokens, top_k) = ys.shape, slots.shape
    y = check_out(what, "out", out, (tokens, hidden), ys)
    with _on_device(ys):
        st = LIB.qm_moe_combine(ys.data_ptr(), code, pitch(ys), rows, slots.data_ptr(), None if weights is None else weights.data_ptr(), wcode,
                                y.data_ptr(), pitch(y), tokens, top_k, hidden, _stream_of(ys))
    check(st, f"{what}(tokens={tokens}, top_k={top_k}, hidden={hidden}, rows={rows})")
    _count(int(y.numel() > 0))
    return y


def moe_sort_grad(dxs, slots, out=None):
    """The gradient of moe_sort with respect to x: dx[t] = sum over j of dxs[slots[t, j]]."""
    return moe_combine(dxs, slots, None, out=out)


def moe_combine_grad(dy, ys, slots, weights, out=None):
    """The gradients of moe_combine -> (dys, dweights): dys[slots[t, j]] = weights[t, j] * dy[t] and
    dweights[t, j] = <dy[t], ys[slots[t, j]]> (0 for a slot outside [0, rows)), of the weights' type.

    The slots within [0, rows) must differ from one another, as those of `moe_sort` do.  Rows of dys that no slot names are left
    as they were in `out` (and undefined in a dys that is allocated here)."""
    what = "moe_combine_grad"
    if _EXT is not None:
        return compiled(_EXT.moe_combine_grad, dy, ys, slots, weights, out)
    torch = _torch()
    code = type_of(what, "dy", dy)
    if type_of(what, "ys", ys) != code:
        raise TypeError(f"{what}: dy is {dy.dtype}, ys is {ys.dtype}")
    check_rows(what, dy=dy, ys=ys)
    _check_slots(what, slots, ys.device)
    wcode = _check_weights(what, weights, slots, ys)
    (rows, hidden), (tokens, top_k) = ys.shape, slots.shape
    if tuple(dy.shape) != (tokens, hidden):
        raise ValueError(f"{what}: dy has shape {tuple(dy.shape)}, expected {(tokens, hidden)}")
    dys = check_out(what, "out", out, (rows, hidden), ys)
    dweights = torch.empty_like(weights)
    with _on_device(ys):
        st = LIB.qm_moe_combine_grad(dy.data_ptr(), pitch(dy), ys.data_ptr(), pitch(ys), code, rows, slots.data_ptr(), weights.data_ptr(), wcode,
                                     dys.data_ptr(), pitch(dys), dweights.data_ptr(), tokens, top_k, hidden, _stream_of(ys))
    check(st, f"{what}(tokens={tokens}, top_k={top_k}, hidden={hidden}, rows={rows})")
    _count(int(dweights.numel() > 0))
    return dys, dweights


def moe_linear_w4(x, expert_ids, weights, b, scales, group: int = 128):
    """One projection of a mixture of experts with 4-bit weights: y[t] = sum over j of weights[t, j] * (x[t] @ w_e^T) with
    e = expert_ids[t, j]; assignments whose id is outside [0, experts) add nothing.  moe_sort, moe_gemm_w4 and moe_combine in turn."""
    if b.dim() != 3:
        raise ValueError("moe_linear_w4: b must be [experts, n, k/2]")
    xs, offsets, slots = moe_sort(x, expert_ids, b.shape[0])
    return moe_combine(moe_gemm_w4(xs, b, scales, offsets, group), slots, weights)
