"""The entry points of the 4-bit-weight products and the expert routing reject bad arguments before they touch CUDA (CPU only)."""
import ctypes

import pytest

F32, F16, BF16 = 0, 1, 2
NULL_, SHAPE, ALIGN, WORKSPACE, ARG = 1, 2, 3, 7, 8


@pytest.fixture()
def lib(qm):
    from quadmul_b200 import _lib

    return _lib.LIB


@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(256)
    p.keep = buf
    return (ctypes.addressof(buf) + 15) & ~15


def test_gemm_w4(lib, p):
    def call(X=p, type=BF16, ldx=64, B=p, scales=p, scale_type=BF16, group=64, out=p, ldo=8, m=4, n=8, k=64):
        return lib.qm_gemm_w4(X, type, ldx, B, scales, scale_type, group, out, ldo, m, n, k, None, 0, None)

    assert call(m=0) == 0 and call(n=0) == 0 and call(m=0, X=None, out=None) == 0
    assert call(k=63) == SHAPE and call(m=-1) == SHAPE and call(n=-1) == SHAPE and call(k=-2) == SHAPE
    assert call(ldx=63) == SHAPE and call(ldo=7) == SHAPE
    assert call(type=F32) == ARG and call(type=3) == ARG and call(type=-1) == ARG
    assert call(scale_type=F16) == ARG and call(scale_type=9) == ARG and call(type=F16, scale_type=BF16) == ARG
    for g in (0, -32, 16, 48, 96, 512):
        assert call(group=g) == ARG
    assert call(X=None) == NULL_ and call(B=None) == NULL_ and call(scales=None) == NULL_ and call(out=None) == NULL_
    # operands off 16-byte boundaries, or k no multiple of 32, need room for copies: rows of k rounded up to 32
    size = lib.qm_gemm_w4_workspace_bytes
    assert size(p, 64, p, 1, 4, 8, 64) == 0 and size(p, 64, p, 1, 0, 8, 66) == 0 and size(p, 64, p, 1, 4, 8, 0) == 0
    assert size(p + 2, 64, p, 1, 4, 8, 64) == size(p, 68, p, 1, 4, 8, 64) == 4 * 64 * 2 and size(p, 64, p + 1, 3, 4, 8, 64) == 3 * 8 * 32
    assert size(p, 66, p, 1, 4, 8, 66) == 4 * 96 * 2 + 8 * 48
    assert call(X=p + 2) == WORKSPACE and call(k=62) == WORKSPACE and call(B=p + 1) == WORKSPACE and call(ldx=65) == WORKSPACE
    assert call(n=2**31 - 512, ldo=2**31) == SHAPE
    assert call(k=2**30 - 30, ldx=2**30) == SHAPE and call(k=2**30 - 30, ldx=2**30, m=0) == SHAPE and call(k=2**31 - 2, ldx=2**31) == SHAPE
    assert call(X=p + 1) == ALIGN and call(out=p + 1) == ALIGN and call(scales=p + 1) == ALIGN and call(scales=p + 2, scale_type=F32) == ALIGN


def test_moe_gemm_w4(lib, p):
    def call(X=p, offsets=p, experts=2, rows=4, n=8, k=64, group=64, out=p):
        return lib.qm_moe_gemm_w4(X, BF16, k, p, p, BF16, group, offsets, experts, out, n, rows, n, k, None, 0, None)

    assert call(rows=0) == 0 and call(n=0) == 0 and call(experts=0) == 0
    assert call(offsets=None) == NULL_ and call(offsets=p + 2) == ALIGN and call(experts=-1) == SHAPE and call(rows=-1) == SHAPE
    assert call(group=40) == ARG and call(X=None) == NULL_ and call(out=None) == NULL_ and call(k=7) == SHAPE


def test_quantize_w4(lib, p):
    def call(W=p, type=F32, ldw=64, packed=p, scales=p, scale_type=F32, rows=4, k=64, group=64):
        return lib.qm_quantize_w4(W, type, ldw, packed, scales, scale_type, rows, k, group, None)

    assert call(rows=0) == 0 and call(k=0) == 0
    assert call(k=63) == SHAPE and call(rows=-1) == SHAPE and call(ldw=62) == SHAPE
    assert call(type=5) == ARG and call(scale_type=BF16) == ARG and call(group=100) == ARG
    assert call(W=None) == NULL_ and call(packed=None) == NULL_ and call(scales=None) == NULL_
    assert call(W=p + 2) == ALIGN and call(scales=p + 2) == ALIGN and call(W=p + 1, type=F16) == ALIGN


def test_moe_sort(lib, p):
    def call(X=p, type=F32, ldx=8, ids=p, id_bytes=8, experts=4, xs=p, ldxs=8, offsets=p, slots=p, tokens=2, top_k=2, hidden=8):
        return lib.qm_moe_sort(X, type, ldx, ids, id_bytes, experts, xs, ldxs, offsets, slots, tokens, top_k, hidden, None, 0, None)

    assert call(tokens=-1) == SHAPE and call(top_k=-1) == SHAPE and call(hidden=-1) == SHAPE and call(experts=-1) == SHAPE and call(experts=4097) == SHAPE
    assert call(tokens=1 << 20, top_k=1 << 12) == SHAPE and call(top_k=4097) == SHAPE and call(ldx=7) == SHAPE and call(ldxs=7) == SHAPE
    assert call(type=4) == ARG and call(id_bytes=2) == ARG
    assert call(offsets=None) == NULL_ and call(slots=None) == NULL_ and call(ids=None) == NULL_ and call(X=None) == NULL_ and call(xs=None) == NULL_
    assert lib.qm_moe_sort_workspace_bytes(16, 8, 64) == 0 and lib.qm_moe_sort_workspace_bytes(1 << 15, 8, 64) > 0
    assert call(tokens=1 << 15, top_k=8) == WORKSPACE
    assert call(offsets=p + 1) == ALIGN and call(slots=p + 2) == ALIGN and call(ids=p + 4) == ALIGN and call(X=p + 2) == ALIGN and call(xs=p + 2) == ALIGN


def test_moe_combine(lib, p):
    def call(ys=p, type=F32, ldys=8, rows=4, slots=p, weights=p, weight_type=F32, y=p, ldy=8, tokens=2, top_k=2, hidden=8):
        return lib.qm_moe_combine(ys, type, ldys, rows, slots, weights, weight_type, y, ldy, tokens, top_k, hidden, None)

    assert call(tokens=0) == 0 and call(hidden=0) == 0
    assert call(tokens=-1) == SHAPE and call(rows=-1) == SHAPE and call(ldys=7) == SHAPE and call(ldy=7) == SHAPE
    assert call(type=7) == ARG and call(weight_type=BF16) == ARG
    assert call(ys=None) == NULL_ and call(slots=None) == NULL_ and call(y=None) == NULL_
    assert call(ys=p + 2) == ALIGN and call(y=p + 2) == ALIGN and call(slots=p + 2) == ALIGN and call(weights=p + 2) == ALIGN


def test_moe_combine_grad(lib, p):
    def call(dy=p, lddy=8, ys=p, ldys=8, type=F32, rows=4, slots=p, weights=p, weight_type=F32, dys=p, lddys=8, dweights=p, tokens=2, top_k=2, hidden=8):
        return lib.qm_moe_combine_grad(dy, lddy, ys, ldys, type, rows, slots, weights, weight_type, dys, lddys, dweights, tokens, top_k, hidden, None)

    assert call(tokens=0) == 0 and call(top_k=0) == 0
    assert call(tokens=-1) == SHAPE and call(rows=-1) == SHAPE and call(ldys=7) == SHAPE and call(lddy=7) == SHAPE and call(lddys=7) == SHAPE
    assert call(type=7) == ARG and call(weight_type=F16) == ARG
    for name in ("dy", "ys", "slots", "weights", "dys", "dweights"):
        assert call(**{name: None}) == NULL_
        assert call(**{name: p + 2}) == ALIGN


def test_python_calls_have_no_cpu_path(qm):
    import torch

    x, b, s = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8, 1, dtype=torch.bfloat16)
    ids, slots = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: qm.gemm_w4(x, b, s), lambda: qm.moe_gemm_w4(x, b[None], s[None], torch.zeros(2, dtype=torch.int32)), lambda: qm.quantize_w4(x),
                 lambda: qm.moe_sort(x, ids, 4), lambda: qm.moe_combine(x, slots), lambda: qm.moe_sort_grad(x, slots),
                 lambda: qm.moe_combine_grad(x, x, slots, torch.zeros(4, 2)), lambda: qm.moe_linear_w4(x, ids, torch.zeros(4, 2), b[None], s[None])):
        with pytest.raises(ValueError):
            call()
