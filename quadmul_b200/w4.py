"""Products of 16-bit activations with packed 4-bit weights that carry one scale per row and group, and their quantiser.

  quantize_w4(w)              weights -> (packed codes, scales): the layout of `pack`, one scale per `group` elements of a row
  gemm_w4(x, b, scales)       x @ dequantised(b)^T
  moe_gemm_w4(x, b, ...)      the same with one matrix per expert over rows sorted by expert (moe.moe_sort)

The reference has no counterpart: its only product is s4 x s4.  Sums are fp32.  The packed weights carry no gradient, and the
products are not recorded by autograd: an input that requires a gradient is refused while gradients are enabled.  An `out` must
not share elements with the inputs.
"""
from __future__ import annotations

from . import _EXT, _count, _on_device, _stream_of, _torch
from ._lib import LIB, QM_TYPE_BF16, QM_TYPE_F16, QM_TYPE_F32, QuadmulError, check

GROUPS = (32, 64, 128, 256)


def compiled(call, *args):
    """A call of the compiled binding, which checks as the ctypes form does; its status errors become QuadmulError."""
    try:
        return call(*args)
    except RuntimeError as exc:
        if type(exc) is not RuntimeError:  # torch's own, such as out of memory
            raise
        raise QuadmulError(-1, str(exc).split("\n")[0]) from exc


def type_of(what: str, name: str, t, allowed=None) -> int:
    """The library's code of a floating tensor's element type."""
    torch = _torch()
    code = {torch.float32: QM_TYPE_F32, torch.float16: QM_TYPE_F16, torch.bfloat16: QM_TYPE_BF16}.get(t.dtype)
    if code is None or (allowed is not None and code not in allowed):
        raise TypeError(f"{what}: {name} is {t.dtype}")
    return code


def check_sizes(what: str, name: str, shape) -> None:
    """The library takes sizes as 32-bit ints, and ctypes would drop what is above them."""
    if any(size >= 1 << 31 for size in shape):
        raise ValueError(f"{what}: {name} is too large")


def check_rows(what: str, **tensors) -> None:
    """2-D CUDA tensors of one device whose rows are contiguous; none that autograd would have to record."""
    torch = _torch()
    device = None
    for name, t in tensors.items():
        if not t.is_cuda:
            raise ValueError(f"{what}: {name} must be a CUDA tensor (there is no CPU path)")
        if device is not None and t.device != device:
            raise ValueError(f"{what}: all tensors must be on one device")
        device = t.device
        if t.dim() != 2:
            raise ValueError(f"{what}: {name} must have two dimensions")
        if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
            raise ValueError(f"{what}: the rows of {name} must be contiguous and must not overlap")
        check_sizes(what, name, t.shape)
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: {name} requires a gradient, which this call does not record")


def check_whole(what: str, device, **tensors) -> None:
    torch = _torch()
    for name, t in tensors.items():
        if not t.is_cuda or t.device != device:
            raise ValueError(f"{what}: {name} must be a CUDA tensor on {device}")
        if not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: {name} requires a gradient, which this call does not record")


def pitch(t) -> int:
    """Elements from one row to the next."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _workspace(x, b, experts, n):
    """(the tensor or None, its pointer, its bytes) for operands that the kernels cannot address as they are."""
    torch = _torch()
    need = LIB.qm_gemm_w4_workspace_bytes(x.data_ptr(), pitch(x), b.data_ptr(), experts, x.shape[0], n, x.shape[1])
    if not need:
        return None, None, 0
    space = torch.empty(need, dtype=torch.uint8, device=x.device)
    return space, space.data_ptr(), need


def _product_launches(x, b, experts, n) -> int:
    """The product's kernel and the copies in front of it."""
    (rows, k) = x.shape
    if not (rows and n and experts):
        return 0
    if not k:
        return 1
    return 1 + bool(k % 32 or pitch(x) % 8 or x.data_ptr() % 16) + bool(k % 32 or b.data_ptr() % 16)


def check_out(what: str, name: str, out, shape, like):
    torch = _torch()
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if out.dtype != like.dtype:
        raise TypeError(f"{what}: {name} is {out.dtype}, expected {like.dtype}")
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} has shape {tuple(out.shape)}, expected {tuple(shape)}")
    check_rows(what, **{"x": like, name: out})
    return out


def _check_weights(what, x, b, scales, group, lead):
    torch = _torch()
    code = type_of(what, "x", x, (QM_TYPE_F16, QM_TYPE_BF16))
    check_rows(what, x=x)
    check_whole(what, x.device, b=b, scales=scales)
    if b.dtype not in (torch.int8, torch.uint8):
        raise TypeError(f"{what}: b must be int8 or uint8, two codes per byte")
    scode = type_of(what, "scales", scales, (code, QM_TYPE_F32))
    if group not in GROUPS:
        raise ValueError(f"{what}: group must be one of {GROUPS}")
    k = x.shape[1]
    if k % 2:
        raise ValueError(f"{what}: k must be even")
    if b.dim() != 2 + len(lead) or tuple(b.shape[:-2]) != lead or b.shape[-1] != k // 2:
        raise ValueError(f"{what}: b has shape {tuple(b.shape)}, x has {k} columns")
    check_sizes(what, "b", b.shape)
    n = b.shape[-2]
    if tuple(scales.shape) != (*lead, n, -(-k // group)):
        raise ValueError(f"{what}: scales have shape {tuple(scales.shape)}, expected {(*lead, n, -(-k // group))}")
    return code, scode, n, k


def gemm_w4(x, b, scales, group: int = 128, out=None):
    """out[m, n] = x[m, k] @ w^T with w[c, i] = scales[c, i // group] * code(b)[c, i].

    x: float16 or bfloat16, rows contiguous (a column slab of a wider tensor is fine); b: packed codes [n, k/2] as `pack` and
    `quantize_w4` write them; scales [n, ceil(k / group)]: x's type or float32; group: 32, 64, 128 or 256.  Returns out, of x's
    type (allocated when not passed in).  Sums are fp32.  With up to 8 rows (experts: 6 on average) x is read to 22 bits below the largest of its neighbours
    under one scale (a row that would lose more than a few elements' digits by that is summed as it is); with more rows, or where 8
    rows of k elements do not fit the kernel for few rows, a weight is rounded to x's type before it is multiplied.
    k a multiple of 32 and rows of x and b on 16-byte boundaries are fastest: others are copied first.  Asynchronous on the
    current stream of x's device."""
    what = "gemm_w4"
    if _EXT is not None:
        return compiled(_EXT.gemm_w4, x, b, scales, group, out)
    code, scode, n, k = _check_weights(what, x, b, scales, group, ())
    m = x.shape[0]
    out = check_out(what, "out", out, (m, n), x)
    with _on_device(x):
        space, ptr, size = _workspace(x, b, 1, n)
        st = LIB.qm_gemm_w4(x.data_ptr(), code, pitch(x), b.data_ptr(), scales.data_ptr(), scode, group, out.data_ptr(), pitch(out), m, n, k, ptr,
                            size, _stream_of(x))
    check(st, f"{what}(m={m}, n={n}, k={k}, group={group})")
    _count(_product_launches(x, b, 1, n))
    return out


def moe_gemm_w4(x, b, scales, offsets, group: int = 128, out=None):
    """out[r] = x[r] @ w_e^T for the rows offsets[e] <= r < offsets[e + 1] of every expert e.

    x: [rows, k] sorted by expert; b [experts, n, k/2] and scales [experts, n, ceil(k / group)] as in gemm_w4; offsets: int32
    [experts + 1] on the device, as `moe_sort` returns them.  Rows that belong to no expert are left as they were in `out` (and
    undefined in an `out` that is allocated here).  The launch does not depend on the values of offsets."""
    what = "moe_gemm_w4"
    if _EXT is not None:
        return compiled(_EXT.moe_gemm_w4, x, b, scales, offsets, group, out)
    torch = _torch()
    if b.dim() != 3:
        raise ValueError(f"{what}: b must be [experts, n, k/2]")
    experts = b.shape[0]
    code, scode, n, k = _check_weights(what, x, b, scales, group, (experts,))
    check_whole(what, x.device, offsets=offsets)
    if offsets.dtype != torch.int32 or tuple(offsets.shape) != (experts + 1,):
        raise ValueError(f"{what}: offsets must be int32 of experts + 1 elements")
    rows = x.shape[0]
    out = check_out(what, "out", out, (rows, n), x)
    with _on_device(x):
        space, ptr, size = _workspace(x, b, experts, n)
        st = LIB.qm_moe_gemm_w4(x.data_ptr(), code, pitch(x), b.data_ptr(), scales.data_ptr(), scode, group, offsets.data_ptr(), experts,
                                out.data_ptr(), pitch(out), rows, n, k, ptr, size, _stream_of(x))
    check(st, f"{what}(rows={rows}, n={n}, k={k}, experts={experts}, group={group})")
    _count(_product_launches(x, b, experts, n))
    return out


def quantize_w4(w, group: int = 128, scale_dtype=None):
    """w [n, k] (float32, float16 or bfloat16) -> (packed codes [n, k/2] int8, scales [n, ceil(k / group)]).

    Per group of a row: scale = max |w| times the float32 value of 1/7, rounded to scale_dtype (w's type by default, or float32);
    code = w / scale rounded to the nearest integer, ties to even, within [-8, 7].  A group of zeros has scale 0; a group that
    holds an infinity or a NaN has a scale that is not finite and codes 0."""
    what = "quantize_w4"
    torch = _torch()
    scale_dtype = w.dtype if scale_dtype is None else scale_dtype
    if scale_dtype not in (w.dtype, torch.float32):
        raise TypeError(f"{what}: scale_dtype must be {w.dtype} or torch.float32")
    if _EXT is not None:
        return compiled(_EXT.quantize_w4, w, group, scale_dtype == torch.float32)
    code = type_of(what, "w", w)
    check_rows(what, w=w)
    if group not in GROUPS:
        raise ValueError(f"{what}: group must be one of {GROUPS}")
    n, k = w.shape
    if k % 2:
        raise ValueError(f"{what}: k must be even")
    packed = torch.empty((n, k // 2), dtype=torch.int8, device=w.device)
    scales = torch.empty((n, -(-k // group)), dtype=scale_dtype, device=w.device)
    with _on_device(w):
        st = LIB.qm_quantize_w4(w.data_ptr(), code, pitch(w), packed.data_ptr(), scales.data_ptr(), type_of(what, "scales", scales), n, k, group,
                                _stream_of(w))
    check(st, f"{what}(n={n}, k={k}, group={group})")
    _count(int(n > 0 and k > 0))
    return packed, scales
