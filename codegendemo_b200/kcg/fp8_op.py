"""The operators of an 8-bit linear layer: the norm in front of it, its 8-bit operands, its product, and what training takes.

``rms_norm`` / ``rms_norm_fp8`` (the residual's addition and the norm; the result in the inputs' type, or as 8-bit values with a scale
for each 128 of a row), ``rms_norm_backward``, ``quantize_fp8`` (weights in blocks of 128 x 128, activations and gradients in blocks of
1 x 128, as they lie or transposed) and ``matmul_fp8``, the product of such operands. The reference names a float8 type
(Runtime/python/kcg/Utils.py, EnumKernelDType) but has no kernel that computes with it.

A linear layer ``y = x w^T`` in 8 bits, and its gradients::

    h8, hs, h = rms_norm_fp8(x, norm_weight, residual)                  # or quantize_fp8(x)
    w8, ws = quantize_fp8(w, rows=128)
    y = matmul_fp8(h8, hs, w8, ws)

    dx = matmul_fp8(*quantize_fp8(dy), *quantize_fp8(w, rows=128, transposed=True))
    dw = matmul_fp8(*quantize_fp8(dy, transposed=True), *quantize_fp8(x, transposed=True), out_dtype=torch.float32)

All work on CUDA tensors of any device, on torch's current stream of that device; results come from torch's allocator. Matrices
are 2-D (tokens x width: a batch of sequences is viewed as its tokens) and may be views with a row pitch (contiguous rows). Like the
other operators of this library these are no autograd functions: results carry no gradient, and a backward pass is made of the
calls above.
"""
import ctypes

from codegendemo_b200 import _lib
from codegendemo_b200.kcg.Utils import DeviceInfo

MAX_NORM_WIDTH = 32768
MAX_SIZE = 2 ** 31 - 256  # rows or columns of an 8-bit matrix

_warm = None  # csrc/kcg_torchcall.cpp once something was launched, False where it was not built for this torch


def _launched(status):
    """The end of a call that went this way: its error, or the next call's shorter way."""
    global _warm
    if status:
        _lib.check(status)
    if _warm is None:
        from codegendemo_b200.kcg import matmul_op
        _warm = matmul_op._warm_calls()


def _dtype_code(t, what):
    import torch
    codes = {torch.float16: 2, torch.float32: 4, torch.bfloat16: 62}
    if t.dtype not in codes:
        raise ValueError(f"{what} must be float16, bfloat16 or float32, not {t.dtype}")
    return codes[t.dtype]


def _fp8_code(dtype, what):
    import torch
    codes = {torch.float8_e4m3fn: 1, torch.float8_e5m2: 2}
    if dtype not in codes:
        raise ValueError(f"{what} must be float8_e4m3fn or float8_e5m2, not {dtype}")
    return codes[dtype]


def _pitch(t, what, like=None, shape=None):
    """Elements between the rows of a matrix whose rows are contiguous; checks it against another's device and type, and a shape."""
    sizes = t.shape
    if len(sizes) != 2 or (sizes[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} must be a 2-D tensor with contiguous rows (a view with a row pitch is fine)")
    if shape is not None and (sizes[0] != shape[0] or sizes[1] != shape[1]):
        raise ValueError(f"{what} must be {shape[0]} x {shape[1]}, not {sizes[0]} x {sizes[1]}")
    if like is not None and (t.device != like.device or t.dtype != like.dtype):
        raise ValueError(f"{what} must be {like.dtype} on {like.device}, not {t.dtype} on {t.device}")
    pitch = t.stride(0) if sizes[0] > 1 else sizes[1]
    if pitch < sizes[1]:
        raise ValueError(f"{what}: rows overlap")
    return pitch


def _device(t, what):
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    return t.device.index or 0


def _norm_operands(x, weight, other, eps, names=("x", "residual")):
    """Checks rows, weight and a second matrix of the rows' shape (or None): device, type, rows, width and the matrices' pitches."""
    dev = _device(x, names[0])
    code = _dtype_code(x, names[0])
    ldx = _pitch(x, names[0])
    rows, width = x.shape
    if not 1 <= width <= MAX_NORM_WIDTH:
        raise ValueError(f"rows must hold 1 to {MAX_NORM_WIDTH} values, not {width}")
    if weight.shape != (width,) or weight.dtype != x.dtype or weight.device != x.device or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous tensor of {width} values, {x.dtype} on {x.device}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be finite and not negative")
    return dev, code, rows, width, ldx, 0 if other is None else _pitch(other, names[1], x, (rows, width))


def _sum_of(x, residual, residual_out):
    """Where x + residual is stored, and its pitch."""
    if residual is None:
        if residual_out is not None:
            raise ValueError("residual_out without a residual")
        return None, 0
    if residual_out is None:
        return x.new_empty(x.shape), 0
    return residual_out, _pitch(residual_out, "residual_out", x, x.shape)


def rms_norm(x, weight, residual=None, eps=1e-6, out=None, residual_out=None):
    """``h / sqrt(mean(h^2) + eps) * weight`` row by row, with ``h = x + residual`` (or x): returns the norm, or (norm, h) with a
    residual. Sums in fp32 (a row whose sum of squares passes 3.4e38 gives zeros), each result rounded once (the norm is taken of
    the unrounded sum). ``x`` and ``residual`` are rows x width, fp16, bf16 or fp32, ``weight`` width values of the same type. ``out``
    and ``residual_out`` take the results; each may be ``x`` or ``residual`` itself (not both the same one), other overlaps are not allowed."""
    if _warm and out is None and residual_out is None:
        results = _warm.rms_norm(x, weight, residual, eps)
        if results is not None:
            return results
    dev, code, rows, width, ldx, ldr = _norm_operands(x, weight, residual, eps)
    ldy = 0
    if out is None:
        out = x.new_empty((rows, width))
    else:
        ldy = _pitch(out, "out", x, (rows, width))
    h, ldh = _sum_of(x, residual, residual_out)
    if h is not None and h.data_ptr() == out.data_ptr() and rows > 0:
        raise ValueError("out and residual_out must be different tensors")
    _launched(_lib.get_lib().kcg_rms_norm(dev, DeviceInfo.get_cuda_stream(dev), x.data_ptr(), ldx,
                                          0 if residual is None else residual.data_ptr(), ldr, weight.data_ptr(), out.data_ptr(), ldy,
                                          0 if h is None else h.data_ptr(), ldh, rows, width, eps, code))
    return out if h is None else (out, h)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6, residual_out=None):
    """``rms_norm`` whose result leaves in 8 bits, blocks of 1 x 128 of the unrounded norm as in ``quantize_fp8``: returns (values, scales),
    or (values, scales, h) with a residual. Scales are off by a few units of fp32's last place, as the norm itself is; a value that lies as
    near the middle between two 8-bit ones may become either, and may become the other one where the rows lie at another alignment."""
    if _warm and residual_out is None:
        results = _warm.rms_norm_fp8(x, weight, residual, eps)
        if results is not None:
            return results
    import torch
    dev, code, rows, width, ldx, ldr = _norm_operands(x, weight, residual, eps)
    q = _rows_of_fp8(x, rows, width, torch.float8_e4m3fn)
    scales = x.new_empty((rows, -(-width // 128)), dtype=torch.float32)
    h, ldh = _sum_of(x, residual, residual_out)
    if rows > 0:
        _launched(_lib.get_lib().kcg_rms_norm_fp8(dev, DeviceInfo.get_cuda_stream(dev), x.data_ptr(), ldx,
                                                  0 if residual is None else residual.data_ptr(), ldr, weight.data_ptr(), q.data_ptr(),
                                                  -(-width // 16) * 16, scales.data_ptr(), 0 if h is None else h.data_ptr(), ldh, rows,
                                                  width, eps, code))
    return (q, scales) if h is None else (q, scales, h)


def _rows_of_fp8(like, rows, cols, dtype):
    """An 8-bit matrix whose rows start on 16-byte boundaries, as the products want them."""
    pitch = -(-cols // 16) * 16
    q = like.new_empty((rows, pitch), dtype=dtype)
    return q if pitch == cols else q[:, :cols]


def rms_norm_backward(dy, h, weight, eps=1e-6, dh=None):
    """Gradients of ``rms_norm`` at ``h`` (x, or x + residual): returns (dx, dweight) for the gradient ``dy`` of its result. ``dh``, the
    gradient that reaches h past the norm, is added to dx, which then is the gradient of both x and the residual. The order of
    dweight's sums is fixed by the shape and the device."""
    if _warm:
        results = _warm.rms_norm_backward(dy, h, weight, eps, dh)
        if results is not None:
            return results
    dev, code, rows, width, ldh, lddy = _norm_operands(h, weight, dy, eps, ("h", "dy"))
    lddh = 0 if dh is None else _pitch(dh, "dh", h, (rows, width))
    dx = h.new_empty((rows, width))
    if rows == 0:
        return dx, weight.new_zeros(width)
    import torch
    dw = weight.new_empty(width)
    lib = _lib.get_lib()
    size = lib.kcg_rms_norm_backward_workspace(dev, rows, width)
    workspace = h.new_empty(max(size, 16), dtype=torch.uint8)
    _launched(lib.kcg_rms_norm_backward(dev, DeviceInfo.get_cuda_stream(dev), dy.data_ptr(), lddy, h.data_ptr(), ldh, weight.data_ptr(),
                                        0 if dh is None else dh.data_ptr(), lddh, dx.data_ptr(), 0, dw.data_ptr(), workspace.data_ptr(),
                                        size, rows, width, eps, code))
    return dx, dw


def quantize_fp8(x, rows=1, transposed=False, dtype=None):
    """(values, scales) of a matrix in blocks of ``rows`` (1 or 128) x 128 values: scale = max(largest magnitude / 448, 2^-126) (e5m2:
    57344), values x * (1 / scale): reciprocal and product rounded to fp32, then to the nearest 8-bit value, ties to even (x / scale may
    give the neighbour where it lies within 2^-23 of itself of the middle between two). ``transposed``: of ``x.t()``, cut into blocks
    along what were x's rows.
    ``dtype`` is float8_e4m3fn (default) or float8_e5m2. Scales are (row blocks) x ceil(columns / 128), fp32."""
    if _warm and dtype is None:
        results = _warm.quantize_fp8(x, rows, transposed)
        if results is not None:
            return results
    import torch
    dev = _device(x, "x")
    code = _dtype_code(x, "x")
    ldx = _pitch(x, "x")
    if rows not in (1, 128):
        raise ValueError(f"blocks have 1 or 128 rows, not {rows}")
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    code8 = _fp8_code(dtype, "dtype")
    n, cols = x.shape
    if max(n, cols) > MAX_SIZE:
        raise ValueError(f"x has more than {MAX_SIZE} rows or columns")
    r, c = (cols, n) if transposed else (n, cols)
    q = _rows_of_fp8(x, r, c, dtype)
    scales = x.new_empty((-(-r // rows), -(-c // 128)), dtype=torch.float32)
    if n > 0 and cols > 0:
        _launched(_lib.get_lib().kcg_quantize_fp8(dev, DeviceInfo.get_cuda_stream(dev), x.data_ptr(), ldx, q.data_ptr(), -(-c // 16) * 16,
                                                  scales.data_ptr(), n, cols, rows, int(bool(transposed)), code, code8))
    return q, scales


def matmul_fp8(a, a_scale, b, b_scale, c=None, beta=0.0, bias=None, relu=False, out_dtype=None):
    """``c = act(a @ b.t() + beta * c + bias)`` of 8-bit operands as ``quantize_fp8`` makes them: ``a`` is M x K in blocks of 1 x 128 with
    ``a_scale`` M x ceil(K / 128); ``b`` is N x K (a weight as linear layers keep it) in blocks of 128 x 128, ``b_scale``
    ceil(N / 128) x ceil(K / 128), or of 1 x 128, ``b_scale`` N x ceil(K / 128). e4m3 or e5m2, each its own. Sums in fp32, one rounding
    to ``out_dtype`` (bf16 by default; fp16, fp32) or c's type. Rows of a and b have to start on 16-byte boundaries, as
    ``quantize_fp8`` and ``rms_norm_fp8`` lay them out. ReLU leaves a NaN one. Scales may reach 2^88 (values of 1e29), and the product
    of two, but for blocks of zeros, has to be a normal fp32 number."""
    if _warm and c is None and type(beta) is float and beta == 0.0:
        c = _warm.matmul_fp8(a, a_scale, b, b_scale, bias, relu, out_dtype)
        if c is not None:
            return c
    import torch
    dev = _device(a, "a")
    fa, fb = _fp8_code(a.dtype, "a"), _fp8_code(b.dtype, "b")
    lda, ldb = _pitch(a, "a"), _pitch(b, "b")
    M, K = a.shape
    N, K2 = b.shape
    if K != K2:
        raise ValueError(f"a has rows of {K} values, b of {K2}")
    if max(M, N, K) > MAX_SIZE:
        raise ValueError(f"an operand has more than {MAX_SIZE} rows or columns")
    if N < 1 or K < 1:
        raise ValueError("a product of no columns, or of rows without values")
    kb = -(-K // 128)
    if b_scale.shape[:1] == (N,) and N > 1:
        block_b = 1
    else:
        block_b = 128
    for t, what, shape in ((a_scale, "a_scale", (M, kb)), (b_scale, "b_scale", (N if block_b == 1 else -(-N // 128), kb))):
        if t.dtype != torch.float32 or t.device != a.device:
            raise ValueError(f"{what} must be float32 on {a.device}")
        _pitch(t, what, None, shape)
    if b.device != a.device:
        raise ValueError(f"b must be on {a.device}")
    if c is None:
        if beta != 0.0:
            raise ValueError("beta != 0 needs the c to scale")
        c = a.new_empty((M, N), dtype=torch.bfloat16 if out_dtype is None else out_dtype)
    elif out_dtype is not None and c.dtype != out_dtype:
        raise ValueError(f"c is {c.dtype}, out_dtype {out_dtype}")
    ldc = _pitch(c, "c", None, (M, N))
    if c.device != a.device:
        raise ValueError(f"c must be on {a.device}")
    code = _dtype_code(c, "c")
    if bias is not None and (bias.shape != (N,) or bias.dtype != c.dtype or bias.device != a.device or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous tensor of {N} values, {c.dtype} on {a.device}")
    if M == 0:
        return c
    p = _lib.Fp8Product(a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(), c.data_ptr(),
                        0 if bias is None else bias.data_ptr(), lda, _pitch(a_scale, "a_scale"), ldb, _pitch(b_scale, "b_scale"), ldc,
                        M, N, K, block_b, fa, fb, code, beta, int(bool(relu)))
    _launched(_lib.get_lib().kcg_matmul_fp8(dev, DeviceInfo.get_cuda_stream(dev), ctypes.byref(p)))
    return c


def matmul_fp8_status(device: int = 0) -> None:
    """Synchronises the device and raises if a bounded wait of an 8-bit product ran out."""
    out = (ctypes.c_uint32 * 4)()
    _lib.check(_lib.get_lib().kcg_matmul_fp8_status(int(device), out))
