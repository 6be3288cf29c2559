"""Quantisation in blocks against torch's arithmetic on the same definition: a scale is one division, a value one product with the
scale's reciprocal and one rounding, so scales and values are equal bit by bit. (Quotients are taken in 64 bits and rounded to 32, which
is the correctly rounded quotient, 53 >= 2 x 24 + 2; torch divides by a number as a product with its reciprocal.)"""
import pytest
import torch

from codegendemo_b200 import _lib
from codegendemo_b200.kcg import matmul_op

MAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
SHAPES = [(1, 1), (1, 128), (3, 100), (128, 128), (129, 257), (17, 1376), (200, 1008), (127, 5507), (1000, 16), (256, 264)]


def plain(x, rows, transposed, dtype):
    x = (x.t() if transposed else x).float()
    r, c = x.shape
    br, bc = -(-r // rows), -(-c // 128)
    full = torch.zeros((br * rows, bc * 128), device=x.device)
    full[:r, :c] = x
    b = full.view(br, rows, bc, 128)
    s = torch.clamp((b.abs().amax(dim=(1, 3)).double() / torch.full((), MAX[dtype], dtype=torch.float64, device=x.device)).float(), min=2.0 ** -126)
    q = torch.clamp(b * (1.0 / s.double()).float()[:, None, :, None], -MAX[dtype], MAX[dtype]).to(dtype)
    return q.view(torch.uint8).reshape(br * rows, bc * 128)[:r, :c], s


def values(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(2 * torch.randn(1, cols, generator=g, device="cuda"))
    return x.to(dtype)


def same(got, want):
    q, s = got
    return q.shape == want[0].shape and torch.equal(q.view(torch.uint8), want[0]) and torch.equal(s, want[1])


class _OnGpu(torch.Tensor):
    is_cuda = True


def _fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_OnGpu)


@pytest.mark.parametrize("call,message", [
    (lambda: matmul_op.quantize_fp8(torch.zeros(4, 4)), "CUDA"),
    (lambda: matmul_op.quantize_fp8(_fake(4)), "2-D"),
    (lambda: matmul_op.quantize_fp8(_fake(4, 4), rows=64), "1 or 128"),
    (lambda: matmul_op.quantize_fp8(_fake(4, 4, dtype=torch.float64)), "float32"),
    (lambda: matmul_op.quantize_fp8(_fake(4, 4), dtype=torch.int8), "float8"),
    (lambda: matmul_op.quantize_fp8(_fake(4, 8)[:, ::2]), "contiguous rows"),
    (lambda: matmul_op.quantize_fp8(_fake(8, 4).t()), "contiguous rows"),
])
def test_wrong_arguments_are_refused(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_the_c_entry_refuses_what_it_cannot_take():
    lib = _lib.get_lib()

    def call(X=256, ldx=0, Q=256, ldq=128, S=256, rows=4, cols=128, block=1, transposed=0, dtype=62, dtype8=1):
        return lib.kcg_quantize_fp8(0, 0, X, ldx, Q, ldq, S, rows, cols, block, transposed, dtype, dtype8)
    assert call(rows=0) == 0
    for bad in (dict(X=0), dict(Q=0), dict(S=0), dict(ldx=64), dict(ldq=64), dict(ldq=136), dict(Q=264), dict(X=257), dict(S=258),
                dict(block=2), dict(dtype=1), dict(dtype8=3), dict(cols=0), dict(rows=-1), dict(transposed=1, ldq=0)):
        assert call(**bad) == _lib.E_BAD_ARG, bad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("block", [1, 128])
def test_every_shape(block, transposed, dtype):
    for i, (rows, cols) in enumerate(SHAPES):
        x = values(rows, cols, dtype, i)
        for d8 in MAX:
            got = matmul_op.quantize_fp8(x, rows=block, transposed=transposed, dtype=d8)
            assert got[0].dtype == d8 and got[0].stride(0) % 16 == 0
            assert same(got, plain(x, block, transposed, d8)), (rows, cols, d8)


@pytest.mark.gpu
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("block", [1, 128])
def test_zeros_tiny_values_infinities_and_nan(block, transposed):
    x = values(256, 256, torch.float32, 3)
    x[:128, :128] = 0
    x[128:, :128] *= 1e-42   # below the smallest scale's reach: values a small multiple of the 8-bit step, or zero
    clean = plain(x, block, transposed, torch.float8_e4m3fn)
    assert same(matmul_op.quantize_fp8(x, rows=block, transposed=transposed), clean)
    x[200, 200], x[5, 140] = float("inf"), float("nan")
    q, s = matmul_op.quantize_fp8(x, rows=block, transposed=transposed)
    q = q.float()
    if transposed:
        q = q.t()
    assert torch.isnan(q[200, 200]) and torch.isnan(q[5, 140]) and torch.isinf(s).sum() == 1 and torch.isnan(s).sum() == 1
    same_column = torch.isnan(q[5, 128:]).all() if block == 128 or not transposed else torch.isnan(q[:128, 140]).all()
    assert same_column
    finite = torch.isfinite(s)
    assert torch.equal(s[finite], clean[1][finite])


@pytest.mark.gpu
def test_views_and_alignments():
    wide = values(140, 700, torch.bfloat16, 4)
    for c0, c1 in ((8, 264), (3, 300), (0, 700), (1, 129)):
        x = wide[5:, c0:c1]
        for block in (1, 128):
            for transposed in (False, True):
                got = matmul_op.quantize_fp8(x, rows=block, transposed=transposed)
                assert same(got, plain(x, block, transposed, torch.float8_e4m3fn)), (c0, c1, block, transposed)


@pytest.mark.gpu
def test_no_values():
    for shape in ((0, 64), (64, 0)):
        x = torch.empty(shape, device="cuda")
        for transposed in (False, True):
            q, s = matmul_op.quantize_fp8(x, transposed=transposed)
            assert q.shape == (shape[::-1] if transposed else shape) and s.numel() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("block,transposed", [(1, False), (128, False), (1, True)])
def test_offsets_past_32_bits(block, transposed):
    rows, cols = 131328, 16384
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-128:] = values(128, cols, torch.bfloat16, 5)
    q, s = matmul_op.quantize_fp8(x, rows=block, transposed=transposed)
    want = plain(x[-128:], block, transposed, torch.float8_e4m3fn)
    if transposed:
        q, s = q[:, -128:], s[:, -1:]
    else:
        q, s = q[-128:], s[-(128 // block):]
    assert torch.equal(q.contiguous().view(torch.uint8), want[0]) and torch.equal(s, want[1])
