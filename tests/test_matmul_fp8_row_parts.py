"""Operands that are parts of wider matrices whose other values are NaN: K ends anywhere in 16 bytes, in a block and in a tile, rows and
scales end anywhere, and nothing past them may come in."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op
from tests.test_matmul_fp8 import E4, E5, operand

NAN_BYTE = {E4: 0x7f, E5: 0x7f}


def inside(q, rows_more, cols_more):
    """q as the first rows and columns of a matrix of NaN."""
    r, c = q.shape
    pitch = -(-(c + cols_more) // 16) * 16
    wide = torch.full((r + rows_more, pitch), NAN_BYTE[q.dtype], dtype=torch.uint8, device="cuda")
    wide[:r, :c] = q.view(torch.uint8)
    return wide.view(q.dtype)[:r, :c]


def scales_inside(s):
    wide = torch.full((s.shape[0] + 2, s.shape[1] + 3), float("nan"), device="cuda")
    wide[:s.shape[0], :s.shape[1]] = s
    return wide[:s.shape[0], :s.shape[1]]


@pytest.mark.gpu
@pytest.mark.parametrize("fa,fb", [(E4, E4), (E5, E4)], ids=str)
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("m,n", [(1, 300), (7, 130), (20, 1000), (40, 257), (200, 300), (2049, 2305)])
def test_nothing_past_the_operands_comes_in(m, n, block_b, fa, fb):
    for k in (1, 7, 15, 16, 17, 100, 120, 127, 129, 250, 255, 263, 520, 1025, 2047):
        a, sa = operand(m, k, 1, 0, fa)
        b, sb = operand(n, k, block_b, 1, fb)
        clean = lambda q: torch.zeros((q.shape[0], -(-q.shape[1] // 16) * 16), dtype=torch.uint8, device="cuda")  # noqa: E731
        za, zb = clean(a), clean(b)
        za[:, :k], zb[:, :k] = a.view(torch.uint8), b.view(torch.uint8)
        want = matmul_op.matmul_fp8(za.view(fa)[:, :k], sa, zb.view(fb)[:, :k], sb, out_dtype=torch.float32)
        assert bool(torch.isfinite(want).all())
        for more in (1, 40):
            got = matmul_op.matmul_fp8(inside(a, more, more), scales_inside(sa), inside(b, more, more), scales_inside(sb), out_dtype=torch.float32)
            assert torch.equal(got, want), (k, more)
    matmul_op.matmul_fp8_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,width", [(3, 7), (5, 129), (9, 1000), (70, 333), (3, 4097), (2, 16390)])
def test_nothing_past_the_rows_comes_in(rows, width, dtype):
    """The same of the norm, its gradient and the quantisation."""
    g = torch.Generator(device="cuda").manual_seed(rows + width)

    def make(seed):
        x = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
        wide = torch.full((rows + 2, width + 24), float("nan"), dtype=dtype, device="cuda")
        wide[:rows, 8:8 + width] = x
        return x, wide[:rows, 8:8 + width]
    (x, xw), (r, rw), (d, dw) = make(0), make(1), make(2)
    w = torch.randn(width, generator=g, device="cuda").to(dtype)
    same = lambda p, q: torch.equal(p.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))  # noqa: E731
    for f in (lambda x, r, d: matmul_op.quantize_fp8(x), lambda x, r, d: matmul_op.quantize_fp8(x, rows=128),
              lambda x, r, d: matmul_op.quantize_fp8(x, transposed=True), lambda x, r, d: matmul_op.quantize_fp8(x, rows=128, transposed=True)):
        assert all(same(p, q) for p, q in zip(f(x, r, d), f(xw, rw, dw)))
    for f in (lambda x, r, d: matmul_op.rms_norm(x, w, r), lambda x, r, d: matmul_op.rms_norm_backward(d, x, w, dh=r),
              lambda x, r, d: [t.float() for t in matmul_op.rms_norm_fp8(x, w, r)]):
        assert all(bool(torch.isfinite(q).all()) for q in f(xw, rw, dw))
