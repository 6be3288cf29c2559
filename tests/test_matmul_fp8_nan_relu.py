"""ReLU of an 8-bit product leaves NaN in place, whichever kernel and epilogue a value takes: a NaN in a row of a, a row of b, the bias, the C
that is added."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op
from tests.test_matmul_fp8 import _plan

SHAPES = [(7, 512, 1024), (60, 300, 640), (200, 512, 1024), (2304, 2304, 256)]


def test_the_shapes_reach_every_kernel():
    assert {tuple(_plan(*s, 1)[:3]) for s in SHAPES} == {(0, 1, 16), (0, 1, 64), (0, 0, 128), (1, 0, 256)}
    assert {tuple(_plan(*s, 128)[:2]) for s in SHAPES} == {(0, 1), (0, 0), (1, 0)}


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_nan_passes_relu(m, n, k, block_b, out):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x, w = torch.randn(m, k, generator=g, device="cuda"), torch.randn(n, k, generator=g, device="cuda")
    bias, c = torch.randn(n, generator=g, device="cuda").to(out), torch.randn(m, n, generator=g, device="cuda").to(out)
    x[1, 3], bias[5], c[3, 9] = float("nan"), float("nan"), float("nan")
    if block_b == 1:
        w[11, 7] = float("nan")
    a, b = matmul_op.quantize_fp8(x), matmul_op.quantize_fp8(w, rows=block_b)
    for kw in (dict(), dict(bias=bias), dict(bias=bias, beta=0.5)):
        call = lambda relu: matmul_op.matmul_fp8(*a, *b, out_dtype=out, relu=relu, **kw, **(dict(c=c.clone()) if "beta" in kw else {}))  # noqa: E731
        plain, got = call(False), call(True)
        nan = torch.isnan(plain)
        assert nan[1].all() and (nan[:, 5].all() or not kw) and (nan[3, 9] or "beta" not in kw) and (nan[:, 11].all() or block_b != 1)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[~nan], plain[~nan].clamp(min=0))
    matmul_op.matmul_fp8_status()
