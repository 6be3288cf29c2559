"""The norm into 8 bits where a row's value times its weight leaves the range of fp32, and the norm itself does not.

Tolerances are those of tests/test_rms_norm.py: the products (h r) w, each rounded once, are among the roundings counted there. Below
2^-126, where fp32's numbers lie 2^-149 apart, the last of them is off by half of that instead of a share of itself. Its block's scale is
2^-126 then, whose reciprocal, and the product with it, are exact: half a step of e4m3 and 2^-150 are allowed. A norm past fp32's largest
number is an infinity: its block's scale is one too, the block's other values 0 and itself a NaN."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op
from tests.test_rms_norm import U, near, norm64, rows_of

LARGEST = torch.finfo(torch.float32).max


def near_fp8(q, scales, want, relative=80 * U):
    r, c = want.shape
    nb = -(-c // 128)
    assert scales.shape == (r, nb) and q.shape == (r, c) and q.dtype == torch.float8_e4m3fn
    full = torch.zeros((r, nb * 128), dtype=torch.float64, device=want.device)
    full[:, :c] = want
    top = full.view(r, nb, 128).abs().amax(dim=2)
    assert torch.equal(torch.isinf(scales), top > LARGEST)
    s = (top / 448).clamp(min=2.0 ** -126)
    assert bool(((scales.double() - s).abs() <= (relative + 4 * U) * s)[top <= LARGEST].all())
    past = (top > LARGEST).repeat_interleave(128, 1)[:, :c]
    q = q.double()
    assert torch.equal(torch.isnan(q), want.abs() > LARGEST) and bool((q[past & ~torch.isnan(q)] == 0).all())
    s = scales.double().repeat_interleave(128, 1)[:, :c]
    allowed = s * torch.maximum(want.abs() / s * 2.0 ** -4, torch.full_like(s, 2.0 ** -10)) * (1 + 1e-5) + 2 * relative * want.abs() + 2.0 ** -150
    assert bool(((q * s - want).abs() <= allowed)[~past].all())


@pytest.mark.gpu
@pytest.mark.parametrize("width", [129, 256, 1000, 2048, 5504, 16384])
@pytest.mark.parametrize("rows_at,weight_at", [(1e15, 1e25), (1e-15, 1e-28), (1e-10, 1e-29), (1e15, 1e-40), (1e-15, 1e30), (1.0, 3e37)])
def test_products_of_value_and_weight_outside_the_range_of_fp32(width, rows_at, weight_at):
    """All weights, and those of every other block of 128 (the others are of order 1): a block is taken by itself. No eps: the
    smallest rows would drown in it."""
    x, w = rows_of(5, width, torch.float32, 1, rows_at), rows_of(1, width, torch.float32, 2)[0]
    x[2] = 0.5 * x[2].abs().max()  # no spread: every value the largest of its block, up to its weight
    every = w * weight_at
    other = torch.where(torch.arange(width, device="cuda") // 128 % 2 == 0, every, w)
    for weight in (every, other):
        want = norm64(x.double(), weight, 0.0)
        near_fp8(*matmul_op.rms_norm_fp8(x, weight, eps=0.0), want)
        y, past = matmul_op.rms_norm(x, weight, eps=0.0), want.abs() > LARGEST
        assert torch.equal(torch.isinf(y), past)
        near(y[~past], want[~past], torch.float32)
        r = rows_of(5, width, torch.float32, 3, rows_at)
        h64 = x.double() + r.double()
        q, s, h = matmul_op.rms_norm_fp8(x, weight, r, eps=0.0)
        near(h, h64, torch.float32, 2.0 ** -24)
        near_fp8(q, s, norm64(h64, weight, 0.0))
