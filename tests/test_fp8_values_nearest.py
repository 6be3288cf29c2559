"""How far 8-bit values may be from x / scale.

A value is the nearest one to v = x * (1 / scale), both operations rounded to fp32: v is off from x / scale by 2 x 2^-24 of itself (and a
2^-48). Where the nearest value to v is not the nearest to x / scale, the middle between the two lies between v and x / scale, so
no further than that from either, and the distance to x / scale exceeds the nearest value's by at most twice that."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op

TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def grid_of(dtype):
    values = torch.arange(256, dtype=torch.uint8).view(dtype).double()
    return values[torch.isfinite(values)].unique().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("d8", list(TOP), ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("block,transposed", [(1, False), (128, False), (1, True), (128, True)])
def test_values_are_the_nearest_but_for_the_middle_between_two(block, transposed, dtype, d8):
    g = torch.Generator(device="cuda").manual_seed(11)
    x = (0.02 * torch.randn(1029, 1376, generator=g, device="cuda")).to(dtype)
    q, s = matmul_op.quantize_fp8(x, rows=block, transposed=transposed, dtype=d8)
    x64 = (x.t() if transposed else x).double()
    r, c = x64.shape
    blocks = torch.zeros((s.shape[0] * block, s.shape[1] * 128), dtype=torch.float64, device="cuda")
    blocks[:r, :c] = x64
    top = blocks.view(s.shape[0], block, s.shape[1], 128).abs().amax(dim=(1, 3)) / TOP[d8]
    assert bool(((s.double() - top).abs() <= 2.0 ** -24 * top).all())  # one division
    each = s.double().repeat_interleave(128, 1)[:, :c].repeat_interleave(block, 0)[:r]
    t, grid = x64 / each, grid_of(d8)
    above = torch.searchsorted(grid, t.contiguous()).clamp(1, grid.numel() - 1)
    nearest = torch.minimum((grid[above] - t).abs(), (grid[above - 1] - t).abs())
    off = (q.double() - t).abs()
    assert bool((off <= nearest + 2 * (2.0 ** -23 + 2.0 ** -48) * t.abs()).all())
    assert (off > nearest).sum().item() <= 0.005 * off.numel()  # (the middles are few)
