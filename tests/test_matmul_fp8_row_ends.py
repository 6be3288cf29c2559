"""Results of 8-bit products written into part of a wider matrix: what lies past a row's last value stays, wherever in 16 bytes the row ends.
Rows that start on 16-byte boundaries are the case in which a product of many tiles stores by TMA."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op
from tests.test_matmul_fp8 import _plan, check, operand

M, K = {"pairs": 18944, "tiles": 300, "few": 20}, 128


def test_the_shapes_reach_every_kernel():
    for b in (1, 128):
        assert {tuple(_plan(M["pairs"], n, K, b)[:2]) for n in (449, 488, 515)} == {(1, 0)}
        assert _plan(M["tiles"], 483, K, b)[:2] == [0, 0] and _plan(M["few"], 483, K, b)[:2] == [0, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("form", list(M))
def test_what_lies_past_the_rows_stays(form, block_b, out):
    m, each = M[form], 4 if out == torch.float32 else 8  # (values of 16 bytes)
    a, sa = operand(m, K, 1, 0)
    for n in [448 + i for i in range(1, 9)] + [481, 483, 515, 545, 577]:
        b, sb = operand(n, K, block_b, 1)
        want = matmul_op.matmul_fp8(a, sa, b, sb, out_dtype=out)
        for width in (-(-n // each) * each, -(-n // each) * each + 5 * each):
            wide = torch.full((m, width), 7.0, dtype=out, device="cuda")
            matmul_op.matmul_fp8(a, sa, b, sb, c=wide[:, :n])
            assert torch.equal(wide[:, :n], want), n
            assert bool((wide[:, n:] == 7.0).all()), n
    matmul_op.matmul_fp8_status()


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
def test_two_results_side_by_side(block_b):
    """The columns of one matrix by two products, on two streams at once."""
    m, n1, n2 = M["pairs"], 483, 541
    a, sa = operand(m, K, 1, 0)
    b1, b2 = operand(n1, K, block_b, 1), operand(n2, K, block_b, 2)
    want = torch.cat([matmul_op.matmul_fp8(a, sa, *b1), matmul_op.matmul_fp8(a, sa, *b2)], dim=1)
    both, side = torch.zeros((m, n1 + n2), dtype=torch.bfloat16, device="cuda"), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        matmul_op.matmul_fp8(a, sa, *b1, c=both[:, :n1])
        with torch.cuda.stream(side):
            matmul_op.matmul_fp8(a, sa, *b2, c=both[:, n1:])
        torch.cuda.synchronize()
        assert torch.equal(both, want)
        both.zero_()
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("out,pitch", [(torch.bfloat16, 13), (torch.float16, 5), (torch.float32, 1), (torch.float32, 33)])
def test_values_with_every_epilogue(out, pitch, block_b):
    check(M["pairs"], 483, K, block_b, out, pitch=pitch)
    check(9000, 1107, 300, block_b, out, pitch=pitch, beta=0.5, bias=True)
    check(3000, 2307, 520, block_b, out, pitch=pitch, bias=True, relu=True)
