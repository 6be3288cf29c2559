"""Results of 8-bit products whose tiles end after an odd number of stores: the block of shared memory that the next tile begins with
must not be overwritten while the last store reads it. The order of blocks and waits on the CPU, and such shapes on the GPU."""
import os
import subprocess

import pytest
import torch

from codegendemo_b200.kcg import matmul_op
from tests.test_matmul_fp8 import _plan, check, operand, wide64

TESTS = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("columns", [64, 32])  # 16-bit and fp32 results
def test_no_block_is_overwritten_while_a_store_reads_it(columns, tmp_path):
    kernels = os.path.join(os.path.dirname(TESTS), "codegendemo_b200", "csrc", "kernels")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I" + kernels, "-o", str(tmp_path / "check"), os.path.join(TESTS, "store_blocks_check.cpp")],
                   check=True)
    r = subprocess.run([str(tmp_path / "check"), str(columns)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "OK\n", r.stdout


# Many tiles a pair and one block of K, the shortest walk between two tiles' stores: widths of 32, 64 and 96 past a multiple of 128
MANY = [(20000, 352, 128), (20000, 320, 128), (60000, 64, 128), (16000, 416, 100), (30000, 1120, 128), (9000, 2336, 128)]


def test_the_shapes_reach_the_kernel():
    assert {_plan(*s, b)[0] for s in MANY for b in (1, 128)} == {1}


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("m,n,k", MANY)
def test_tiles_of_an_odd_number_of_stores(m, n, k, block_b):
    for out in (torch.bfloat16, torch.float32, torch.float16):
        check(m, n, k, block_b, out)


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
def test_the_same_bits_every_time(block_b):
    m, n, k = 30000, 352, 128
    a, sa = operand(m, k, 1, 2)
    b, sb = operand(n, k, block_b, 3)
    first = matmul_op.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    a64, b64 = wide64(a, sa, 1), wide64(b, sb, block_b)
    assert bool(((first.double() - a64 @ b64.t()).abs() <= 2.0 ** -16 * (a64.abs() @ b64.abs().t())).all())
    for _ in range(50):
        assert torch.equal(matmul_op.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32), first)
