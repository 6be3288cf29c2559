"""fp32 products through fp16 parts behind the kernels that write their operands, into the same memory again and again. The split may be on
the GPU while the kernel before it still writes (programmatic dependent launch): what it reads is not read-only for its life."""
import os

import pytest
import torch

from codegendemo_b200.kcg import matmul_op
from tests.test_f32_split import _kernel
from tests.test_fp8_dependent_launches import SOURCES, non_coherent_loads


def test_no_kernel_asks_for_memory_that_is_read_only_for_its_life():
    """Every kernel of the library may be launched behind one that has not ended."""
    files = [os.path.join(d, f) for d in (SOURCES, os.path.join(SOURCES, "kernels")) for f in sorted(os.listdir(d)) if f.endswith((".cu", ".cuh"))]
    assert len(files) > 10
    assert {f: found for f in files if (found := non_coherent_loads(f))} == {}


@pytest.mark.gpu
@pytest.mark.parametrize("bn", [128, 256])
def test_operands_that_the_call_before_wrote(bn):
    """Norms into A, products into B, by turns with others; the bits of the same calls with a wait behind each."""
    M, N, K = 768, 640, 1024
    kern, g = _kernel(M, N, K, bn), torch.Generator(device="cuda").manual_seed(1)
    weight = torch.ones(K, device="cuda")
    xs = [torch.randn(M, K, generator=g, device="cuda") * 2.0 ** i for i in range(4)]
    left, rights = torch.randn(K, 256, generator=g, device="cuda"), [torch.randn(256, N, generator=g, device="cuda") * 2.0 ** -i for i in range(4)]
    ws = [weight * 2.0 ** (3 * i) for i in range(4)]
    a, b = torch.empty(M, K, device="cuda"), torch.empty(K, N, device="cuda")
    before = _kernel(K, N, 256, bn)

    def step(i, c):
        before.run(left, rights[i], b)
        matmul_op.rms_norm(xs[i], ws[i], out=a)
        kern.run(a, b, c)
    want = []
    for i in range(4):
        c = torch.empty(M, N, device="cuda")
        before.run(left, rights[i], b)
        matmul_op.rms_norm(xs[i], ws[i], out=a)
        torch.cuda.synchronize()
        kern.run(a, b, c)
        torch.cuda.synchronize()
        assert (c.double() - a.double() @ b.double()).norm() <= 1e-5 * c.double().norm()
        want.append(c)
    got = [torch.empty(M, N, device="cuda") for _ in range(24)]
    torch.cuda.synchronize()
    for i, c in enumerate(got):
        step(i % 4, c)
    torch.cuda.synchronize()
    kern.checkStatus()
    for i, c in enumerate(got):
        assert torch.equal(c, want[i % 4]), i
