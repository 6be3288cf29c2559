"""8-bit products behind the kernels that write their operands and scales into the same memory again and again. A kernel may be on the
GPU while the one before it still writes (programmatic dependent launch), so what that one writes is not read-only for its life."""
import ctypes
import os
import re

import pytest
import torch

from codegendemo_b200 import _lib

SOURCES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "codegendemo_b200", "csrc")
CODES = {torch.bfloat16: 62, torch.float32: 4}


def non_coherent_loads(path):
    text = re.sub(r"//[^\n]*", "", open(path).read())
    return re.findall(r"__ldg\s*\([^\n]*|ld\.global\.nc[^\n]*", text)


@pytest.mark.parametrize("file", ["kcg_fp8.cu", "kcg_norm.cu", "kcg_quantize.cu", "fp8_common.cuh"])
def test_no_load_asks_for_memory_that_is_read_only_for_the_kernels_life(file):
    assert non_coherent_loads(os.path.join(SOURCES, file)) == []


def aligned(cols):
    return -(-cols // 16) * 16


class Chain:
    """quantise -> product, or norm into 8 bits -> product, through the C entries, every result into memory that stays."""

    def __init__(self, m, n, k, block_b, dtype, norm):
        self.lib, self.m, self.n, self.k, self.block_b, self.dtype, self.norm = _lib.get_lib(), m, n, k, block_b, dtype, norm
        empty = lambda *s, dtype: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        self.x, self.w = empty(m, k, dtype=dtype), empty(n, k, dtype=dtype)
        self.nw = torch.ones(k, dtype=dtype, device="cuda")
        kb = -(-k // 128)
        self.a, self.sa = empty(m, aligned(k), dtype=torch.uint8), empty(m, kb, dtype=torch.float32)
        self.b, self.sb = empty(n, aligned(k), dtype=torch.uint8), empty(-(-n // block_b), kb, dtype=torch.float32)
        self.c = empty(m, n, dtype=torch.float32)

    def _ok(self, status):
        assert status == 0, self.lib.kcg_last_error()

    def step(self):
        stream, code, ld = torch.cuda.current_stream().cuda_stream, CODES[self.dtype], aligned(self.k)
        self._ok(self.lib.kcg_quantize_fp8(0, stream, self.w.data_ptr(), 0, self.b.data_ptr(), ld, self.sb.data_ptr(), self.n, self.k,
                                           self.block_b, 0, code, 1))
        if self.norm:
            self._ok(self.lib.kcg_rms_norm_fp8(0, stream, self.x.data_ptr(), 0, 0, 0, self.nw.data_ptr(), self.a.data_ptr(), ld,
                                               self.sa.data_ptr(), 0, 0, self.m, self.k, 1e-6, code))
        else:
            self._ok(self.lib.kcg_quantize_fp8(0, stream, self.x.data_ptr(), 0, self.a.data_ptr(), ld, self.sa.data_ptr(), self.m, self.k, 1, 0,
                                               code, 1))
        p = _lib.Fp8Product(self.a.data_ptr(), self.sa.data_ptr(), self.b.data_ptr(), self.sb.data_ptr(), self.c.data_ptr(), 0, ld, 0, ld, 0, 0,
                            self.m, self.n, self.k, self.block_b, 1, 1, 4, 0.0, 0)
        self._ok(self.lib.kcg_matmul_fp8(0, stream, ctypes.byref(p)))


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("m,n,k", [(3, 512, 1024), (40, 640, 512), (200, 768, 640), (2304, 2304, 256), (700, 2816, 1500)])
def test_scales_that_change_from_call_to_call(m, n, k, block_b, norm):
    """Values whose scales differ by powers of two from step to step: a stale scale is a wrong power of two in the product. The bits
    of the same calls with a wait behind each."""
    chain = Chain(m, n, k, block_b, torch.bfloat16, norm)
    g = torch.Generator(device="cuda").manual_seed(5)
    inputs = [(torch.randn(m, k, generator=g, device="cuda").bfloat16() * 2.0 ** (i % 7 - 3),
               torch.randn(n, k, generator=g, device="cuda").bfloat16() * 2.0 ** (i % 5 - 2)) for i in range(8)]
    want = []
    for x, w in inputs:
        chain.x.copy_(x), chain.w.copy_(w)
        torch.cuda.synchronize()
        chain.step()
        torch.cuda.synchronize()
        want.append(chain.c.clone())
    results = torch.empty((3 * len(inputs), m, n), device="cuda")
    torch.cuda.synchronize()
    for i in range(3 * len(inputs)):
        x, w = inputs[i % len(inputs)]
        chain.x.copy_(x), chain.w.copy_(w)
        chain.step()
        results[i].copy_(chain.c)
    torch.cuda.synchronize()
    for i in range(3 * len(inputs)):
        assert torch.equal(results[i], want[i % len(inputs)]), i
    # nothing between the launches: x and w, then their halves (exact: the products a quarter), by turns in one captured graph
    half = Chain(m, n, k, block_b, torch.bfloat16, norm)
    half.a, half.sa, half.b, half.sb = chain.a, chain.sa, chain.b, chain.sb
    chain.x.copy_(inputs[0][0]), chain.w.copy_(inputs[0][1])
    half.x.copy_(inputs[0][0] / 2), half.w.copy_(inputs[0][1] / 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(4):
            chain.step()
            half.step()
    for _ in range(5):
        chain.c.zero_(), half.c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(chain.c, want[0])
        if not norm:  # (a norm of x / 2 differs from that of x by the eps)
            assert torch.equal(half.c * 4, want[0])
