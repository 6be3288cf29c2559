"""The warm calls of the 8-bit linear layer's operators: what they take, and that they give the bits of the operators' own way."""
import pytest
import torch

from codegendemo_b200 import build as kbuild
from codegendemo_b200.kcg import fp8_op, matmul_op


@pytest.fixture(scope="module")
def warm():
    if kbuild.build_torchcall() is None or not matmul_op._warm_calls():
        pytest.skip("no module of warm calls for this torch")
    return matmul_op._warm_calls()


def test_everything_but_right_plain_cuda_arguments_goes_the_operators_way(warm):
    x, w = torch.zeros((4, 16)), torch.zeros(16)
    for a in (x, x.t(), x.to("meta"), x.to_sparse(), None, 3, "a", w):
        assert warm.rms_norm(a, w, None, 1e-6) is None and warm.rms_norm_fp8(a, w, None, 1e-6) is None
        assert warm.rms_norm_backward(a, a, w, 1e-6, None) is None
        assert warm.quantize_fp8(a, 1, False) is None and warm.matmul_fp8(a, a, a, a, None, False, None) is None
    assert warm.rms_norm() is None and warm.quantize_fp8(x, 1 << 80, False) is None and warm.matmul_fp8(x) is None


def _calls(rows, width, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    x, r, dy = (torch.randn(rows, width, generator=g, device="cuda").to(dtype) for _ in range(3))
    w = torch.randn(width, generator=g, device="cuda").to(dtype)
    n = 200
    a, sa = fp8_op.quantize_fp8(x)
    weight = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    bias = torch.randn(n, generator=g, device="cuda").to(dtype)
    return [lambda: fp8_op.rms_norm(x, w), lambda: fp8_op.rms_norm(x, w, r, eps=1e-5), lambda: fp8_op.rms_norm_fp8(x, w),
            lambda: fp8_op.rms_norm_fp8(x, w, r), lambda: fp8_op.rms_norm_backward(dy, x, w), lambda: fp8_op.rms_norm_backward(dy, x, w, dh=r),
            lambda: fp8_op.quantize_fp8(x), lambda: fp8_op.quantize_fp8(x, rows=128), lambda: fp8_op.quantize_fp8(x, transposed=True),
            lambda: fp8_op.quantize_fp8(x, rows=128, transposed=True)] + \
           [lambda b=b: fp8_op.matmul_fp8(a, sa, *fp8_op.quantize_fp8(weight, rows=b)) for b in (1, 128)] + \
           [lambda: fp8_op.matmul_fp8(a, sa, *fp8_op.quantize_fp8(weight), bias=bias, relu=True, out_dtype=dtype)]


def _flat(r):
    return list(r) if isinstance(r, tuple) else [r]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,dtype", [(3, 256, torch.bfloat16), (1, 1000, torch.float16), (40, 77, torch.float32), (130, 1, torch.bfloat16)])
def test_the_same_results_either_way(warm, monkeypatch, rows, width, dtype):
    for call in _calls(rows, width, dtype):
        monkeypatch.setattr(fp8_op, "_warm", False)
        want = _flat(call())
        monkeypatch.setattr(fp8_op, "_warm", warm)
        got = _flat(call())
        assert len(got) == len(want)
        for p, q in zip(got, want):
            assert p.dtype == q.dtype and p.shape == q.shape and p.stride() == q.stride() and p.device == q.device
            assert torch.equal(p.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))


@pytest.mark.gpu
def test_refusals_stay_the_operators(warm, monkeypatch):
    monkeypatch.setattr(fp8_op, "_warm", warm)
    x, w = torch.zeros((4, 16), device="cuda"), torch.zeros(16, device="cuda")
    for call in (lambda: fp8_op.rms_norm(x, w[:15]), lambda: fp8_op.rms_norm(x, w, eps=-1.0), lambda: fp8_op.rms_norm(x, w.half()),
                 lambda: fp8_op.rms_norm(x, w, x[:3]), lambda: fp8_op.rms_norm_backward(x, x, w, dh=x[:, :8]), lambda: fp8_op.quantize_fp8(x, rows=2),
                 lambda: fp8_op.rms_norm(x[:, ::2], w[:8]), lambda: fp8_op.rms_norm(x[:1].expand(4, 16), w)):
        with pytest.raises(ValueError):
            call()
    assert fp8_op.rms_norm(x[:0], w).shape == (0, 16)


@pytest.mark.gpu
def test_a_mode_that_watches_torch_sees_the_results_made(warm, monkeypatch):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))
    monkeypatch.setattr(fp8_op, "_warm", warm)
    x, w = torch.ones((4, 16), device="cuda"), torch.ones(16, device="cuda")
    with Seen():
        fp8_op.rms_norm(x, w)
    assert any("empty" in n for n in Seen.names)
