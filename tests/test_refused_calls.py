"""A call that the CUDA runtime refuses (here: of a device that is not there) leaves nothing behind for the next one."""
import ctypes

import pytest
import torch

from codegendemo_b200 import _lib

GONE = 63  # (a device's index is below 64)


def _refused():
    """One call of every entry that goes through the CUDA runtime, with arguments right but for the device."""
    lib = _lib.get_lib()
    x = torch.ones((8, 64), dtype=torch.bfloat16, device="cuda")
    q, k = (torch.ones((2, n, 64), dtype=torch.bfloat16, device="cuda") for n in (300, 64))
    f = torch.ones((8, 64), device="cuda")
    s, y = torch.empty((8, 128), device="cuda"), torch.empty((8, 128), dtype=torch.uint8, device="cuda")
    work = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    p = _lib.Fp8Product(y.data_ptr(), s.data_ptr(), y.data_ptr(), s.data_ptr(), f.data_ptr(), 0, 128, 0, 128, 0, 0, 8, 8, 64, 128, 1, 1, 4, 0.0, 0)
    at = {"x": x.data_ptr(), "f": f.data_ptr(), "s": s.data_ptr(), "y": y.data_ptr()}
    calls = {
        "quantize": lambda: lib.kcg_quantize_fp8(GONE, 0, at["x"], 0, at["y"], 128, at["s"], 8, 64, 1, 0, 62, 1),
        "norm": lambda: lib.kcg_rms_norm(GONE, 0, at["x"], 0, 0, 0, at["x"], at["y"], 0, 0, 0, 4, 64, 1e-6, 62),
        "norm into 8 bits": lambda: lib.kcg_rms_norm_fp8(GONE, 0, at["x"], 0, 0, 0, at["x"], at["y"], 64, at["s"], 0, 0, 4, 64, 1e-6, 62),
        "norm's gradient": lambda: lib.kcg_rms_norm_backward(GONE, 0, at["x"], 0, at["x"], 0, at["x"], 0, 0, at["y"], 0, at["s"], work.data_ptr(),
                                                             work.numel(), 4, 64, 1e-6, 62),
        "workspace": lambda: lib.kcg_rms_norm_backward_workspace(GONE, 4, 64),
        "product": lambda: lib.kcg_matmul_fp8(GONE, 0, ctypes.byref(p)),
        "product's status": lambda: lib.kcg_matmul_fp8_status(GONE, (ctypes.c_uint32 * 4)()),
        "softmax": lambda: lib.kcg_softmax_rows(GONE, 0, at["x"], 8, 64, 64, 1.0, 62),
        "attention": lambda: lib.kcg_attention_fwd(GONE, 0, q.data_ptr(), k.data_ptr(), k.data_ptr(), q.data_ptr(), 62, 2, 300, 64, 64, 0.125),
        "attention's status": lambda: lib.kcg_attention_status(GONE, (ctypes.c_uint32 * 4)()),
    }
    return calls, (x, q, k, f, s, y, work, p)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["quantize", "norm", "norm into 8 bits", "norm's gradient", "workspace", "product", "product's status", "softmax",
                                  "attention", "attention's status"])
def test_the_next_call_is_not_refused_for_it(what):
    lib = _lib.get_lib()
    calls, alive = _refused()
    x, stream = torch.randn((16, 64), device="cuda").bfloat16(), torch.cuda.current_stream().cuda_stream
    want = torch.softmax(x.float(), dim=1)
    assert calls[what]() != 0
    assert lib.kcg_softmax_rows(0, stream, x.data_ptr(), 16, 64, 64, 1.0, 62) == 0, lib.kcg_last_error()
    assert (x.float() - want).abs().max() <= 2.0 ** -8
    assert calls[what]() != 0
    q, o = torch.randn((2, 300, 64), device="cuda").bfloat16(), torch.empty((2, 300, 64), device="cuda").bfloat16()
    assert lib.kcg_attention_fwd(0, stream, q.data_ptr(), q.data_ptr(), q.data_ptr(), o.data_ptr(), 62, 2, 300, 300, 64, 0.125) == 0, lib.kcg_last_error()
    torch.cuda.synchronize()
    assert torch.isfinite(o).all()
