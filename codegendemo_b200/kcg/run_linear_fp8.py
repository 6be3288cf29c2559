"""Run, time and check ONE 8-bit linear layer from the command line (the counterpart of run_attention for ``matmul_fp8`` and the
operators around it): norm with residual into 8 bits, weight in blocks of 128 x 128, product; with ``--backward`` the operands and products of
its gradients too. A small, self-ending workload for profilers and a quick check of the kernels.

    python -m codegendemo_b200.kcg.run_linear_fp8 --m 2048 --n 4096 --k 4096 --launches 5 --backward
"""
import argparse
import sys


def main(argv=None) -> int:
    import torch
    from codegendemo_b200.kcg.matmul_op import (matmul_fp8, matmul_fp8_status, quantize_fp8, rms_norm_backward, rms_norm_fp8)
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--m", type=int, default=2048, help="tokens")
    ap.add_argument("--n", type=int, default=4096, help="width of the result")
    ap.add_argument("--k", type=int, default=4096, help="width of the input")
    ap.add_argument("--dtype", default="bf16", choices=["bf16", "fp16", "fp32"])
    ap.add_argument("--launches", type=int, default=5)
    ap.add_argument("--warmup", type=int, default=2)
    ap.add_argument("--device", type=int, default=0)
    ap.add_argument("--backward", action="store_true")
    ap.add_argument("--no-check", action="store_true")
    a = ap.parse_args(argv)
    tdt = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[a.dtype]
    torch.cuda.set_device(a.device)
    dev = f"cuda:{a.device}"
    g = torch.Generator(device=dev).manual_seed(0)
    x, r = (torch.randn(a.m, a.k, generator=g, device=dev).to(tdt) for _ in range(2))
    nw = (1 + 0.1 * torch.randn(a.k, generator=g, device=dev)).to(tdt)
    w = (torch.randn(a.n, a.k, generator=g, device=dev) / a.k ** 0.5).to(tdt)
    dy = torch.randn(a.m, a.n, generator=g, device=dev).to(tdt)
    flops, size = 2.0 * a.m * a.n * a.k, x.element_size()

    def timed(what, fn, work, unit):
        for _ in range(a.warmup):
            out = fn()
        torch.cuda.synchronize()
        times = []
        for _ in range(a.launches):
            s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            s.record()
            out = fn()
            e.record()
            torch.cuda.synchronize()
            times.append(s.elapsed_time(e))
        med = sorted(times)[len(times) // 2]
        print(f"{what:44s} median {med * 1e3:9.1f} us  {work / (med * 1e-3) / unit[1]:8.1f} {unit[0]}")
        return out

    gbs, tfs = ("GB/s", 1e9), ("TFLOP/s", 1e12)
    w8, ws = timed("weight in 128 x 128 blocks", lambda: quantize_fp8(w, rows=128), w.numel() * (size + 1), gbs)
    q, s, h = timed("norm with residual, into 8 bits", lambda: rms_norm_fp8(x, nw, r), x.numel() * (3 * size + 1), gbs)
    y = timed("product", lambda: matmul_fp8(q, s, w8, ws, out_dtype=tdt), flops, tfs)
    if a.backward:
        d8 = timed("gradient in blocks along the outputs", lambda: quantize_fp8(dy), dy.numel() * (size + 1), gbs)
        wt = timed("weight transposed", lambda: quantize_fp8(w, rows=128, transposed=True), w.numel() * (size + 1), gbs)
        du = timed("gradient of the input", lambda: matmul_fp8(*d8, *wt, out_dtype=tdt), flops, tfs)
        dt = timed("gradient in blocks along the tokens", lambda: quantize_fp8(dy, transposed=True), dy.numel() * (size + 1), gbs)
        xt = timed("input in blocks along the tokens", lambda: quantize_fp8(x, transposed=True), x.numel() * (size + 1), gbs)
        timed("gradient of the weight, fp32", lambda: matmul_fp8(*dt, *xt, out_dtype=torch.float32), flops, tfs)
        timed("gradient of the norm", lambda: rms_norm_backward(du, h, nw), 3 * x.numel() * size, gbs)
    matmul_fp8_status(a.device)
    if not a.no_check:
        rows = min(a.m, 256)
        h64 = x[:rows].double() + r[:rows].double()
        u = h64 * (h64.square().mean(dim=1, keepdim=True) + 1e-6).rsqrt() * nw.double()
        ref = u @ w.double().t()
        err = ((y[:rows].double() - ref).norm() / ref.norm()).item()
        # both operands off by 2^-4 of a value at most, about 2^-5.2 of their norm: their product by sqrt(2) times that
        print(f"relative error, first {rows} rows, 64 bits without quantisation {err:.3e}  tolerance 0.08  {'OK' if err <= 0.08 else 'FAIL'}")
        return 0 if err <= 0.08 else 1
    return 0


if __name__ == "__main__":
    sys.exit(main())
