"""Run, time and check ONE step of attention over a paged cache from the command line (the counterpart of run_attention for ``append_kv`` and
``attention_paged``): the step's rows are turned and stored in their pages, then attend over them. A small, self-ending workload for profilers
and a quick check of the kernels.

    python -m codegendemo_b200.kcg.run_paged --batch 8 --length 4096 --launches 5              # a decode step: one new token each
    python -m codegendemo_b200.kcg.run_paged --batch 2 --length 4096 --tokens 4096 --window 1024 --sinks 4      # prompts
"""
import argparse
import math
import sys


def append_errors(q, k, v, turned, k_cache, v_cache, table_row, first, rotary):
    """What ``append_kv`` made of one sequence's rows at positions first, first + 1, ..: the relative errors of its turned queries and of the keys in its
    pages (halves of a head in pairs) against 64 bits, and whether its values lie there as they were."""
    import torch
    cos, sin = (t[first:first + q.shape[0], None].double() for t in rotary)
    half = cos.shape[-1]

    def relative(x, got):
        x = x.double()
        want = torch.cat([x[..., :half] * cos - x[..., half:2 * half] * sin, x[..., half:2 * half] * cos + x[..., :half] * sin, x[..., 2 * half:]], -1)
        return ((got.double() - want).norm() / want.norm()).item()
    p = torch.arange(first, first + q.shape[0], device=q.device)
    page = k_cache.shape[2]
    at, slot = table_row.long()[p // page], p % page
    return relative(q, turned), relative(k, k_cache[at, :, slot]), torch.equal(v_cache[at, :, slot], v)


def main(argv=None) -> int:
    import torch
    from codegendemo_b200.kcg.matmul_op import append_kv, attention_paged, attention_paged_status, rotary_table
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=8, help="sequences")
    ap.add_argument("--length", type=int, default=4096, help="tokens of a sequence, the step's among them")
    ap.add_argument("--tokens", type=int, default=1, help="new tokens of each sequence")
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--d", type=int, default=128, choices=[64, 128])
    ap.add_argument("--page", type=int, default=64)
    ap.add_argument("--window", type=int, default=0, help="keys that a token looks back on (0: all)")
    ap.add_argument("--sinks", type=int, default=0, help="first tokens that stay visible")
    ap.add_argument("--dtype", default="bf16", choices=["bf16", "fp16"])
    ap.add_argument("--launches", type=int, default=5)
    ap.add_argument("--warmup", type=int, default=2)
    ap.add_argument("--device", type=int, default=0)
    ap.add_argument("--no-check", action="store_true")
    a = ap.parse_args(argv)
    if not 1 <= a.tokens <= a.length:
        ap.error("--tokens is 1 to --length")
    tdt = torch.bfloat16 if a.dtype == "bf16" else torch.float16
    torch.cuda.set_device(a.device)
    dev = f"cuda:{a.device}"
    g = torch.Generator(device=dev).manual_seed(0)
    rows, used = a.batch * a.tokens, -(-a.length // a.page)
    k_cache, v_cache = (torch.randn(a.batch * used, a.kv_heads, a.page, a.d, generator=g, device=dev, dtype=tdt) for _ in range(2))
    table = torch.randperm(a.batch * used, generator=g, device=dev).int().view(a.batch, used)
    lengths = torch.full((a.batch,), a.length, dtype=torch.int32, device=dev)
    qkv = torch.randn(rows, a.heads + 2 * a.kv_heads, a.d, generator=g, device=dev).to(tdt)
    q, k, v = qkv[:, :a.heads], qkv[:, a.heads:a.heads + a.kv_heads], qkv[:, a.heads + a.kv_heads:]
    rotary = rotary_table(a.length, a.d, device=dev)
    window = a.window or None

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

    turned = timed("rows into the cache, queries and keys turned", lambda: append_kv(k, v, k_cache, v_cache, table, lengths, q=q, rotary=rotary),
                   4 * qkv.numel() + 4 * rows * a.d, ("GB/s", 1e9))
    first = a.length - a.tokens
    seen = sum(min(p + 1, a.window + min(a.sinks, max(0, p + 1 - a.window))) if a.window else p + 1 for p in range(first, a.length))
    near = min(a.length, a.tokens - 1 + a.window) if a.window else a.length
    read = 4 * a.batch * a.kv_heads * a.d * (near + min(a.sinks, a.length - near)) + 4 * rows * a.heads * a.d
    flops = 4.0 * a.batch * seen * a.heads * a.d
    few = a.tokens * (a.heads // a.kv_heads) <= 64
    out = timed("attention", lambda: attention_paged(turned, k_cache, v_cache, table, lengths, window=window, sinks=a.sinks),
                read if few else flops, ("GB/s", 1e9) if few else ("TFLOP/s", 1e12))
    attention_paged_status(a.device)
    if not a.no_check:
        b, n, group = a.batch // 2, min(a.tokens, 128), a.heads // a.kv_heads
        own = slice(b * a.tokens, (b + 1) * a.tokens)
        off_q, off_k, same = append_errors(q[own], k[own], v[own], turned[own], k_cache, v_cache, table[b], first, rotary)
        # each value rounded to 16 bits once, of products and a sum in fp32
        most = torch.finfo(tdt).eps / 2 + 2.0 ** -20
        right = max(off_q, off_k) <= most and same
        print(f"relative error, sequence {b}, turned queries {off_q:.3e} and keys in their pages {off_k:.3e}  tolerance {most:.1e}, values "
              f"{'as they were' if same else 'elsewhere'}  {'OK' if right else 'FAIL'}")
        kf, vf = (c[table[b].long()].transpose(0, 1).reshape(a.kv_heads, -1, a.d)[:, :a.length].double() for c in (k_cache, v_cache))
        x = turned[(b + 1) * a.tokens - n:(b + 1) * a.tokens].double().view(n, a.kv_heads, group, a.d).permute(1, 2, 0, 3)
        p, j = torch.arange(a.length - n, a.length, device=dev)[:, None], torch.arange(a.length, device=dev)[None]
        hidden = (j > p) | ((p - j >= a.window) & (j >= a.sinks)) if a.window else j > p
        s = (x @ kf[:, None].transpose(-1, -2) / math.sqrt(a.d)).masked_fill(hidden, -math.inf)
        ref = (torch.softmax(s, -1) @ vf[:, None]).permute(2, 0, 1, 3).reshape(n, a.heads, a.d)
        err = ((out[(b + 1) * a.tokens - n:(b + 1) * a.tokens].double() - ref).norm() / ref.norm()).item()
        # weights and result rounded to 16 bits, at most 2^-8 each of values that average to less than the largest
        print(f"relative error, sequence {b}, last {n} tokens, against 64 bits {err:.3e}  tolerance 0.01  {'OK' if err <= 0.01 else 'FAIL'}")
        return 0 if right and err <= 0.01 else 1
    return 0


if __name__ == "__main__":
    sys.exit(main())
