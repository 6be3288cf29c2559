"""The calls that the 8-bit linear layer's operators are measured on: a residual stream's norm (in 16 or 32 bits, or straight into
8-bit values with a scale for each 128 of a row), that norm's gradient, the quantisation of weights, activations and gradients
in blocks, and the product of such operands.

Every case goes through the entry points of ``codegendemo_b200.kcg.matmul_op`` on GPU tensors: operands in hand, results
allocated by the call.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126  # of a block whose values are all (nearly) zero
EPS = 1e-6


def listed():
    return [
        # the residual stream of a decode step of 8 sequences: latency is all of it
        {"name": "norm_decode_bf16", "op": "norm", "rows": 8, "d": 4096, "dtype": "bf16", "residual": True},
        # the same over a long prompt (or a training batch) of a wide model
        {"name": "norm_prompt_bf16", "op": "norm", "rows": 16384, "d": 8192, "dtype": "bf16", "residual": True},
        # a decode step of 32 sequences in front of an 8-bit linear layer
        {"name": "norm_fp8_decode_bf16", "op": "norm_fp8", "rows": 32, "d": 8192, "dtype": "bf16", "residual": True},
        # a packed batch of prompts, of no even length, in front of an 8-bit linear layer
        {"name": "norm_fp8_ragged_fp16", "op": "norm_fp8", "rows": 5001, "d": 5504, "dtype": "fp16", "residual": False},
        # backward pass of a training batch: gradient of the residual stream and of the weight
        {"name": "norm_grad_bf16", "op": "norm_grad", "rows": 8192, "d": 4096, "dtype": "bf16", "dh": True},
        # a small model trained in 32 bits, odd number of tokens
        {"name": "norm_grad_ragged_fp32", "op": "norm_grad", "rows": 513, "d": 1376, "dtype": "fp32", "dh": False},
        # a linear layer's weight, once after each optimizer step (or at load)
        {"name": "quantize_weight_bf16", "op": "quantize", "rows": 11008, "cols": 4096, "dtype": "bf16", "block": 128, "transposed": False},
        # a gradient in front of the weight's gradient: blocks along the tokens, laid out along them
        {"name": "quantize_grad_bf16", "op": "quantize", "rows": 8192, "cols": 4096, "dtype": "bf16", "block": 1, "transposed": True},
        # one new token through a down projection: streams the weight once
        {"name": "matmul_token_bf16", "op": "matmul", "m": 1, "n": 4096, "k": 11008, "out": "bf16", "b_block": 128, "bias": False},
        # a short prompt through a layer of no even sizes, with a bias
        {"name": "matmul_ragged_bf16", "op": "matmul", "m": 777, "n": 2752, "k": 1488, "out": "bf16", "b_block": 128, "bias": True},
        # a long prompt, or a training batch, through a square projection
        {"name": "matmul_prompt_bf16", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "b_block": 128, "bias": False},
        # a weight's gradient: both operands in blocks of 1 x 128 along the tokens, the result in 32 bits
        {"name": "matmul_grad_fp32", "op": "matmul", "m": 4096, "n": 4096, "k": 8192, "out": "fp32", "b_block": 1, "bias": False},
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, steps):
    """Between lo and hi, evenly over the logarithm, a multiple of one of the steps."""
    step = rng.choice(steps)
    return max(lo, min(hi, int(round(_log(rng, lo, hi) / step)) * step))


def draw(rng):
    op = rng.choice(["norm", "norm_fp8", "norm_grad", "quantize", "quantize", "matmul", "matmul", "matmul"])
    while True:
        if op == "matmul":
            # tokens: any number; widths of real layers, now and then odd ones (operands then have padded rows)
            c = {"op": op, "m": _size(rng, 1, 8192, [1]), "n": _size(rng, 256, 16384, [1, 64, 128, 128]),
                 "k": _size(rng, 128, 16384, [1, 16, 64, 128, 128]), "out": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                 "b_block": rng.choice([128, 128, 1]), "bias": rng.random() < 0.25}
            if c["m"] * c["n"] * c["k"] > 8192 ** 3:
                continue
        elif op == "quantize":
            c = {"op": op, "rows": _size(rng, 1, 16384, [1, 1, 128]), "cols": _size(rng, 64, 16384, [1, 64, 128, 128]),
                 "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "block": rng.choice([1, 128]), "transposed": rng.random() < 0.5}
            if c["rows"] * c["cols"] > 16384 * 8192:
                continue
        else:
            c = {"op": op, "rows": _size(rng, 1, 16384, [1]), "d": _size(rng, 64, 16384, [1, 64, 128, 128]),
                 "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
            if op == "norm_grad":
                c["dh"] = rng.random() < 0.5
            else:
                c["residual"] = rng.random() < 0.6
            if c["rows"] * c["d"] > 16384 * 4096:
                continue
        return c


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, d):
    """Normal values, their channels of different sizes, a few of them large: as a residual stream is."""
    channel = torch.exp(0.5 * _normal(g, d))
    large = torch.rand(d, generator=g, device="cuda") < 0.004
    return _normal(g, rows, d) * torch.where(large, 12.0 * channel, channel)


def _padded(q):
    """The 8-bit matrix as a view of one whose rows start on 16-byte boundaries."""
    pitch = -(-q.shape[1] // 16) * 16
    if pitch == q.shape[1]:
        return q.contiguous()
    wide = torch.zeros((q.shape[0], pitch), dtype=q.dtype, device=q.device)
    wide.view(torch.uint8)[:, :q.shape[1]] = q.view(torch.uint8)
    return wide[:, :q.shape[1]]


def _blocks(x, rows):
    """x, filled up with zeros, as (block rows, rows, block columns, 128)."""
    r, c = x.shape
    br, bc = -(-r // rows), -(-c // 128)
    full = torch.zeros((br * rows, bc * 128), dtype=x.dtype, device=x.device)
    full[:r, :c] = x
    return full.view(br, rows, bc, 128)


def _quantized(x, rows):
    """(values, scales): 8-bit values of x / scale, a scale for each block of rows x 128."""
    b = _blocks(x, rows)
    scale = (b.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp(min=SMALLEST_SCALE)
    q = (b / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).reshape(b.shape[0] * rows, -1)[:x.shape[0], :x.shape[1]].view(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        a, sa = _quantized(_activations(g, m, k), 1)
        b, sb = _quantized(0.02 * _normal(g, n, k) * torch.exp(0.3 * _normal(g, n, 1)), case["b_block"])
        bias = (0.1 * _normal(g, n)).to(DTYPES[case["out"]]) if case["bias"] else None
        return {"case": case, "a": _padded(a), "sa": sa, "b": _padded(b), "sb": sb, "bias": bias}
    dt = DTYPES[case["dtype"]]
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        x = 0.02 * _normal(g, r, c) if case["block"] == 128 else 1e-3 * _activations(g, r, c)
        return {"case": case, "x": x.to(dt)}
    r, d = case["rows"], case["d"]
    state = {"case": case, "x": _activations(g, r, d).to(dt), "w": (1.0 + 0.2 * _normal(g, d)).to(dt)}
    if op == "norm_grad":
        state["dy"] = (1e-2 * _normal(g, r, d)).to(dt)
        state["dh"] = (1e-2 * _normal(g, r, d)).to(dt) if case["dh"] else None
    else:
        state["residual"] = (2.0 * _activations(g, r, d)).to(dt) if case["residual"] else None
    return state


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from codegendemo_b200.kcg import matmul_op
        if op == "norm":
            return matmul_op.rms_norm(state["x"], state["w"], state["residual"], eps=EPS)
        if op == "norm_fp8":
            return matmul_op.rms_norm_fp8(state["x"], state["w"], state["residual"], eps=EPS)
        if op == "norm_grad":
            return matmul_op.rms_norm_backward(state["dy"], state["x"], state["w"], eps=EPS, dh=state["dh"])
        if op == "quantize":
            return matmul_op.quantize_fp8(state["x"], rows=case["block"], transposed=case["transposed"])
        return matmul_op.matmul_fp8(state["a"], state["sa"], state["b"], state["sb"], bias=state["bias"],
                                    out_dtype=DTYPES[case["out"]])
    if op in ("norm", "norm_fp8"):
        dt = state["x"].dtype
        h = state["x"].float()
        if state["residual"] is not None:
            h = h + state["residual"].float()
        y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * state["w"].float()
        first = (y.to(dt),) if op == "norm" else _quantized(y, 1)
        if state["residual"] is not None:
            return (*first, h.to(dt))
        return first[0] if op == "norm" else first
    if op == "norm_grad":
        dt = state["x"].dtype
        h, dy = state["x"].float(), state["dy"].float()
        rs = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
        g = dy * state["w"].float()
        dx = rs * g - h * (rs * rs * rs * (g * h).mean(dim=1, keepdim=True))
        if state["dh"] is not None:
            dx = dx + state["dh"].float()
        return dx.to(dt), (dy * h * rs).sum(dim=0).to(dt)
    if op == "quantize":
        x = state["x"].float()
        return _quantized(x.t() if case["transposed"] else x, case["block"])
    k = case["k"]
    a = state["a"].float() * state["sa"].repeat_interleave(128, 1)[:, :k]
    sb = state["sb"] if case["b_block"] == 1 else state["sb"].repeat_interleave(128, 0)[:case["n"]]
    b = state["b"].float() * sb.repeat_interleave(128, 1)[:, :k]
    c = a @ b.t()
    if state["bias"] is not None:
        c = c + state["bias"].float()
    return c.to(DTYPES[case["out"]])


def work(case):
    op = case["op"]
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        kb, out = -(-k // 128), 4 if case["out"] == "fp32" else 2
        scales = 4 * kb * (m + (n if case["b_block"] == 1 else -(-n // 128)))
        return {"bytes": m * k + n * k + scales + m * n * out + (n * out if case["bias"] else 0), "flops": 2.0 * m * n * k}
    e = 4 if case["dtype"] == "fp32" else 2
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        p, s = (c, r) if case["transposed"] else (r, c)
        return {"bytes": r * c * (e + 1) + 4 * -(-p // case["block"]) * -(-s // 128), "flops": 3.0 * r * c}
    r, d = case["rows"], case["d"]
    if op == "norm_grad":
        return {"bytes": r * d * e * (4 if case["dh"] else 3) + 2 * d * e, "flops": 12.0 * r * d}
    read = r * d * e * (3 if case["residual"] else 1) + d * e
    return {"bytes": read + (r * d * e if op == "norm" else r * d + 4 * r * -(-d // 128)), "flops": 6.0 * r * d}


def exact(case, seed):
    """In 64 bits, from the definitions: 8-bit values before their rounding, as x over its block's scale."""
    s = prepare(case, seed)
    op = case["op"]

    def in_blocks(v, rows):
        """v over the scale of its block, and the scales, block column by block column."""
        r, c = v.shape
        values, scales = torch.empty_like(v), []
        for c0 in range(0, c, 128):
            part = v[:, c0:c0 + 128]
            top = part.abs().max(dim=1).values
            if rows > 1:
                top = torch.stack([t.max() for t in top.split(rows)])
            scale = torch.maximum(top / 448.0, torch.full_like(top, 2.0 ** -126))
            values[:, c0:c0 + 128] = part / scale.repeat_interleave(rows)[:r, None]
            scales.append(scale)
        return values, torch.stack(scales, dim=1)

    if op == "matmul":
        total = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for i, k0 in enumerate(range(0, case["k"], 128)):
            a = s["a"][:, k0:k0 + 128].double() * s["sa"][:, i].double()[:, None]
            sb = s["sb"][:, i].double()
            if case["b_block"] == 128:
                sb = sb[torch.arange(case["n"], device="cuda") // 128]
            total.addmm_(a, (s["b"][:, k0:k0 + 128].double() * sb[:, None]).T)
        return total if s["bias"] is None else total + s["bias"].double()
    if op == "quantize":
        x = s["x"].double()
        return in_blocks(x.T.contiguous() if case["transposed"] else x, case["block"])
    h, w = s["x"].double(), s["w"].double()
    if op == "norm_grad":
        d = case["d"]
        root = (h.square().sum(1) / d + EPS).sqrt()[:, None]
        unit = h / root
        g = s["dy"].double() * w
        dx = (g - unit * ((g * unit).sum(1) / d)[:, None]) / root
        return dx if s["dh"] is None else dx + s["dh"].double(), (s["dy"].double() * unit).sum(0)
    if s["residual"] is not None:
        h = h + s["residual"].double()
    y = h / (h.square().sum(1) / case["d"] + EPS).sqrt()[:, None] * w
    out = (y,) if op == "norm" else in_blocks(y, 1)
    if s["residual"] is not None:
        return (*out, h)
    return out[0] if op == "norm" else out
