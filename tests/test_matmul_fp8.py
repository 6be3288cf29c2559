"""The product of 8-bit operands in blocks against the same sums in 64 bits, and the chain that a linear layer makes of it.

Tolerance: products of two 8-bit values and sums of powers of two of them are exact in fp32 but for the alignment in the tensor core,
at least 24 bits wide: an instruction of 32 products into an accumulator is off by 33 x 2^-23 of its largest term at most, four of
them a block by 2^-18 of the block's magnitudes (A = sum of |a b| with their scales, of which the largest term is at most one share, and
132 x 2^-23 = 2^-16 holds if ONE term is all of A; spread over 128 terms it is far below). Each block's addition is off by 2^-24 of the sum, and its scales by 2 x 2^-24. In
all 2^-16 A + blocks x 2^-24 A, and half a step of the result's type.
"""
import ctypes

import pytest
import torch

from codegendemo_b200 import _lib
from codegendemo_b200.kcg import matmul_op
from tests.test_rms_norm import half_step

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def operand(rows, k, block, seed, dtype=E4, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device=device) * torch.exp(torch.randn(rows, 1, generator=g, device=device))
    return matmul_op.quantize_fp8(x, rows=block, dtype=dtype)


def wide64(q, s, block):
    s = s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.double() * (s.repeat_interleave(128, 0)[:q.shape[0]] if block == 128 else s)


def check(m, n, k, block_b=128, out=torch.bfloat16, bias=False, relu=False, beta=0.0, fa=E4, fb=E4, seed=0, pitch=0):
    a, sa = operand(m, k, 1, seed, fa)
    b, sb = operand(n, k, block_b, seed + 1, fb)
    bias = torch.randn(n, device="cuda").to(out) if bias else None
    c = None
    if beta or pitch:
        store = torch.full((m, n + pitch), float("nan"), dtype=out, device="cuda")
        c = store[:, :n]
        if beta:
            c.copy_(torch.randn(m, n, device="cuda"))
    old = c.double() if beta else 0.0
    got = matmul_op.matmul_fp8(a, sa, b, sb, c=c, beta=beta, bias=bias, relu=relu, out_dtype=out)
    matmul_op.matmul_fp8_status()
    if pitch:
        assert torch.isnan(store[:, n:]).all()
    a64, b64 = wide64(a, sa, 1), wide64(b, sb, block_b)
    want = a64 @ b64.t() + beta * old + (0 if bias is None else bias.double())
    size = a64.abs() @ b64.abs().t()
    if relu:
        want = want.clamp(min=0)
    allowed = (2.0 ** -16 + (-(-k // 128) + 4) * 2.0 ** -24) * size
    rest = 4 * 2.0 ** -24 * (want.abs() + (abs(beta) * old.abs() if beta else 0) + (0 if bias is None else bias.double().abs()))
    allowed = allowed + rest + half_step(want, out) * (1 + 2.0 ** -8)
    off = (got.double() - want).abs()
    # a value from half a step past the type's largest on is rounded to infinity (fp16: 65520)
    top = torch.finfo(out).max
    past = torch.isinf(got) & (torch.sign(got).double() == torch.sign(want)) & (want.abs() + allowed >= top * (1 + torch.finfo(out).eps / 4))
    off = torch.where(past, torch.zeros_like(off), off)
    assert got.dtype == out and got.shape == (m, n)
    assert bool((off <= allowed).all()), f"{m}x{n}x{k}: off by {(off / allowed).max().item():.3f} of what is allowed"


class _OnGpu(torch.Tensor):
    is_cuda = True


def _fake(*shape, dtype=E4):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype).as_subclass(_OnGpu) if dtype in (E4, E5) else \
        torch.zeros(shape, dtype=dtype).as_subclass(_OnGpu)


def _scales(*shape):
    return _fake(*shape, dtype=torch.float32)


@pytest.mark.parametrize("call,message", [
    (lambda: matmul_op.matmul_fp8(torch.zeros(4, 128).to(E4), torch.ones(4, 1), torch.zeros(8, 128).to(E4), torch.ones(1, 1)), "CUDA"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128, dtype=torch.bfloat16), _scales(4, 1), _fake(8, 128), _scales(1, 1)), "a must be float8"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128, dtype=torch.int8), _scales(1, 1)), "b must be float8"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 256), _scales(1, 2)), "rows of 128 values"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 2), _fake(8, 128), _scales(1, 1)), "a_scale"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(1, 1), _fake(8, 128), _scales(1, 1)), "a_scale"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128), _scales(2, 1)), "b_scale"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128), _scales(8, 2)), "b_scale"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _fake(4, 1, dtype=torch.bfloat16), _fake(8, 128), _scales(1, 1)), "float32"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128), _scales(1, 1), beta=1.0), "needs the c"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128), _scales(1, 1), out_dtype=torch.float64), "float32"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128), _scales(1, 1), c=_scales(4, 9)), "c must be 4 x 8"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128), _scales(1, 1), c=_scales(4, 8), out_dtype=torch.bfloat16), "out_dtype"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 128), _scales(4, 1), _fake(8, 128), _scales(1, 1), bias=_scales(8)), "bias"),
    (lambda: matmul_op.matmul_fp8(_fake(4, 0), _scales(4, 0), _fake(8, 0), _scales(1, 0)), "no columns"),
    (lambda: matmul_op.matmul_fp8(_fake(128, 4).t(), _scales(4, 1), _fake(8, 128), _scales(1, 1)), "contiguous rows"),
])
def test_wrong_arguments_are_refused(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_the_c_entry_refuses_what_it_cannot_take():
    lib = _lib.get_lib()
    ok = dict(A=256, scale_a=256, B=256, scale_b=256, C=256, m=4, n=8, k=128, block_b=128, dtype_a=1, dtype_b=1, dtype_c=62)

    def call(**kw):
        return lib.kcg_matmul_fp8(0, 0, ctypes.byref(_lib.Fp8Product(**{**ok, **kw})))
    assert call(m=0) == 0
    for bad in (dict(A=0), dict(B=0), dict(C=0), dict(scale_a=0), dict(scale_b=0), dict(m=-1), dict(n=0), dict(k=0), dict(lda=64),
                dict(lda=136), dict(ldb=130), dict(k=130), dict(A=264), dict(ldc=4), dict(C=257), dict(bias=1), dict(block_b=64),
                dict(dtype_a=3), dict(dtype_b=0), dict(dtype_c=1), dict(k=256, ld_scale_a=1)):
        assert call(**bad) == _lib.E_BAD_ARG, bad
    assert lib.kcg_matmul_fp8(0, 0, None) == _lib.E_BAD_ARG


def test_sizes_that_no_32_bits_hold_are_refused():
    lib = _lib.get_lib()
    ok = dict(A=256, scale_a=256, B=256, scale_b=256, C=256, m=8, n=8, k=128, block_b=128, dtype_a=1, dtype_b=1, dtype_c=62)
    for bad in (dict(m=2 ** 31 - 1), dict(n=2 ** 31 - 255), dict(k=2 ** 31 - 1)):
        assert lib.kcg_matmul_fp8(0, 0, ctypes.byref(_lib.Fp8Product(**{**ok, **bad}))) == _lib.E_TOO_LARGE, bad
    for rows, cols in ((2 ** 31 - 255, 8), (8, 2 ** 31 - 1)):
        for block, transposed in ((1, 0), (1, 1), (128, 0), (128, 1)):
            assert lib.kcg_quantize_fp8(0, 0, 256, 0, 256, 2 ** 31, 256, rows, cols, block, transposed, 62, 1) == _lib.E_TOO_LARGE


def _plan(m, n, k, block_b=128, sms=148):
    out = (ctypes.c_int * 4)()
    _lib.get_lib().kcg_internal_fp8_plan(m, n, k, block_b, sms, out)
    return list(out)


def test_every_plan_gives_every_part_work():
    """Splits are a power of two, at most 8 (tiles of 128 columns: 4) and at most half the blocks of K, for any GPU; few tokens are columns
    of a tile."""
    for m in (1, 16, 17, 32, 33, 64, 65, 128, 500, 2048, 30000):
        for n in (1, 100, 128, 1000, 4096, 11008):
            for k in (1, 128, 129, 512, 4096, 11008):
                for sms in (148, 132, 20, 1):
                    for block_b in (1, 128):
                        pair, swap, bn, splits = _plan(m, n, k, block_b, sms)
                        assert splits in (1, 2, 4, 8) and (splits == 1 or 2 * splits <= -(-k // 128) and not pair)
                        assert bn == 256 if pair else bn in (16, 32, 64, 128) and (swap or bn == 128)
                        assert splits < 8 or swap
                        assert not swap or bn >= m


# (m, n, k): tokens at each width of a tile, full and one past it; widths and sums that end inside a tile or a block, one of one
# column and one value; K shared by 2, 4, 8 CTAs; tiles of 128 x 128, alone and shared; CTA pairs, one tile each and several
FEW = [(1, 4096, 11008), (1, 1, 1), (1, 128, 128), (2, 130, 144), (16, 256, 1024), (17, 1000, 528), (32, 100, 2048), (31, 2752, 1376), (32, 4096, 512),
       (25, 11008, 4096), (5, 257, 16384), (9, 64, 100), (3, 10240, 640)]
SOME = [(33, 2752, 1376), (64, 4096, 512), (48, 64, 100), (64, 300, 8192), (50, 10240, 700)]
MIDDLING = [(65, 64, 100), (127, 4096, 4096), (128, 257, 1040), (129, 1000, 127), (300, 128, 8192), (256, 4096, 2000), (100, 14336, 300)]
MANY = [(2049, 2305, 300), (2304, 2304, 128), (5000, 1024, 1000), (256, 18944, 257), (777, 2752, 1488), (4000, 4000, 520)]


def test_the_shapes_reach_every_kernel():
    assert {_plan(*s, b)[1] for s in FEW for b in (1, 128)} == {1} and {_plan(*s)[2] for s in FEW} == {16, 32}
    assert {_plan(*s)[3] for s in FEW} == {1, 2, 4, 8}
    assert {_plan(*s, 1)[2] for s in SOME} == {64} and {_plan(*s, 1)[3] for s in SOME} == {1, 2, 4, 8}
    for b in (1, 128):
        assert {tuple(_plan(*s, b)[:2]) for s in MIDDLING} == {(0, 0)} and {_plan(*s, b)[3] for s in MIDDLING} == {1, 2, 4}
        assert {tuple(_plan(*s, b)[:2]) for s in MANY} == {(1, 0)}


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("m,n,k", FEW + SOME + MIDDLING + MANY)
def test_shapes(m, n, k, block_b):
    for out in (torch.bfloat16, torch.float32, torch.float16):
        check(m, n, k, block_b, out)


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("m,n,k", [(3, 300, 1024), (200, 300, 1024), (200, 304, 500), (2049, 2305, 300)])
def test_bias_relu_beta_and_a_pitch(m, n, k, block_b):
    check(m, n, k, block_b, bias=True)
    check(m, n, k, block_b, bias=True, relu=True, out=torch.float32)
    check(m, n, k, block_b, beta=0.5, out=torch.float32, pitch=8)
    check(m, n, k, block_b, beta=-2.0, bias=True, relu=True, out=torch.bfloat16, pitch=3)
    check(m, n, k, block_b, out=torch.float16, pitch=8)


@pytest.mark.gpu
@pytest.mark.parametrize("fa,fb", [(E5, E4), (E4, E5), (E5, E5)])
def test_both_8_bit_types(fa, fb):
    for m, n, k in ((3, 300, 1024), (200, 300, 500), (2049, 2305, 300)):
        check(m, n, k, 128, fa=fa, fb=fb, out=torch.float32)
        check(m, n, k, 1, fa=fa, fb=fb)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(8, 200), (300, 200), (2304, 2304)])
def test_each_value_meets_its_partner(m, n):
    """One value of each row of a, at a place of its own, picks a column of b: exact in every type."""
    k = 384
    g = torch.Generator(device="cuda").manual_seed(1)
    at = torch.randint(0, k, (m,), generator=g, device="cuda")
    a = torch.zeros((m, k), device="cuda")
    a[torch.arange(m), at] = 1.0
    b = torch.randint(-15, 16, (n, k), generator=g, device="cuda").float()
    sa = torch.exp2(torch.randint(-3, 4, (m, 3), generator=g, device="cuda").float())
    for block_b in (1, 128):
        sb = torch.exp2(torch.randint(-3, 4, (n if block_b == 1 else -(-n // 128), 3), generator=g, device="cuda").float())
        got = matmul_op.matmul_fp8(a.to(E4), sa, b.to(E4), sb, out_dtype=torch.float32)
        rows = torch.arange(n, device="cuda") // block_b
        want = b[:, at].t() * sa[torch.arange(m), at // 128][:, None] * sb[rows][:, at // 128].t()
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(7, 512, 1024), (200, 512, 1024), (2304, 2304, 256)])
def test_nan_and_infinity_reach_their_row_and_blocks_of_zeros_nothing(m, n, k):
    x, w = torch.randn(m, k, device="cuda"), torch.randn(n, k, device="cuda")
    x[1, 3], x[2, 130], x[3] = float("nan"), float("inf"), 0.0
    w[:128, :128] = 0
    a, sa = matmul_op.quantize_fp8(x)
    b, sb = matmul_op.quantize_fp8(w, rows=128)
    y = matmul_op.matmul_fp8(a, sa, b, sb)
    matmul_op.matmul_fp8_status()
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any() and torch.all(y[3] == 0)
    rest = [i for i in range(m) if i not in (1, 2)]
    assert torch.isfinite(y[rest]).all()
    x[1, 3], x[2, 130] = 0.0, 0.0
    a, sa = matmul_op.quantize_fp8(x)
    assert torch.equal(matmul_op.matmul_fp8(a, sa, b, sb)[rest], y[rest])


@pytest.mark.gpu
def test_scales_whose_product_leaves_the_range_of_fp32():
    """0 times a product of scales past the largest fp32 number is 0."""
    a, b = torch.zeros((4, 128), device="cuda").to(E4), torch.ones((300, 128), device="cuda").to(E4)
    big = torch.full((4, 1), 2.0 ** 100, device="cuda")
    for m in (4, 200):
        y = matmul_op.matmul_fp8(a[:1].repeat(m, 1), big[:1].repeat(m, 1), b, torch.full((3, 1), 2.0 ** 100, device="cuda"))
        assert torch.all(y == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("m", [4, 40, 200, 2304])
def test_a_large_scale_meets_a_small_one(m, block_b):
    """The largest parts, and the largest scale on either side: exact."""
    n, k = 2304, 256
    a, b = torch.full((m, k), 57344.0, device="cuda").to(E5), torch.full((n, k), 57344.0, device="cuda").to(E5)
    for ea, eb in ((88, -60), (-60, 88)):
        sa = torch.full((m, 2), 2.0 ** ea, device="cuda")
        sb = torch.full((n if block_b == 1 else n // 128, 2), 2.0 ** eb, device="cuda")
        y = matmul_op.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
        assert bool((y == 49 * 2.0 ** (26 + 8 + 28)).all())


@pytest.mark.gpu
def test_operands_and_scales_with_a_pitch():
    m, n, k = 40, 300, 512
    a, sa = operand(m, 2 * k, 1, 0)
    b, sb = operand(n + 128, 2 * k, 128, 1)
    part = matmul_op.matmul_fp8(a[:, k:], sa[:, 4:], b[128:, k:], sb[1:, 4:])
    whole = matmul_op.matmul_fp8(a[:, k:].contiguous(), sa[:, 4:].contiguous(), b[128:, k:].contiguous(), sb[1:, 4:].contiguous())
    assert torch.equal(part, whole)
    with pytest.raises(_lib.KCGError, match="16-byte"):
        matmul_op.matmul_fp8(a[:, 8:k + 8], sa[:, :4], b[:n, :k], sb[:3, :4])


@pytest.mark.gpu
def test_no_tokens():
    b, sb = operand(300, 256, 128, 1)
    y = matmul_op.matmul_fp8(torch.empty((0, 256), device="cuda").to(E4), torch.empty((0, 2), device="cuda"), b, sb)
    assert y.shape == (0, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("block_b", [128, 1])
@pytest.mark.parametrize("k", [128, 640, 200, 1100])
def test_many_tiles_a_pair_and_groups_of_few_blocks(k, block_b):
    """Scales of one to four blocks come together, those of the next group while a group is used; a pair walks about six tiles."""
    a, sa = operand(6144, k, 1, 2)
    b, sb = operand(5120, k, block_b, 3)
    assert _plan(6144, 5120, k, block_b)[0] == 1
    want = wide64(a, sa, 1) @ wide64(b, sb, block_b).t()
    size = wide64(a, sa, 1).abs() @ wide64(b, sb, block_b).abs().t()
    first = matmul_op.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    assert bool(((first.double() - want).abs() <= (2.0 ** -16 + 2.0 ** -20) * size).all())
    for _ in range(5):
        assert torch.equal(matmul_op.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32), first)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    m, n, k = 70000, 32768, 128  # 2.3e9 results
    a, sa = operand(m, k, 1, 0)
    b, sb = operand(n, k, 128, 1)
    y = matmul_op.matmul_fp8(a, sa, b, sb)
    want = matmul_op.matmul_fp8(a[-256:], sa[-256:], b, sb)
    assert torch.equal(y[-256:], want)


def layer(x, r, nw, w8, ws):
    q, s, h = matmul_op.rms_norm_fp8(x, nw, r)
    return matmul_op.matmul_fp8(q, s, w8, ws), h


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 50, 700])
def test_a_layer_captured_replayed_and_on_another_stream(m):
    """Norm, 8-bit product, on new inputs through a captured graph, beside the same on another stream: the bits of plain calls."""
    d, n = 1024, 2304
    w8, ws = operand(n, d, 128, 1)
    nw = torch.rand(d, device="cuda").to(torch.bfloat16)
    xs = [(torch.randn(m, d, device="cuda").to(torch.bfloat16), torch.randn(m, d, device="cuda").to(torch.bfloat16)) for _ in range(6)]
    want = [layer(x, r, nw, w8, ws) for x, r in xs]
    x, r = xs[0][0].clone(), xs[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = layer(x, r, nw, w8, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, beside = [], []
    for i, (a, b) in enumerate(xs):
        x.copy_(a), r.copy_(b)
        graph.replay()
        with torch.cuda.stream(side):
            beside.append(layer(*xs[i], nw, w8, ws))
        got.append((y.clone(), h.clone()))
    torch.cuda.synchronize()
    for results in (got, beside):
        assert all(torch.equal(p[0], q[0]) and torch.equal(p[1], q[1]) for p, q in zip(results, want))
    matmul_op.matmul_fp8_status()


@pytest.mark.gpu
def test_a_training_step_of_a_layer():
    """y = norm(x + r) w^T and its gradients through the five operators, against the same layer in 64 bits. Every 8-bit operand is off by
    2^-4 of a value at most, 2^-5.2 (rms, uniform within a step) of its norm on average; a product of two such is off by sqrt(2) times that of
    the product of their norms, which a sum of K random products makes of the result's norm too: 4 %; 8 % are allowed."""
    m, d, n = 500, 768, 1024
    torch.manual_seed(3)
    x, r = (torch.randn(m, d, device="cuda").to(torch.bfloat16) for _ in range(2))
    nw = (1 + 0.1 * torch.randn(d, device="cuda")).to(torch.bfloat16)
    w = (torch.randn(n, d, device="cuda") / d ** 0.5).to(torch.bfloat16)
    dy = torch.randn(m, n, device="cuda").to(torch.bfloat16)
    q, s, h = matmul_op.rms_norm_fp8(x, nw, r)
    y = matmul_op.matmul_fp8(q, s, *matmul_op.quantize_fp8(w, rows=128))
    u = matmul_op.rms_norm(h, nw)
    du = matmul_op.matmul_fp8(*matmul_op.quantize_fp8(dy), *matmul_op.quantize_fp8(w, rows=128, transposed=True))
    dw = matmul_op.matmul_fp8(*matmul_op.quantize_fp8(dy, transposed=True), *matmul_op.quantize_fp8(u, transposed=True), out_dtype=torch.float32)
    dx, dnw = matmul_op.rms_norm_backward(du, h, nw)
    leaves = [t.double().requires_grad_() for t in (x, nw, w)]
    h64 = leaves[0] + r.double()
    y64 = (h64 * (h64.square().mean(dim=1, keepdim=True) + 1e-6).rsqrt() * leaves[1]) @ leaves[2].t()
    y64.backward(dy.double())
    for got, want in ((y, y64.detach()), (dx, leaves[0].grad), (dnw, leaves[1].grad), (dw, leaves[2].grad)):
        assert (got.double() - want).norm() <= 0.08 * want.norm()
    # the same step adds to a gradient that is there
    twice = matmul_op.matmul_fp8(*matmul_op.quantize_fp8(dy, transposed=True), *matmul_op.quantize_fp8(u, transposed=True), c=dw.clone(), beta=1.0)
    assert (twice - 2 * dw).norm() <= 1e-6 * dw.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("args", [[], ["--backward", "--dtype", "fp32"]])
def test_the_command_runs_and_checks(args, capsys):
    from codegendemo_b200.kcg.run_linear_fp8 import main
    assert main(["--m", "300", "--n", "520", "--k", "768", "--launches", "2", "--warmup", "1"] + args) == 0
    assert "OK" in capsys.readouterr().out


_FIRST_CALL_CAPTURED = """
import torch
from codegendemo_b200.kcg import matmul_op
x = torch.randn(200, 1024, device="cuda").bfloat16()
w = torch.randn(300, 1024, device="cuda").bfloat16()
nw = torch.ones(1024, device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for m in (200, 3):
        h = x[:m]
        q, s, _ = matmul_op.rms_norm_fp8(h, nw, h)
        y = matmul_op.matmul_fp8(q, s, *matmul_op.quantize_fp8(w, rows=128))
        z = matmul_op.rms_norm(h, nw)
        dx, dw = matmul_op.rms_norm_backward(h, h, nw)
        t = matmul_op.quantize_fp8(h, transposed=True)
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
q, s, _ = matmul_op.rms_norm_fp8(x[:3], nw, x[:3])
assert torch.equal(y, matmul_op.matmul_fp8(q, s, *matmul_op.quantize_fp8(w, rows=128)))
assert torch.equal(z, matmul_op.rms_norm(x[:3], nw)) and torch.equal(dx, matmul_op.rms_norm_backward(x[:3], x[:3], nw)[0])
matmul_op.matmul_fp8_status()
print("replayed")
"""


@pytest.mark.gpu
def test_the_first_calls_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", _FIRST_CALL_CAPTURED], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "replayed" in run.stdout, run.stderr[-2000:]


@pytest.mark.gpu
def test_threads_with_streams_of_their_own():
    """Four host threads, each with its stream and inputs, through the whole layer at once: the bits of calls one after another."""
    import threading
    d, n = 768, 1000
    w8, ws = operand(n, d, 128, 9)
    nw = torch.rand(d, device="cuda").to(torch.bfloat16)
    inputs = [(torch.randn(m, d, device="cuda").to(torch.bfloat16), torch.randn(m, d, device="cuda").to(torch.bfloat16)) for m in (1, 40, 300, 2500)]

    def work(x, r):
        y, h = layer(x, r, nw, w8, ws)
        return y, h, *matmul_op.rms_norm_backward(r, h, nw, dh=x), *matmul_op.quantize_fp8(x, transposed=True)
    want = [work(*i) for i in inputs]
    torch.cuda.synchronize()
    got, failed = [None] * 4, []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = work(*inputs[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed
    for p, q in zip(got, want):
        assert all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(p, q))
    matmul_op.matmul_fp8_status()
