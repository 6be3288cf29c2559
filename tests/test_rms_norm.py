"""Root-mean-square norm, forward (in the rows' type and in 8 bits) and backward, against its formula in 64 bits.

Tolerances, u = 2^-24: a row's sum of squares has positive terms and goes through at most 128 additions in a thread (32768 values, 256
threads) and 10 in the exchange, so it is off by 138 u of itself and the root by half of that; with the root's, the mean's and the
products' roundings a norm is off by less than 80 u of itself before its last rounding (half a step of its type).
"""
import pytest
import torch

from codegendemo_b200 import _lib
from codegendemo_b200.kcg import matmul_op

U = 2.0 ** -24
EPS = 1e-6
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# (rows, width): one value; a warp a row, its pieces full and not; a CTA a row; two and four pieces a thread; widths and rows
# that are no whole pieces; the widest
SHAPES = [(1, 1), (3, 8), (9, 120), (1, 256), (17, 264), (8, 1000), (5, 1024), (7, 1032), (33, 2752), (2, 4096), (3, 5504), (2, 16384),
          (2, 16392), (1, 32768), (4, 7), (6, 129), (3, 1781), (2, 5507), (1, 32767)]


def rows_of(rows, width, dtype, seed, size=1.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (size * torch.randn(rows, width, generator=g, device=device)).to(dtype)


def norm64(h, w, eps=EPS):
    return h * (h.square().mean(dim=1, keepdim=True) + eps).rsqrt() * w.double()


def half_step(t, dtype):
    """Half a step of the type at the values t, those below its smallest normal number included."""
    info = torch.finfo(dtype)
    return (t.abs() * (info.eps / 2)).clamp(min=info.smallest_normal * info.eps / 2)


def near(got, want, dtype, relative=80 * U):
    off = (got.double() - want).abs()
    allowed = half_step(want, dtype) * (1 + 2 * relative) + relative * want.abs()
    assert bool((off <= allowed).all()), f"off by {(off / allowed.clamp(min=1e-300)).max().item():.3f} of what is allowed"


def near_fp8(q, scales, want, relative=80 * U):
    """8-bit values and scales of `want` in blocks of 1 x 128: half a step of e4m3 (2^-4 of a value, 2^-10 below 2^-6)."""
    r, c = want.shape
    nb = -(-c // 128)
    assert scales.shape == (r, nb) and q.shape == (r, c) and q.dtype == torch.float8_e4m3fn
    full = torch.zeros((r, nb * 128), dtype=torch.float64, device=want.device)
    full[:, :c] = want
    top = full.view(r, nb, 128).abs().amax(dim=2)
    s = (top / 448).clamp(min=2.0 ** -126)
    assert bool(((scales.double() - s).abs() <= (relative + 4 * U) * s).all())
    s = scales.double().repeat_interleave(128, 1)[:, :c]
    off = (q.double() * s - want).abs()
    allowed = s * torch.maximum(want.abs() / s * 2.0 ** -4, torch.full_like(s, 2.0 ** -10)) * (1 + 1e-5) + 2 * relative * want.abs()
    assert bool((off <= allowed).all())


def test_refusals():
    x, w = torch.zeros((4, 16)), torch.zeros(16)
    for f in (matmul_op.rms_norm, matmul_op.rms_norm_fp8, lambda x, w: matmul_op.rms_norm_backward(x, x, w)):
        with pytest.raises(ValueError, match="CUDA"):
            f(x, w)


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is a CUDA one: whatever is refused, is refused before memory is touched."""
    is_cuda = True


def _fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_OnGpu)


@pytest.mark.parametrize("call,message", [
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(15)), "weight"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(16, dtype=torch.float32)), "weight"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(32)[::2]), "weight"),
    (lambda: matmul_op.rms_norm(_fake(4, 16, dtype=torch.float64), _fake(16, dtype=torch.float64)), "float32"),
    (lambda: matmul_op.rms_norm(_fake(16), _fake(16)), "2-D"),
    (lambda: matmul_op.rms_norm(_fake(4, 32)[:, ::2], _fake(16)), "contiguous rows"),
    (lambda: matmul_op.rms_norm(_fake(1, 16).expand(4, 16), _fake(16)), "overlap"),
    (lambda: matmul_op.rms_norm(_fake(4, 0), _fake(0)), "1 to 32768"),
    (lambda: matmul_op.rms_norm(_fake(1, 32769), _fake(32769)), "1 to 32768"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(16), eps=-1.0), "eps"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(16), eps=float("nan")), "eps"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(16), _fake(3, 16)), "residual"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(16), _fake(4, 16, dtype=torch.float16)), "residual"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(16), residual_out=_fake(4, 16)), "residual_out without"),
    (lambda: matmul_op.rms_norm(_fake(4, 16), _fake(16), out=_fake(4, 17)), "out"),
    (lambda: matmul_op.rms_norm_fp8(_fake(4, 16), _fake(16), _fake(4, 16), residual_out=_fake(4, 8)), "residual_out"),
    (lambda: matmul_op.rms_norm_backward(_fake(4, 8), _fake(4, 16), _fake(16)), "dy"),
    (lambda: matmul_op.rms_norm_backward(_fake(4, 16), _fake(4, 16), _fake(16), dh=_fake(5, 16)), "dh"),
])
def test_wrong_arguments_are_refused(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_the_same_tensor_for_both_results_is_refused():
    x, w, y = _fake(4, 16), _fake(16), _fake(4, 16)
    with pytest.raises(ValueError, match="different tensors"):
        matmul_op.rms_norm(x, w, x, out=y, residual_out=y)


def test_the_c_entries_refuse_what_they_cannot_take():
    """Before any device is touched."""
    lib = _lib.get_lib()
    ok = dict(rows=4, width=16, eps=1e-6, dtype=62)

    def norm(X=256, ldx=0, R=0, ldr=0, W=256, Y=256, ldy=0, H=0, ldh=0, **kw):
        kw = {**ok, **kw}
        return lib.kcg_rms_norm(0, 0, X, ldx, R, ldr, W, Y, ldy, H, ldh, kw["rows"], kw["width"], kw["eps"], kw["dtype"])
    assert norm(rows=0) == 0
    for bad in (dict(X=0), dict(W=0), dict(Y=0), dict(R=256), dict(H=256), dict(ldx=8), dict(X=257), dict(rows=-1), dict(width=0),
                dict(width=40000), dict(dtype=1), dict(eps=-1.0), dict(eps=float("inf"))):
        assert norm(**bad) == _lib.E_BAD_ARG, bad
    assert lib.kcg_rms_norm_fp8(0, 0, 256, 0, 0, 0, 256, 256, 0, 0, 0, 0, 4, 16, 1e-6, 62) == _lib.E_BAD_ARG  # no scales
    assert lib.kcg_rms_norm_backward(0, 0, 256, 0, 256, 0, 256, 0, 0, 256, 0, 256, 0, 0, 4, 16, 1e-6, 62) == _lib.E_BAD_ARG
    assert lib.kcg_rms_norm_backward(0, 0, 256, 0, 256, 0, 256, 0, 0, 256, 0, 256, 256, 64, 0, 16, 1e-6, 62) == _lib.E_BAD_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_forward(rows, width, dtype):
    x, r, w = rows_of(rows, width, dtype, 1), rows_of(rows, width, dtype, 2, 3.0), rows_of(1, width, dtype, 3)[0]
    near(matmul_op.rms_norm(x, w, eps=EPS), norm64(x.double(), w), dtype)
    y, h = matmul_op.rms_norm(x, w, r, eps=EPS)
    h64 = x.double() + r.double()
    near(h, h64, dtype, U)
    # (a sum that cancels is off by u of itself: one rounding)
    near(y, norm64(h64, w), dtype)
    near_fp8(*matmul_op.rms_norm_fp8(x, w, eps=EPS), norm64(x.double(), w))
    q, s, h8 = matmul_op.rms_norm_fp8(x, w, r, eps=EPS)
    assert torch.equal(h8, h)
    near_fp8(q, s, norm64(h64, w))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", [509, 511, 513, 2047, 2049, 4095, 4097, 8191, 8193, 12001, 16383, 16385])
def test_rows_of_no_whole_pieces_either_side_of_each_form(width, dtype):
    test_forward(3, width, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [512, 2048, 4096, 8192, 16384])
def test_rows_that_start_anywhere(width):
    """Whole pieces, but no row on a 16-byte boundary; written over x and over the residual."""
    x = rows_of(5, width + 1, torch.bfloat16, 1)[:, 1:]
    r = rows_of(5, width + 1, torch.bfloat16, 2)[:, 1:]
    w = rows_of(1, width, torch.bfloat16, 3)[0]
    h64 = x.double() + r.double()
    q, scales, h = matmul_op.rms_norm_fp8(x, w, r, eps=EPS)
    near_fp8(q, scales, norm64(h64, w))
    y, h2 = matmul_op.rms_norm(x, w, r, eps=EPS, out=x, residual_out=r)
    assert torch.equal(h2, h) and h2.data_ptr() == r.data_ptr() and y.data_ptr() == x.data_ptr()
    near(y, norm64(h64, w), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", SHAPES + [(513, 1376), (1000, 264), (700, 129)])
def test_backward_against_the_formula(rows, width, dtype):
    """dx: two terms whose difference may be small, each off by 100 u of itself (80 of the root's, and the second sum's 140 u of
    its terms' magnitudes). dw: a sum over rows of terms off by 80 u, in at most rows additions."""
    h, dy, dh = (rows_of(rows, width, dtype, s) for s in (1, 2, 3))
    w = rows_of(1, width, dtype, 4)[0]
    for extra in (None, dh):
        dx, dw = matmul_op.rms_norm_backward(dy, h, w, eps=EPS, dh=extra)
        h64, g = h.double(), dy.double() * w.double()
        r = (h64.square().mean(dim=1, keepdim=True) + EPS).rsqrt()
        t1, t2 = r * g, h64 * r ** 3 * (g * h64).mean(dim=1, keepdim=True)
        worst = (r * g).abs() * 100 * U + (h64 * r ** 3).abs() * (g * h64).abs().mean(dim=1, keepdim=True) * 300 * U
        want = t1 - t2 + (0 if extra is None else extra.double())
        allowed = half_step(want, dtype) + worst * (1 + 2 * torch.finfo(dtype).eps) + 2 * U * want.abs()
        assert bool(((dx.double() - want).abs() <= allowed).all())
        terms = dy.double() * h64 * r
        want = terms.sum(dim=0)
        allowed = half_step(want, dtype) + (rows + 100) * U * terms.abs().sum(dim=0) * (1 + torch.finfo(dtype).eps)
        assert bool(((dw.double() - want).abs() <= allowed).all())
        again = matmul_op.rms_norm_backward(dy, h, w, eps=EPS, dh=extra)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.gpu
def test_backward_against_differences():
    """(f(h + t d) - f(h - t d)) / 2t of f = sum(c * norm(h)) in 64 bits, t = 1e-5: off by t^2 / 6 of a third derivative of order f's, 1e-10."""
    torch.manual_seed(0)
    rows, width = 5, 264
    h, w, c = (torch.randn(n, width, dtype=torch.float32, device="cuda") for n in (rows, 1, rows))
    dx, dw = matmul_op.rms_norm_backward(c, h, w[0], eps=EPS)
    f = lambda h, w: (c.double() * norm64(h, w)).sum()  # noqa: E731
    for _ in range(4):
        d, e = torch.randn_like(h).double(), torch.randn_like(w).double()
        t = 1e-5
        along = (f(h.double() + t * d, w[0].double() + t * e[0]) - f(h.double() - t * d, w[0].double() - t * e[0])) / (2 * t)
        got = (dx.double() * d).sum() + (dw.double() * e[0]).sum()
        assert abs((got - along).item()) <= 1e-4  # 1320 terms of order 1, each off by 300 u


@pytest.mark.gpu
@pytest.mark.parametrize("width", [256, 1040, 129])
def test_views_with_a_pitch_and_results_in_place(width):
    wide = rows_of(6, 2 * width + 48, torch.bfloat16, 5)
    x, r = wide[:, 8:8 + width], wide[:, width + 16:2 * width + 16]
    w = rows_of(1, width, torch.bfloat16, 6)[0]
    y, h = matmul_op.rms_norm(x.contiguous(), w, r.contiguous())
    into = torch.full((6, width + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    before = wide.clone()
    out = matmul_op.rms_norm(x, w, r, out=into[:, 8:8 + width], residual_out=r)
    assert out[1] is r and torch.equal(out[0], y) and torch.equal(r, h)
    assert torch.all(into[:, :8] == 7) and torch.all(into[:, 8 + width:] == 7)
    before[:, width + 16:2 * width + 16] = h
    assert torch.equal(wide, before)
    x2, r2 = x.contiguous(), (before[:, width + 16:2 * width + 16]).contiguous()
    want = matmul_op.rms_norm(x2, w, r2)
    got = matmul_op.rms_norm(x2, w, r2, out=x2, residual_out=r2)
    assert got[0] is x2 and torch.equal(x2, want[0]) and torch.equal(r2, want[1])
    q, s = matmul_op.rms_norm_fp8(x, w)
    q2, s2 = matmul_op.rms_norm_fp8(x.contiguous(), w)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    dx, dw = matmul_op.rms_norm_backward(x, r, w)
    dx2, dw2 = matmul_op.rms_norm_backward(x.contiguous(), r.contiguous(), w)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [128, 2048, 333])
def test_rows_of_zeros_infinities_and_nan_stay_by_themselves(width):
    x = rows_of(5, width, torch.float32, 7)
    w = torch.ones(width, device="cuda")
    clean = matmul_op.rms_norm(x, w)
    x[1], x[2, 3], x[3, 5] = 0.0, float("inf"), float("nan")
    y = matmul_op.rms_norm(x, w)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[4], clean[4]) and torch.all(y[1] == 0)
    assert torch.isnan(y[2, 3]) and torch.all(torch.isnan(y[3]))
    q, s = matmul_op.rms_norm_fp8(x, w)
    assert torch.all(q[1].float() == 0) and torch.all(s[1] == 2.0 ** -126) and torch.all(torch.isnan(s[3])) and torch.all(torch.isnan(q[3].float()))
    assert torch.isnan(s[2, 0]) and torch.isfinite(s[[0, 1, 4]]).all()
    assert torch.all(torch.isfinite(matmul_op.rms_norm(x, w, eps=0.0)[[0, 4]]))


@pytest.mark.gpu
def test_no_rows():
    x, w = torch.empty((0, 64), device="cuda"), torch.ones(64, device="cuda")
    assert matmul_op.rms_norm(x, w).shape == (0, 64)
    y, h = matmul_op.rms_norm(x, w, x)
    assert y.shape == h.shape == (0, 64)
    q, s, h = matmul_op.rms_norm_fp8(x, w, x)
    assert q.shape == h.shape == (0, 64) and s.shape == (0, 1)
    dx, dw = matmul_op.rms_norm_backward(x, x, w)
    assert dx.shape == (0, 64) and torch.all(dw == 0)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    rows, width = 131080, 16384  # 2.1e9 values
    x = torch.zeros((rows, width), dtype=torch.bfloat16, device="cuda")
    x[-3:] = rows_of(3, width, torch.bfloat16, 8)
    w = torch.ones(width, dtype=torch.bfloat16, device="cuda")
    y = matmul_op.rms_norm(x, w)
    near(y[-3:], norm64(x[-3:].double(), w), torch.bfloat16)
    del y
    q, s = matmul_op.rms_norm_fp8(x, w)
    near_fp8(q[-3:], s[-3:], norm64(x[-3:].double(), w))
    del q, s
    dx, _ = matmul_op.rms_norm_backward(x, x, w)
    want = matmul_op.rms_norm_backward(x[-3:], x[-3:], w)[0]
    assert torch.equal(dx[-3:], want) and torch.all(dx[:4] == 0)
