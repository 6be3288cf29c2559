"""Storing a step's rows in a paged cache, and the rotation on the way, against 64 bits."""
import ctypes
import os
import re

import pytest
import torch

from codegendemo_b200 import _lib
from codegendemo_b200.kcg import matmul_op

from tests.helpers_paged import Step
from tests.test_paged_attention import BF, FP, _fake, c_cache

# (lengths, new, query heads, key heads, d, page, type), rotated values of a head, interleaved
CASES = [
    (([1], 1, 1, 1, 64, 16, BF), 64, False), (([5, 0, 17], 1, 4, 2, 128, 8, FP), 128, False), (([33] * 40, 1, 32, 8, 128, 16, BF), 128, True),
    (([300, 64, 1], [300, 1, 1], 14, 2, 64, 32, FP), 32, True), (([129, 700], [129, 63], 3, 3, 128, 64, BF), 16, False),
    (([50, 60, 9], [60, 60, 12], 12, 4, 64, 16, BF), 48, False), (([1000] * 3, 5, 63, 1, 128, 128, FP), 112, True), (([2100], [2100], 32, 8, 128, 256, BF), 128, False),
    (([400, 2, 90] * 12, [3, 0, 7] * 12, 8, 8, 64, 16, BF), 64, False),
]


def ids(c):
    (lens, new, hq, hkv, d, page, dt), rotary, inter = c
    return f"{len(lens)}x{max(lens)}_{hq}of{hkv}x{d}_p{page}_r{rotary}{'i' if inter else ''}_{str(dt)[6:]}"


def turned(x, cos, sin, position, interleaved):
    """(rows, heads, d) in 64 bits, and the largest of the products that each value is a sum of."""
    x = x.double()
    half = cos.shape[1]
    i = torch.arange(half, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos.double()[position][:, None], sin.double()[position][:, None]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    size[..., lo], size[..., hi] = (x[..., lo] * c).abs() + (x[..., hi] * s).abs(), (x[..., hi] * c).abs() + (x[..., lo] * s).abs()
    return y, size


def close(got, want, size, dtype):
    """One rounding to 16 bits (of subnormal fp16 values, half their step), and those of two products and a sum in fp32."""
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 3 * 2.0 ** -24 * size * (1 + torch.finfo(dtype).eps) + (2.0 ** -25 if dtype == torch.float16 else 0)
    return bool(((got.double() - want).abs() <= tol).all())


def rows_of(step):
    """Of each row its sequence and position."""
    b = torch.cat([torch.full((n,), i) for i, n in enumerate(step.new)]).long()
    p = torch.cat([torch.arange(l - n, l) for l, n in zip(step.lens, step.new)]).long()
    return b, p


def check(step, rotary, interleaved, k, v, q, call):
    """Runs call() and looks at the whole pools and the queries."""
    pools = [step.k_cache.clone(), step.v_cache.clone()]
    before = [c.clone() for c in pools]
    cos, sin = matmul_op.rotary_table(max(step.lens) + 1, rotary)
    got = call(pools, cos, sin)
    b, p = rows_of(step)
    live = (p >= 0).nonzero()[:, 0].cuda()
    b, p = b.cuda()[live], p.cuda()[live]
    at, slot = step.table.long()[b, p // step.page], p % step.page
    want_k, size_k = turned(k[live], cos, sin, p, interleaved)
    assert close(pools[0][at, :, slot], want_k, size_k, step.dtype)
    assert torch.equal(pools[1][at, :, slot], v[live])
    for pool, old in zip(pools, before):  # nothing else of the pools
        pool[at, :, slot] = old[at, :, slot]
        assert torch.equal(pool.view(torch.int16), old.view(torch.int16))
    if q is not None:
        want_q, size_q = turned(q[live], cos, sin, p, interleaved)
        assert close(got[live], want_q, size_q, step.dtype)
        dead = torch.ones(sum(step.new), dtype=torch.bool, device="cuda")
        dead[live] = False
        assert bool((got[:sum(step.new)][dead] == 0).all())
    else:
        assert got is None


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=ids)
def test_every_shape(case):
    args, rotary, interleaved = case
    step = Step(*args)
    g = torch.Generator(device="cuda").manual_seed(3)
    n, hq, hkv, d = sum(step.new), step.q_heads, step.kv_heads, step.d
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g, device="cuda").to(step.dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    how = dict(interleaved=interleaved)
    check(step, rotary, interleaved, k, v, q, lambda c, cos, sin: matmul_op.append_kv(k, v, *c, step.table, step.lengths, step.starts, q=q, rotary=(cos, sin), **how))
    check(step, rotary, interleaved, k, v, None, lambda c, cos, sin: matmul_op.append_kv(k, v, *c, step.table, step.lengths, step.starts, rotary=(cos, sin), **how))
    # in place, the caches token by token
    mine = q.contiguous()
    pools = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (step.k_cache, step.v_cache)]
    step.k_cache, step.v_cache = pools

    def in_place(c, cos, sin):
        assert c[0].stride() == pools[0].stride()
        out = matmul_op.append_kv(k, v, *c, step.table, step.lengths, step.starts, q=mine, rotary=(cos, sin), q_out=mine, **how)
        assert out is mine
        return out
    check(step, rotary, interleaved, k, v, q, in_place)


@pytest.mark.gpu
def test_without_rotation_and_with_other_positions():
    step = Step([100, 40, 7], [30, 40, 7], 8, 2, 128, 16, BF, extra_rows=3)
    k, v, q = (torch.randn(80, h, 128, device="cuda").to(BF) for h in (2, 2, 8))
    b, p = (x.cuda() for x in rows_of(step))
    at, slot = step.table.long()[b, p // 16], p % 16
    out = torch.full_like(q, 9.0)
    got = matmul_op.append_kv(k, v, step.k_cache, step.v_cache, step.table, step.lengths, step.starts, q=q, q_out=out)
    assert got is out and torch.equal(got[:77], q[:77]) and bool((got[77:] == 9.0).all())
    assert torch.equal(step.k_cache[at, :, slot], k[:77]) and torch.equal(step.v_cache[at, :, slot], v[:77])
    cos, sin = matmul_op.rotary_table(1000, 128)
    positions = torch.randint(0, 1000, (80,), device="cuda").int()
    positions[5], positions[6] = -1, 1000
    got = matmul_op.append_kv(k, v, step.k_cache, step.v_cache, step.table, step.lengths, step.starts, q=q, rotary=(cos, sin), positions=positions)
    ok = torch.ones(77, dtype=torch.bool, device="cuda")
    ok[5:7] = False
    rows = ok.nonzero()[:, 0]
    want, size = turned(q[rows], cos, sin, positions[rows].long(), False)
    assert close(got[rows], want, size, BF)
    want, size = turned(k[rows], cos, sin, positions[rows].long(), False)
    assert close(step.k_cache[at[rows], :, slot[rows]], want, size, BF)
    assert bool(got[5:7].isnan().all()) and bool(step.k_cache[at[5:7], :, slot[5:7]].isnan().all()) and torch.equal(step.v_cache[at, :, slot], v[:77])


@pytest.mark.gpu
def test_places_that_do_not_exist_are_not_written():
    step = Step([30, 30, 30, 30], 2, 4, 2, 64, 16, FP, spare_width=0)
    k, v, q = (torch.randn(8, h, 64, device="cuda").half() for h in (2, 2, 4))
    cos, sin = matmul_op.rotary_table(64, 64)
    step.table[0, 1], step.table[1, 1] = -1, step.k_cache.shape[0]
    step.lengths[2], step.lengths[3] = 34, 2 ** 31 - 1  # 32 places in the table
    old = step.k_cache.clone(), step.v_cache.clone()
    got = matmul_op.append_kv(k, v, step.k_cache, step.v_cache, step.table, step.lengths, q=q, rotary=(cos, sin))
    for c, o in zip((step.k_cache, step.v_cache), old):
        assert torch.equal(c.view(torch.int16), o.view(torch.int16))
    want, size = turned(q[:6], cos, sin, torch.tensor([28, 29, 28, 29, 32, 33], device="cuda"), False)
    assert close(got[:6], want, size, FP) and bool(got[6:].isnan().all())
    for starts in ([5, 3, 1, 0, -4], [0, 100, 2, 4, 2 ** 31 - 1], [-2 ** 31, 8, 8, 8, 8]):
        step.table[:] = 0
        matmul_op.append_kv(k, v, step.k_cache, step.v_cache, step.table, step.lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"), q=q, rotary=(cos, sin))
        for c, o in zip((step.k_cache, step.v_cache), old):
            assert torch.equal(c[1:].view(torch.int16), o[1:].view(torch.int16))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    pages = 17000
    pool_k, pool_v = (torch.zeros((pages, 8, 128, 128), dtype=BF, device="cuda") for _ in range(2))
    table = torch.tensor([[0, pages - 1], [1, pages - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([129, 256], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(2, 8, 128, device="cuda").to(BF) for _ in range(2))
    matmul_op.append_kv(k, v, pool_k, pool_v, table, lengths)
    assert torch.equal(pool_k[-1, :, 0], k[0]) and torch.equal(pool_k[-2, :, 127], k[1]) and torch.equal(pool_v[-1, :, 0], v[0])
    assert int((pool_k != 0).sum()) == int((k != 0).sum()) and int((pool_v != 0).sum()) == int((v != 0).sum())


@pytest.mark.gpu
def test_generating_token_by_token_is_the_prompt_at_once():
    """A layer's path as a server runs it: a prompt appended and attended to in pieces and then token by token, captured in a graph, gives
    what the whole sequence gives in one go; the steps are queued without a wait."""
    torch.manual_seed(0)
    hq, hkv, d, page, total, window, sinks = 8, 2, 128, 16, 300, 64, 4
    cos, sin = matmul_op.rotary_table(total, d)
    q, k, v = (torch.randn(2, total, h, d, device="cuda").to(BF) for h in (hq, hkv, hkv))
    table = torch.randperm(2 * 20, device="cuda").int().view(2, 20)

    def pools():
        return [torch.full((40, hkv, page, d), float("nan"), dtype=BF, device="cuda") for _ in range(2)]
    whole = pools()
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([total, total], [0, total, 2 * total]))
    flat = [x.reshape(2 * total, -1, d) for x in (q, k, v)]
    turned_q = matmul_op.append_kv(flat[1], flat[2], *whole, table, lengths, starts, q=flat[0], rotary=(cos, sin))
    want = [matmul_op.attention_paged(turned_q, *whole, table, lengths, starts, window=w, sinks=s).view(2, total, hq, d) for w, s in ((None, 0), (window, sinks))]
    step = pools()
    got = [torch.zeros_like(want[0]) for _ in range(2)]
    at = 0
    for piece in (100, 37, 120):
        lengths.fill_(at + piece)
        starts.copy_(torch.tensor([0, piece, 2 * piece]))
        part = [x[:, at:at + piece].reshape(2 * piece, -1, d) for x in (q, k, v)]
        tq = matmul_op.append_kv(part[1], part[2], *step, table, lengths, starts, q=part[0], rotary=(cos, sin))
        for i, (w, s) in enumerate(((None, 0), (window, sinks))):
            got[i][:, at:at + piece] = matmul_op.attention_paged(tq, *step, table, lengths, starts, window=w, sinks=s).view(2, piece, hq, d)
        at += piece
    now = [torch.zeros(2, h, d, dtype=BF, device="cuda") for h in (hq, hkv, hkv)]
    outs = [torch.zeros(2, hq, d, dtype=BF, device="cuda") for _ in range(2)]

    def token():
        lengths.add_(1)
        tq = matmul_op.append_kv(now[1], now[2], *step, table, lengths, q=now[0], rotary=(cos, sin))
        for i, (w, s) in enumerate(((None, 0), (window, sinks))):
            matmul_op.attention_paged(tq, *step, table, lengths, window=w, sinks=s, out=outs[i])
    lengths.fill_(at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token()
    lengths.fill_(at)
    for p in range(at, total):
        for x, y in zip(now, (q, k, v)):
            x.copy_(y[:, p])
        if p % 2:
            graph.replay()
        else:
            token()
        for i in range(2):
            got[i][:, p] = outs[i]
    matmul_op.attention_paged_status(0)
    for a, b in zip(step, whole):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    # each off by the weights' rounding (2^-8 of the largest |v| at most) and its own, twice
    for a, b in zip(got, want):
        assert float((a.float() - b.float()).abs().max()) <= 4 * 2.0 ** -8 * float(v.abs().max())


SOURCES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "codegendemo_b200", "csrc")


@pytest.mark.parametrize("file", ["kcg_paged.cu", "paged.cuh", "paged_tokens.cuh", "paged_prompt.cuh", "attn_common.cuh"])
def test_no_load_asks_for_memory_that_is_read_only_for_the_kernels_life(file):
    """The kernel before in the stream may still write what these read (programmatic dependent launch)."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(SOURCES, file)).read())
    assert re.findall(r"__ldg\s*\(|ld\.global\.nc|__restrict__", text) == []


def test_table_of_angles():
    cos, sin = matmul_op.rotary_table(100001, 64, base=500000.0, device="cpu")
    assert cos.shape == sin.shape == (100001, 32) and cos.dtype == torch.float32
    import math
    for p, i in ((0, 0), (1, 5), (100000, 0), (99999, 31)):
        a = p * 500000.0 ** (-2 * i / 64)
        assert abs(cos[p, i].item() - math.cos(a)) <= 2.0 ** -24 and abs(sin[p, i].item() - math.sin(a)) <= 2.0 ** -24
    for bad in ((0, 64), (10, 7), (10, 0)):
        with pytest.raises(ValueError):
            matmul_op.rotary_table(*bad, device="cpu")


def _call(k=None, v=None, q=None, **how):
    return matmul_op.append_kv(_fake(2, 2, 128) if k is None else k, _fake(2, 2, 128) if v is None else v, _fake(4, 2, 16, 128), _fake(4, 2, 16, 128),
                               _fake(2, 3, dtype=torch.int32), _fake(2, dtype=torch.int32), q=q, **how)


def _angles(rows=10, half=64, dtype=torch.float32):
    return _fake(rows, half, dtype=dtype), _fake(rows, half, dtype=dtype)


@pytest.mark.parametrize("how,message", [
    (dict(k=_fake(2, 3, 128)), "k must be"), (dict(v=_fake(3, 2, 128)), "v must be"), (dict(k=_fake(2, 2, 64)), "k must be"), (dict(k=_fake(2, 256)), "dimensions"),
    (dict(k=_fake(3, 2, 128), v=_fake(3, 2, 128)), "as many"), (dict(v=_fake(2, 2, 128, dtype=FP)), "v must be"), (dict(q_out=_fake(2, 8, 128)), "without q"),
    (dict(q=_fake(3, 8, 128)), "q must be"), (dict(q=_fake(2, 0, 128)), "no heads"), (dict(q=_fake(2, 8, 128), q_out=_fake(2, 4, 128)), "q_out"),
    (dict(q=_fake(2, 8, 128), q_out=_fake(1, 8, 128).expand(2, 8, 128)), "strides"), (dict(positions=_fake(2, dtype=torch.int32)), "without rotary"),
    (dict(rotary=_angles(half=60)), "multiple of 16"), (dict(rotary=_angles(half=72)), "multiple of 16"), (dict(rotary=_angles(half=0)), "multiple of 16"),
    (dict(rotary=_angles(dtype=BF)), "float32"), (dict(rotary=_angles(), positions=_fake(3, dtype=torch.int32)), "positions"),
    (dict(rotary=_angles(), positions=_fake(2, dtype=torch.int64)), "positions"), (dict(rotary=(_fake(9, 64, dtype=torch.float32), _fake(10, 64, dtype=torch.float32))), "sin"),
])
def test_wrong_arguments_are_refused(how, message):
    with pytest.raises(ValueError, match=message):
        _call(**how)


def test_the_c_entry_refuses_what_it_cannot_take():
    lib = _lib.get_lib()

    def call(cache=None, **other):
        two = (ctypes.c_int64 * 2)(1024, 128)
        r = _lib.NewRows(4096, 4096, 4096, 4096, two, two, two, two, 4096, 4096, 0, 10, 2, 8, 64, 0)
        for k, v in other.items():
            setattr(r, k, (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v)
        c = c_cache(**(cache or {}))
        return lib.kcg_append_kv(0, 0, ctypes.byref(c), ctypes.byref(r))
    assert call(rows=0) == 0
    for bad in (dict(K=0), dict(V=0), dict(QO=0), dict(Q=0), dict(K=4104), dict(q_heads=0), dict(k_stride=(1024, 64)), dict(v_stride=(1020, 128)), dict(q_stride=(8, 128)),
                dict(qo_stride=(1024, 1 << 41)), dict(rotary=-16), dict(rotary=144), dict(rotary=24), dict(cos=0), dict(sin=0), dict(angles=0), dict(cos=4100),
                dict(positions=2), dict(rows=-1), dict(rows=3)):
        assert call(**bad) == _lib.E_BAD_ARG, bad
    assert call(cache=dict(page=24)) == _lib.E_BAD_ARG and call(cache=dict(d=32)) == _lib.E_BAD_CONFIG
    assert lib.kcg_append_kv(0, 0, None, None) == _lib.E_BAD_ARG
