"""Attention over a paged cache against 64 bits, where its splits, tiles, masks and pages can go wrong."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from codegendemo_b200 import _lib
from codegendemo_b200.kcg import matmul_op

from tests.helpers_paged import Step, assert_close

BF, FP = torch.bfloat16, torch.float16

# (lengths, new rows of each (a list: row ranges), query heads, key heads, d, page, type)
TOKENS = [
    ([1], 1, 1, 1, 64, 16, BF), ([1, 0, 2], 1, 4, 2, 128, 16, FP), ([63, 64, 65], 1, 8, 8, 64, 8, BF), ([127, 128, 129, 1], 1, 32, 8, 128, 32, BF),
    ([4097], 1, 32, 8, 128, 16, BF), ([4097], 1, 64, 1, 128, 64, FP), ([2048, 5, 0, 700, 33], 1, 14, 2, 64, 128, FP), ([5000] * 3, 1, 16, 16, 128, 256, BF),
    ([300, 1, 2, 5, 4], 4, 32, 8, 128, 16, BF), ([1000, 77], 5, 24, 8, 64, 32, FP), ([600, 2], 3, 63, 3, 128, 64, BF), ([900], 16, 4, 1, 128, 16, FP),
    ([9000, 300], 2, 24, 2, 128, 64, BF), ([9000, 10], 8, 8, 1, 64, 16, FP), ([30000], 1, 64, 1, 128, 128, BF), ([250] * 7, 1, 8, 1, 128, 32, BF),
    ([130] * 40, 1, 8, 4, 128, 16, BF), ([20000, 1, 64], 1, 8, 2, 64, 1024, BF), ([513] * 150, 1, 3, 3, 64, 16, FP), ([0, 0], 1, 8, 2, 128, 16, BF),
]
PROMPTS = [
    ([1], [1], 1, 1, 64, 16, BF), ([127], [127], 1, 1, 128, 16, BF), ([128, 1, 129], [128, 1, 129], 8, 8, 64, 8, FP), ([300, 0, 257], [300, 0, 257], 32, 8, 128, 32, BF),
    ([1000], [1000], 14, 2, 64, 64, FP), ([777, 40], [100, 40], 5, 1, 128, 16, BF), ([2500], [3], 32, 8, 128, 128, FP), ([50, 60, 9], [60, 60, 12], 12, 4, 64, 16, BF),
    ([700, 300], 100, 8, 2, 128, 16, BF), ([64, 500, 2], 65, 1, 1, 64, 32, FP), ([640, 2, 700], [640, 0, 1], 63, 1, 128, 256, BF), ([3000, 1500], [513, 1500], 4, 4, 128, 64, BF), ([400] * 9, [400] * 9, 3, 1, 64, 32, FP),
    ([5 * i + 1 for i in range(33)], [(7 * i) % (5 * i + 1) for i in range(33)], 8, 8, 64, 16, BF), ([90 - i for i in range(64)], [90 - i for i in range(64)], 4, 1, 128, 16, FP),
    ([40] * 70, 20, 8, 2, 64, 16, BF), ([65 + i for i in range(100)], 65, 1, 1, 128, 16, FP), ([90] * 64, 33, 8, 4, 64, 16, BF),
    ([i % 50 for i in range(65)], [i % 50 for i in range(65)], 8, 2, 64, 8, BF), ([(37 * i) % 200 + 1 for i in range(150)], [(i * i) % ((37 * i) % 200 + 1) for i in range(150)], 32, 8, 128, 32, BF),
]


def ids(c):
    return f"{len(c[0])}x{max(c[0])}_{c[1] if isinstance(c[1], int) else max(c[1])}_{c[2]}of{c[3]}x{c[4]}_p{c[5]}_{str(c[6])[6:]}"


def check(step, **how):
    got = matmul_op.attention_paged(*step.args(), **how)
    matmul_op.attention_paged_status(0)
    assert got.dtype == step.dtype and got.shape == step.q.shape
    assert_close(got, *step.oracle(**how))


@pytest.mark.gpu
@pytest.mark.parametrize("case", TOKENS, ids=ids)
def test_one_or_a_few_new_tokens(case):
    check(Step(*case))


@pytest.mark.gpu
@pytest.mark.parametrize("case", PROMPTS, ids=ids)
def test_prompts(case):
    check(Step(*case))


@pytest.mark.gpu
@pytest.mark.parametrize("case", [TOKENS[4], TOKENS[6], TOKENS[8], TOKENS[13], PROMPTS[4], PROMPTS[5], PROMPTS[6], PROMPTS[8], PROMPTS[11], PROMPTS[7]], ids=ids)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (128, 64), (129, 130), (1000, 3), (100000, 5)])
def test_window_and_sinks(case, window, sinks):
    """What no row sees is NaN, and pages of nothing else are not in the table."""
    step = Step(*case, seed=1)
    want = step.oracle(window=window, sinks=sinks)
    step.hide_unseen(window, sinks)
    got = matmul_op.attention_paged(*step.args(), window=window, sinks=sinks)
    matmul_op.attention_paged_status(0)
    assert_close(got, *want)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [([700, 3], 1, 8, 2, 128, 16, BF), ([700, 300], [333, 300], 8, 2, 64, 32, FP)], ids=ids)
def test_views_and_places_of_results(case):
    """Caches that lie token by token, rows that are parts of wider ones, scales; rows behind the last sequence stay as they were."""
    step = Step(*case, extra_rows=0 if isinstance(case[1], int) else 7)
    want, tol = step.oracle(scale=0.3)
    wide = torch.full((step.q.shape[0], 3 * step.q_heads + 1, step.d), 7.0, dtype=step.dtype, device="cuda")
    q, out = wide[:, :step.q_heads], wide[:, step.q_heads + 1:2 * step.q_heads + 1]
    q.copy_(step.q)
    by_token = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (step.k_cache, step.v_cache)]
    got = matmul_op.attention_paged(q, *by_token, step.table[:, :step.table.shape[1]], step.lengths, step.starts, scale=0.3, out=out)
    assert got is out
    assert_close(got, want, tol)
    behind = want.isnan()
    assert bool((out[behind] == 7.0).all()) and bool((wide[:, 2 * step.q_heads + 1:] == 7.0).all()) and bool((wide[:, step.q_heads] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", [TOKENS[3], TOKENS[9], TOKENS[13], TOKENS[15], PROMPTS[3], PROMPTS[5], PROMPTS[6], PROMPTS[9]], ids=ids)
def test_in_the_queries_place(case):
    step = Step(*case)
    want, tol = step.oracle()
    got = matmul_op.attention_paged(*step.args(), out=step.q)
    matmul_op.attention_paged_status(0)
    assert got is step.q
    assert_close(got, want, tol)


_FIRST_CALL = """
import sys
import torch
from tests.helpers_paged import Step, assert_close
from codegendemo_b200.kcg import matmul_op
step = Step(*eval(sys.argv[1]))
cos, sin = matmul_op.rotary_table(1000, step.d)
k = step.k_cache.clone(), step.v_cache.clone()
rows = sum(step.new)
new = torch.randn(rows, step.kv_heads, step.d, device="cuda").to(step.dtype)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    matmul_op.append_kv(new, new, *k, step.table, step.lengths, step.starts, q=step.q, rotary=(cos, sin))
    out = matmul_op.attention_paged(*step.args())
graph.replay()
torch.cuda.synchronize()
assert_close(out, *step.oracle())
print("the same")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["[700, 3], 1, 8, 2, 128, 16, torch.bfloat16", "[20000, 3], 1, 8, 2, 128, 16, torch.bfloat16", "[700, 300], [300, 300], 8, 2, 64, 16, torch.float16",
                                  "[3000], [1], 8, 2, 128, 16, torch.bfloat16"])
def test_a_first_call_may_be_captured(case):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL, case], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("ranges", [False, True])
def test_what_tables_and_lengths_may_say(ranges):
    """Pages that do not exist read as zeros, lengths past the table end with it; nothing outside is touched."""
    lens = [100, 64, 40]
    step = Step(lens, [1, 1, 1] if ranges else 1, 8, 2, 128, 16, BF, spare_width=0)
    want, tol = step.oracle()
    step.table[0, 2] = 1 << 30
    for x in (step.k[0], step.v[0]):
        x[:, 32:48] = 0
    want, tol = step.oracle()
    got = matmul_op.attention_paged(*step.args())
    assert_close(got, want, tol)
    # 112 places in the table: the row sees them all, wherever its own position is
    step.lengths[1] = 2 ** 31 - 1
    step.table[1] = step.table[0]
    full = torch.zeros(2, 112, 128, dtype=BF, device="cuda")
    step.lens = [100, 112, 40]
    step.k[1], step.v[1] = full.clone(), full.clone()
    at, slot = step.places(1, torch.arange(100))
    ok = (at >= 0) & (at < step.k_cache.shape[0])
    step.k_cache[step.k_cache.isnan()] = 0
    step.v_cache[step.v_cache.isnan()] = 0
    at, slot = step.places(1, torch.arange(112))
    ok = (at >= 0) & (at < step.k_cache.shape[0])
    step.k[1][:, ok] = step.k_cache[at[ok], :, slot[ok]].transpose(0, 1)
    step.v[1][:, ok] = step.v_cache[at[ok], :, slot[ok]].transpose(0, 1)
    got = matmul_op.attention_paged(*step.args())
    assert_close(got, *step.oracle())
    step.lengths[:] = torch.tensor([-5, -2 ** 31, 0], dtype=torch.int32)
    got = matmul_op.attention_paged(*step.args())
    matmul_op.attention_paged_status(0)
    assert bool((got == 0).all())


@pytest.mark.gpu
def test_row_ranges_that_make_no_sense():
    """Ranges that fall back, overlap or leave the rows: every row that has a sequence is some row of it, the others stay; nothing else is touched."""
    step = Step([40, 50, 60, 70], [4, 4, 4, 4], 8, 2, 128, 16, BF)
    for starts in ([0, 8, 4, 12, 16], [-5, 3, 9, 12, 1000], [16, 16, 16, 16, 16], [2 ** 31 - 1, -2 ** 31, 0, 5, 7], [0, 0, 0, 0, 0]):
        out = torch.full_like(step.q, 5.0)
        matmul_op.attention_paged(step.q, step.k_cache, step.v_cache, step.table, step.lengths,
                                  torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
        matmul_op.attention_paged_status(0)
        assert bool(torch.isfinite(out).all())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes a tensor and of more than 2^31 values, the live pages at its end."""
    pages, page = 17000, 128
    for case in (([1000, 130], 1, 8, 8, 128, 128, BF), ([300, 130], [300, 20], 8, 8, 128, 128, BF)):
        step = Step(*case)
        pool_k, pool_v = (torch.empty((pages, 8, page, 128), dtype=BF, device="cuda") for _ in range(2))
        n = step.k_cache.shape[0]
        pool_k[-n:], pool_v[-n:] = step.k_cache, step.v_cache
        table = torch.where(step.table >= 0, step.table + pages - n, step.table)
        got = matmul_op.attention_paged(step.q, pool_k, pool_v, table, step.lengths, step.starts)
        assert_close(got, *step.oracle())
        del pool_k, pool_v


@pytest.mark.gpu
@pytest.mark.parametrize("case", [TOKENS[3], TOKENS[4], TOKENS[6], TOKENS[8], PROMPTS[3], PROMPTS[6]], ids=ids)
def test_the_same_bits_every_time(case):
    step = Step(*case)
    want = matmul_op.attention_paged(*step.args())
    for _ in range(20):
        assert torch.equal(matmul_op.attention_paged(*step.args()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [([900, 64, 300], 1, 8, 2, 128, 16, BF), ([900, 64, 300], [64, 64, 64], 8, 2, 128, 16, BF)], ids=ids)
def test_captured_calls_follow_the_lengths(case):
    """Two graphs captured in one stream, replayed on two at once, over lengths that change between replays."""
    step = Step(*case)
    new = case[1] if isinstance(case[1], int) else 64
    matmul_op.attention_paged(*step.args())
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(matmul_op.attention_paged(*step.args()))
        graphs.append(g)
    full = (step.lens, step.k, step.v)
    for cut in (0, 1, 64 - new, 200):
        step.lens = [max(n - cut, 0) for n in full[0]]
        step.k, step.v = ([x[:, :n] for x, n in zip(xs, step.lens)] for xs in full[1:])
        step.lengths.copy_(torch.tensor(step.lens, dtype=torch.int32))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        want, tol = step.oracle()
        for o in outs:
            assert_close(o, want, tol)


@pytest.mark.gpu
def test_other_streams_at_once():
    steps = [Step([2000 + 7 * i, 100], 1, 8, 2, 128, 16, BF, seed=i) for i in range(4)] + [Step([500 + i], [300], 8, 2, 128, 16, BF, seed=i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    outs = [None] * len(steps)
    for _ in range(10):
        for i, (s, st) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(st):
                outs[i] = matmul_op.attention_paged(*s.args())
    torch.cuda.synchronize()
    for s, o in zip(steps, outs):
        assert_close(o, *s.oracle())


@pytest.mark.gpu
@pytest.mark.parametrize("case", [([900, 64], 1, 8, 2, 128, 16, BF), ([20], 1, 4, 4, 64, 16, FP), ([900, 64], [40, 64], 8, 2, 64, 16, FP), ([3000], [1], 8, 2, 128, 16, BF)], ids=ids)
def test_queries_and_scores_that_are_no_numbers(case):
    """A query of NaN gives NaN, a row by itself; scores of +inf give NaN as the formula's inf - inf does, of -inf no weight."""
    step = Step(*case)
    want, tol = step.oracle()
    step.q[0, 1] = float("nan")
    got = matmul_op.attention_paged(*step.args())
    assert bool(got[0, 1].isnan().all())
    got[0, 1], want[0, 1] = 0, 0
    assert_close(got, want, tol)
    step = Step(*case)
    step.k[0][0, -1], step.q[0, 0] = float("inf"), step.q[0, 0].abs() + 0.25
    step.put(0)
    if sum(step.new) == 1 or step.new[0] == 1:  # (the last key: the first row sees it)
        got = matmul_op.attention_paged(*step.args())
        assert bool(got[0, 0].isnan().all())
    step.q[0, 0] = -step.q[0, 0]
    step.k[0][0, -1] = float("inf")
    got = matmul_op.attention_paged(*step.args())
    step.k[0][0, -1] = 60000.0  # a finite key of no weight, in place of one of none
    want, tol = step.oracle()
    if step.lens[0] > 1:
        assert bool(((got[0, 0].double() - want[0, 0]).abs() <= tol[0, 0]).all())


@pytest.mark.gpu
def test_a_refused_call_leaves_nothing_for_the_next():
    """Calls for a device that is not there, then right ones."""
    lib, gone = _lib.get_lib(), 63
    for case in (([300, 20], 1, 8, 2, 128, 16, BF), ([300, 200], [300, 20], 8, 2, 128, 16, BF)):
        step = Step(*case)
        c = _lib.PagedCache(step.k_cache.data_ptr(), step.v_cache.data_ptr(), (ctypes.c_int64 * 3)(*step.k_cache.stride()[:3]),
                            (ctypes.c_int64 * 3)(*step.v_cache.stride()[:3]), step.table.data_ptr(), step.lengths.data_ptr(),
                            0 if step.starts is None else step.starts.data_ptr(), step.table.stride(0), step.k_cache.shape[0], 16, step.table.shape[1], 2, 2, 128, 62)
        out, room = torch.empty_like(step.q), torch.empty(1 << 23, dtype=torch.uint8, device="cuda")
        a = _lib.PagedQuery(step.q.data_ptr(), out.data_ptr(), (ctypes.c_int64 * 2)(1024, 128), (ctypes.c_int64 * 2)(1024, 128), room.data_ptr(), room.numel(),
                            step.q.shape[0], 8, 0, 0, 128 ** -0.5)
        k = torch.zeros(step.q.shape[0], 2, 128, dtype=BF, device="cuda")
        r = _lib.NewRows(k.data_ptr(), k.data_ptr(), 0, 0, (ctypes.c_int64 * 2)(256, 128), (ctypes.c_int64 * 2)(256, 128))
        r.rows = step.q.shape[0]
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.kcg_attention_paged(gone, stream, ctypes.byref(c), ctypes.byref(a)) != 0
        assert lib.kcg_attention_paged(0, stream, ctypes.byref(c), ctypes.byref(a)) == 0, lib.kcg_last_error()
        assert lib.kcg_append_kv(gone, stream, ctypes.byref(c), ctypes.byref(r)) != 0
        assert lib.kcg_attention_paged_status(gone, (ctypes.c_uint32 * 4)()) != 0
        assert_close(out, *step.oracle())
        a.workspace_bytes = 16
        if step.starts is None:
            assert lib.kcg_attention_paged(0, stream, ctypes.byref(c), ctypes.byref(a)) == _lib.E_BAD_ARG
            assert lib.kcg_attention_paged_workspace(0, ctypes.byref(c), ctypes.byref(a)) > 16
        else:
            assert lib.kcg_attention_paged_workspace(0, ctypes.byref(c), ctypes.byref(a)) == 0
        assert bool(torch.isfinite(matmul_op.attention_paged(*step.args())[:1]).all())


@pytest.mark.gpu
def test_no_rows():
    step = Step([10, 20], 1, 8, 2, 128, 16, BF)
    got = matmul_op.attention_paged(step.q[:0], *step.args()[1:5])
    assert got.shape == (0, 8, 128)
    got = matmul_op.attention_paged(step.q[:0], *step.args()[1:5], torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert got.shape == (0, 8, 128)


class _OnGpu(torch.Tensor):
    is_cuda = True


def _fake(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype).as_subclass(_OnGpu)


def _call(q=None, k=None, v=None, table=None, lengths=None, starts=None, **how):
    matmul_op.attention_paged(_fake(2, 8, 128) if q is None else q, _fake(4, 2, 16, 128) if k is None else k, _fake(4, 2, 16, 128) if v is None else v,
                              _fake(2, 3, dtype=torch.int32) if table is None else table, _fake(2, dtype=torch.int32) if lengths is None else lengths,
                              starts, **how)


@pytest.mark.parametrize("how,message", [
    (dict(k=torch.zeros(4, 2, 16, 128, dtype=BF)), "CUDA"), (dict(k=_fake(4, 2, 16, 128, dtype=torch.float32)), "float16 or bfloat16"),
    (dict(v=_fake(4, 2, 32, 128)), "v_cache"), (dict(k=_fake(4, 2, 16, 96), v=_fake(4, 2, 16, 96)), "64 or 128"),
    (dict(k=_fake(4, 2, 12, 128), v=_fake(4, 2, 12, 128)), "power of two"), (dict(k=_fake(4, 2, 4, 128), v=_fake(4, 2, 4, 128)), "power of two"),
    (dict(q=_fake(2, 7, 128)), "share"), (dict(q=_fake(2, 130, 128)), "share"), (dict(q=_fake(3, 8, 128)), "as many"), (dict(q=_fake(2, 8, 64)), "q must be"),
    (dict(q=_fake(2, 8, 128, dtype=FP)), "q must be"), (dict(q=_fake(2, 8, 256)[..., ::2]), "contiguous"), (dict(q=_fake(2, 8, 132)[..., :128]), "multiples of 8"),
    (dict(q=_fake(2, 1, 128).expand(2, 8, 128)), "strides"), (dict(q=_fake(16, 128)), "rows x heads"), (dict(table=_fake(2, 3, dtype=torch.int64)), "page_table"),
    (dict(table=_fake(3, dtype=torch.int32)), "page_table"), (dict(lengths=_fake(3, dtype=torch.int32)), "lengths"), (dict(starts=_fake(2, dtype=torch.int32)), "starts"),
    (dict(window=0), "window"), (dict(sinks=-1), "sinks"), (dict(scale=0.0), "scale"), (dict(scale=3e38), "scale"), (dict(scale=float("nan")), "scale"), (dict(out=_fake(2, 8, 64)), "out"),
    (dict(k=_fake(4, 2, 16, 129)[..., 1:], v=_fake(4, 2, 16, 128)), "k_cache"),
])
def test_wrong_arguments_are_refused(how, message):
    with pytest.raises(ValueError, match=message):
        _call(**how)


def c_cache(**other):
    c = _lib.PagedCache(4096, 8192, (ctypes.c_int64 * 3)(4096, 2048, 128), (ctypes.c_int64 * 3)(4096, 2048, 128), 64, 64, 0, 3, 4, 16, 3, 2, 2, 128, 62)
    for k, v in other.items():
        setattr(c, k, (ctypes.c_int64 * 3)(*v) if isinstance(v, tuple) else v)
    return c


def test_the_c_entry_refuses_what_it_cannot_take():
    lib = _lib.get_lib()

    def call(cache=None, **other):
        a = _lib.PagedQuery(4096, 8192, (ctypes.c_int64 * 2)(1024, 128), (ctypes.c_int64 * 2)(1024, 128), 0, 0, 2, 8, 0, 0, 0.1)
        for k, v in other.items():
            setattr(a, k, (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v)
        c = c_cache(**(cache or {}))
        got = lib.kcg_attention_paged(0, 0, ctypes.byref(c), ctypes.byref(a))
        assert got == 0 or lib.kcg_attention_paged_workspace(0, ctypes.byref(c), ctypes.byref(a)) == got
        return got
    assert call(rows=0) == 0
    for bad in (dict(Q=0), dict(O=0), dict(Q=4098), dict(q_stride=(1024, 64)), dict(o_stride=(1020, 128)), dict(q_heads=0), dict(q_heads=7), dict(q_heads=130),
                dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(rows=-2), dict(rows=3), dict(workspace=8)):
        assert call(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(K=0), dict(V=0), dict(K=4104), dict(table=0), dict(lengths=0), dict(table=62), dict(page=12), dict(page=4), dict(page=0), dict(pages=0),
                dict(width=0), dict(table_ld=2), dict(sequences=0), dict(kv_heads=0), dict(dtype=4), dict(k_stride=(4096, 2048, 64)),
                dict(v_stride=(4096, 2044, 128)), dict(k_stride=(4096, 1 << 40, 128))):
        assert call(cache=bad) == _lib.E_BAD_ARG, bad
    assert call(cache=dict(d=96)) == _lib.E_BAD_CONFIG
    assert call(cache=dict(width=1 << 28, table_ld=1 << 28)) == _lib.E_TOO_LARGE
    assert lib.kcg_attention_paged(0, 0, None, None) == _lib.E_BAD_ARG
    assert lib.kcg_attention_paged_status(0, None) == _lib.E_BAD_ARG
