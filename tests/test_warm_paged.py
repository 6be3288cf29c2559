"""The warm calls of the paged cache's operators: what they take, and that they give the bits of the operators' own way."""
import pytest
import torch

from codegendemo_b200 import build as kbuild
from codegendemo_b200.kcg import matmul_op, paged_op

from tests.helpers_paged import Step

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def warm():
    if kbuild.build_torchcall() is None or not matmul_op._warm_calls():
        pytest.skip("no module of warm calls for this torch")
    return matmul_op._warm_calls()


def test_everything_but_right_plain_cuda_arguments_goes_the_operators_way(warm):
    x, i = torch.zeros((4, 2, 16, 64), dtype=BF), torch.zeros((2, 3), dtype=torch.int32)
    for a in (x, x[0], x.to("meta"), x.to_sparse(), None, 3, "a", i):
        assert warm.attention_paged(a, a, a, a, a, None, None, None, 0) is None
        assert warm.append_kv(a, a, a, a, a, a, None, a, (a, a), False, None) is None
    assert warm.attention_paged() is None and warm.append_kv(x) is None
    assert warm.append_kv(x, x, x, x, i, i, None, x, None, False, None) is None and warm.append_kv(x, x, x, x, i, i, None, x, (x,), 0, None) is None


def both(monkeypatch, warm, call):
    monkeypatch.setattr(paged_op, "_warm", False)
    want = call()
    monkeypatch.setattr(paged_op, "_warm", warm)
    got = call()
    assert got.dtype == want.dtype and got.shape == want.shape and got.stride() == want.stride() and got.device == want.device
    assert torch.equal(got.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("case", [([1], 1, 1, 1, 64, 8, BF), ([300, 0, 65], 1, 14, 2, 64, 16, FP), ([300, 20], 4, 32, 8, 128, 64, BF), ([300, 20], [100, 20], 32, 8, 128, 64, BF),
                                  ([700], [1], 4, 4, 64, 16, FP)], ids=str)
def test_the_same_results_either_way(warm, monkeypatch, case):
    step = Step(*case)
    for how in (dict(), dict(scale=0.25), dict(window=50, sinks=4), dict(window=1)):
        both(monkeypatch, warm, lambda: paged_op.attention_paged(*step.args(), **how))
        taken = warm.attention_paged(*step.args(), how.get("scale"), how.get("window"), how.get("sinks", 0))
        assert taken is not None
    n, hq, hkv, d = sum(step.new), step.q_heads, step.kv_heads, step.d
    qkv = torch.randn(n, hq + 2 * hkv, d, device="cuda").to(step.dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    positions = torch.arange(n, device="cuda").int()
    for rotary, how in ((d, dict()), (16, dict(interleaved=True)), (d // 2, dict(positions=positions))):
        tables = paged_op.rotary_table(1000, rotary)
        pools = []
        for w in (False, warm):
            monkeypatch.setattr(paged_op, "_warm", w)
            pool = [step.k_cache.clone(), step.v_cache.clone()]
            turned = paged_op.append_kv(k, v, *pool, step.table, step.lengths, step.starts, q=q, rotary=tables, **how)
            pools.append([turned] + pool)
        for a, b in zip(*pools):
            assert a.shape == b.shape and a.stride() == b.stride() and torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))
        assert warm.append_kv(k, v, *pool, step.table, step.lengths, step.starts, q, tables, how.get("interleaved", False), how.get("positions")) is not None


@pytest.mark.gpu
def test_refusals_stay_the_operators(warm, monkeypatch):
    monkeypatch.setattr(paged_op, "_warm", warm)
    step = Step([10, 20], 1, 8, 2, 128, 16, BF)
    q, kc, vc, table, lengths, _ = step.args()
    attend, k = paged_op.attention_paged, torch.zeros(2, 2, 128, dtype=BF, device="cuda")
    cos, sin = paged_op.rotary_table(100, 128)
    wrong = [lambda: attend(q[:1], kc, vc, table, lengths), lambda: attend(q[:, :7], kc, vc, table, lengths), lambda: attend(q.half(), kc, vc, table, lengths),
             lambda: attend(q, kc, vc[:2], table, lengths), lambda: attend(q, kc, vc, table.long(), lengths), lambda: attend(q, kc, vc, table, lengths[:1]),
             lambda: attend(q, kc, vc, table, lengths, lengths), lambda: attend(q, kc, vc, table, lengths, window=0), lambda: attend(q, kc, vc, table, lengths, sinks=-1),
             lambda: attend(q, kc, vc, table, lengths, scale=-1.0), lambda: attend(q, kc[:, :, :12], vc[:, :, :12], table, lengths),
             lambda: attend(q[:1].expand(2, 8, 128), kc, vc, table, lengths), lambda: attend(q, kc.cpu(), vc.cpu(), table, lengths),
             lambda: paged_op.append_kv(k[:1], k, kc, vc, table, lengths, q=q, rotary=(cos, sin)), lambda: paged_op.append_kv(k, k, kc, vc, table, lengths, q=q, rotary=(cos[:, :9], sin[:, :9])),
             lambda: paged_op.append_kv(k, k, kc, vc, table, lengths, q=q, rotary=(cos, sin.double())),
             lambda: paged_op.append_kv(k, k, kc, vc, table, lengths, q=q, rotary=(cos, sin), positions=lengths[:1])]
    for call in wrong:
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_a_mode_that_watches_torch_sees_the_results_made(warm, monkeypatch):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))
    monkeypatch.setattr(paged_op, "_warm", warm)
    step = Step([10, 20], 1, 8, 2, 128, 16, BF)
    with Seen():
        paged_op.attention_paged(*step.args())
    assert any("empty" in n for n in Seen.names)
