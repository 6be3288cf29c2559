"""The warm calls of the paged cache's operators with results into given places, without queries and without rotation."""
import pytest
import torch

from codegendemo_b200 import build as kbuild
from codegendemo_b200.kcg import matmul_op, paged_op

from tests.helpers_paged import Step

BF, FP = torch.bfloat16, torch.float16
CASES = [([1], 1, 1, 1, 64, 8, BF), ([300, 0, 65], 1, 14, 2, 64, 16, FP), ([300, 20], 4, 32, 8, 128, 64, BF), ([300, 20], [100, 20], 32, 8, 128, 64, BF)]


@pytest.fixture(scope="module")
def warm():
    if kbuild.build_torchcall() is None or not matmul_op._warm_calls():
        pytest.skip("no module of warm calls for this torch")
    return matmul_op._warm_calls()


def bits(t):
    return t.contiguous().view(torch.int16)


def wide(like, fill=7.0):
    """A place for rows x heads x d inside of wider rows, and all of it."""
    rows, heads, d = like.shape
    whole = torch.full((rows, heads + 3, d), fill, dtype=like.dtype, device=like.device)
    return whole[:, 1:heads + 1], whole


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention_into_given_places(warm, monkeypatch, case):
    step = Step(*case)
    for how in (dict(), dict(scale=0.25, window=50, sinks=4)):
        monkeypatch.setattr(paged_op, "_warm", False)
        want = paged_op.attention_paged(*step.args(), **how)
        monkeypatch.setattr(paged_op, "_warm", warm)
        place, whole = wide(step.q)
        assert paged_op.attention_paged(*step.args(), out=place, **how) is place
        assert torch.equal(bits(place), bits(want)) and bool((whole[:, 0] == 7).all()) and bool((whole[:, -2:] == 7).all())
        mine = step.q.clone()
        assert paged_op.attention_paged(mine, *step.args()[1:], out=mine, **how) is mine and torch.equal(bits(mine), bits(want))
        assert warm.attention_paged(*step.args(), how.get("scale"), how.get("window"), how.get("sinks", 0), place) is place


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rows_with_and_without_queries_rotation_and_places(warm, monkeypatch, case):
    step = Step(*case)
    n, hq, hkv, d = sum(step.new), step.q_heads, step.kv_heads, step.d
    qkv = torch.randn(n, hq + 2 * hkv, d, device="cuda").to(step.dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    tables, positions = paged_op.rotary_table(1000, d // 2), torch.arange(n, device="cuda").int()
    for rotary, how in ((None, dict()), (tables, dict()), (tables, dict(interleaved=True)), (tables, dict(positions=positions))):
        for queries in ("none", "new", "in place", "wide"):
            got = []
            for w in (False, warm):
                monkeypatch.setattr(paged_op, "_warm", w)
                pool = [step.k_cache.clone(), step.v_cache.clone()]
                x, more, whole = None, {}, None
                if queries != "none":
                    x = q.clone()
                if queries == "in place":
                    more = dict(q_out=x)
                elif queries == "wide":
                    place, whole = wide(q)
                    more = dict(q_out=place)
                turned = paged_op.append_kv(k, v, *pool, step.table, step.lengths, step.starts, q=x, rotary=rotary, **how, **more)
                assert (turned is None) == (queries == "none") and (not more or turned is more["q_out"])
                got.append([t for t in (turned, whole) if t is not None] + pool)
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(*got))
            taken = warm.append_kv(k, v, *pool, step.table, step.lengths, step.starts, x, rotary, how.get("interleaved", False), how.get("positions"), more.get("q_out"))
            assert taken is (True if queries == "none" else taken) and taken is not None


@pytest.mark.gpu
def test_places_that_do_not_fit_are_refused(warm, monkeypatch):
    monkeypatch.setattr(paged_op, "_warm", warm)
    step = Step([10, 20], 1, 8, 2, 128, 16, BF)
    q, kc, vc, table, lengths, _ = step.args()
    k = torch.zeros(2, 2, 128, dtype=BF, device="cuda")
    rotary = paged_op.rotary_table(100, 128)
    for out in (q[:1], q[:, :4].contiguous(), q.half(), q.cpu(), q[:1].expand(2, 8, 128), q[0], torch.empty(2, 8, 132, dtype=BF, device="cuda")[..., :128],
                torch.empty(2, 8, 136, dtype=BF, device="cuda")[..., 1:129]):
        with pytest.raises(ValueError):
            paged_op.attention_paged(q, kc, vc, table, lengths, out=out)
        for r in (rotary, None):
            with pytest.raises(ValueError):
                paged_op.append_kv(k, k, kc, vc, table, lengths, q=q, rotary=r, q_out=out)
    for wrong in (dict(q_out=q), dict(positions=lengths), dict(q=q[:1]), dict(q=q, rotary=rotary, positions=lengths[:1]), dict(rotary=(rotary[0], rotary[1][:5]))):
        with pytest.raises(ValueError):
            paged_op.append_kv(k, k, kc, vc, table, lengths, **wrong)


@pytest.mark.gpu
def test_given_places_that_share_their_memory_become_their_own(warm, monkeypatch):
    """A lazy clone as the result's place: what it was cloned from stays."""
    monkeypatch.setattr(paged_op, "_warm", warm)
    step = Step([300, 65], 1, 8, 2, 128, 16, BF)
    want = paged_op.attention_paged(*step.args())
    before = step.q.clone()
    mine = step.q._lazy_clone()
    assert paged_op.attention_paged(mine, *step.args()[1:], out=mine) is mine
    assert torch.equal(bits(mine), bits(want)) and torch.equal(bits(step.q), bits(before))
    k, pool = torch.randn(2, 2, 128, device="cuda").to(BF), [step.k_cache.clone(), step.v_cache.clone()]
    rotary = paged_op.rotary_table(400, 128)
    want = paged_op.append_kv(k, k, *pool, step.table, step.lengths, q=step.q, rotary=rotary)
    mine = step.q._lazy_clone()
    assert paged_op.append_kv(k, k, *pool, step.table, step.lengths, q=mine, rotary=rotary, q_out=mine) is mine
    assert torch.equal(bits(mine), bits(want)) and torch.equal(bits(step.q), bits(before))
