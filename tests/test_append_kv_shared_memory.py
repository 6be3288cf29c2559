"""A cache that shares its memory until it is written (a lazy clone) takes a copy of its own first."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op, paged_op

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("cpp", [False, True])
def test_a_lazy_clone_of_a_cache_is_written_the_cache_is_not(cpp, monkeypatch):
    warm = matmul_op._warm_calls()
    if cpp and not warm:
        pytest.skip("no module of warm calls for this torch")
    monkeypatch.setattr(paged_op, "_warm", warm if cpp else False)
    q, k, v = (torch.randn(2, h, 64, device="cuda").to(BF) for h in (4, 2, 2))
    pools = [torch.zeros(8, 2, 16, 64, dtype=BF, device="cuda") for _ in range(2)]
    mine = [p._lazy_clone() for p in pools]
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lengths = torch.tensor([1, 30], dtype=torch.int32, device="cuda")
    rotary = matmul_op.rotary_table(64, 64)
    matmul_op.append_kv(k, v, *mine, table, lengths, q=q, rotary=rotary)
    want = [torch.zeros_like(p) for p in pools]
    matmul_op.append_kv(k, v, *want, table, lengths, q=q, rotary=rotary)
    for pool, own, right in zip(pools, mine, want):
        assert bool((pool == 0).all())
        assert torch.equal(own, right) and bool((own != 0).any())
