"""Rows of sequences whose length is negative: no position, whatever the number."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op, paged_op

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("cpp", [False, True])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("ranges", [False, True])
@pytest.mark.parametrize("length", [-1, -5, -2 ** 31 + 1, -2 ** 31])
def test_rows_of_a_negative_length_are_zeros_and_not_stored(length, ranges, given, cpp, monkeypatch):
    """Also where the angles of other positions are given, of which there are some."""
    warm = matmul_op._warm_calls()
    if cpp and not warm:
        pytest.skip("no module of warm calls for this torch")
    monkeypatch.setattr(paged_op, "_warm", warm if cpp else False)
    q, k, v = (torch.randn(4, h, 64, device="cuda").to(BF) for h in (4, 2, 2))
    pools = [torch.zeros(8, 2, 16, 64, dtype=BF, device="cuda") for _ in range(2)]
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lengths = torch.tensor([length, 30], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda") if ranges else None
    positions = torch.tensor([3, 4, 28, 29], dtype=torch.int32, device="cuda") if given else None
    got = matmul_op.append_kv(k, v, *pools, table, lengths, starts, q=q, rotary=matmul_op.rotary_table(64, 64), positions=positions)
    assert bool((got[:2] == 0).all()) and bool((got[2:] != 0).any(-1).all())
    for pool, rows in zip(pools, (k, v)):
        assert bool((pool[5, :, 12:14] != 0).any(-1).all())
        pool[5, :, 12:14] = 0
        assert bool((pool == 0).all())
