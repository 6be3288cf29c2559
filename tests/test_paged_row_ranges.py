"""Row ranges that fall back, overlap, leave the rows or are all empty: which rows are written, and with what."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op

from tests.helpers_paged import Step

BF = torch.bfloat16
ROWS = 16
PATTERNS = [[0, 4, 8, 12, 16], [0, 0, 0, 0, 0], [16, 16, 16, 16, 16], [-5, 3, 9, 12, 1000], [0, 8, 4, 12, 16], [16, 12, 8, 4, 0], [2 ** 31 - 1, -2 ** 31, 0, 5, 7],
            [3, 3, 3, 9, 9], [-2 ** 31, -7, 0, 0, 2 ** 31 - 1]]


def owners(starts):
    """Of each row the (sequence, rows of it, place among them) whose range holds it."""
    s = [min(max(x, 0), ROWS) for x in starts]
    return [[(b, s[b + 1] - s[b], r - s[b]) for b in range(len(s) - 1) if s[b] <= r < s[b + 1]] for r in range(ROWS)]


def test_the_owners_of_rows():
    assert [len(o) for o in owners(PATTERNS[4])] == [1] * 4 + [2] * 4 + [1] * 8 and all(not o for o in owners(PATTERNS[5]))
    assert owners(PATTERNS[3])[0] == [(0, 3, 0)] and owners(PATTERNS[3])[15] == [(3, 4, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(8, 2, 128), (14, 2, 64), (3, 3, 64)], ids=str)
@pytest.mark.parametrize("starts", PATTERNS, ids=str)
def test_rows_that_belong_to_a_sequence_are_its_own_and_others_stay(starts, heads):
    hq, hkv, d = heads
    step = Step([40, 50, 60, 70], [4, 4, 4, 4], hq, hkv, d, 16, BF, seed=3)
    whole = torch.full((ROWS + 4, hq + 2, d), 5.0, dtype=BF, device="cuda")
    out = whole[2:ROWS + 2, 1:hq + 1]
    got = matmul_op.attention_paged(*step.args()[:5], torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    matmul_op.attention_paged_status(0)
    for r, of in enumerate(owners(starts)):
        if not of:
            assert bool((got[r] == 5.0).all()), r
            continue
        fits = torch.zeros(hq, d, dtype=torch.bool, device="cuda")  # (of a row that two sequences have, each value is one's or the other's)
        for b, n, i in of:
            one = Step.__new__(Step)
            one.__dict__.update(step.__dict__)
            one.lens, one.k, one.v, one.new = [step.lens[b] - n + i + 1], [step.k[b][:, :step.lens[b] - n + i + 1]], [step.v[b][:, :step.lens[b] - n + i + 1]], [1]
            one.q = step.q[r:r + 1]
            want, tol = one.oracle()
            fits |= (got[r].double() - want[0]).abs() <= tol[0]
        assert bool(fits.all()), (r, of)
    out.fill_(5.0)
    assert bool((whole == 5.0).all())
