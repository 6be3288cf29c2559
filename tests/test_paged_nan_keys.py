"""Keys of NaN reach every row that sees them, whichever CTA they lie in and however little the others' scores leave them."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op

from tests.helpers_paged import Step, assert_close

BF, FP = torch.bfloat16, torch.float16

# (lengths, new rows, query heads, key heads, d, page, type), pages of the table behind the sequences': as many places as choose the form
FORMS = [
    (([65, 640, 700], 1, 8, 2, 128, 16, BF), 0),       # a CTA, or a cluster of few, a (sequence, head)
    (([65, 2048, 700], 1, 8, 2, 128, 16, BF), 0),      # a cluster of up to 16
    (([65, 1000], 1, 2, 2, 64, 32, FP), 32),           # the same, tiles of 128 keys
    (([300, 65], 8, 8, 2, 128, 16, BF), 60),           # 32 rows a key head
    (([300, 65], 16, 8, 2, 128, 16, FP), 60),          # 64 rows
    (([65, 9000], 1, 8, 2, 128, 64, BF), 2000),        # ranges of all sequences' keys
    (([130, 20000], 4, 8, 2, 64, 64, FP), 1000),
    (([2500], [3], 8, 2, 128, 64, BF), 0),             # prompts, the keys of a pair shared by a cluster
    (([700, 300] * 40, [200, 300] * 40, 8, 2, 64, 32, FP), 0),  # prompts, a CTA a pair
]


def ids(c):
    return f"{len(c[0][0])}x{max(c[0][0])}_{c[0][1] if isinstance(c[0][1], int) else max(c[0][1])}x{c[0][4]}_{c[1]}_{str(c[0][6])[6:]}"


def rows_of(step, b):
    """(first row, positions of its rows) of a sequence."""
    return sum(step.new[:b]), torch.arange(step.lens[b] - step.new[b], step.lens[b], device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORMS, ids=ids)
@pytest.mark.parametrize("where", ["first", "last", "64 of the middle", "all behind the first 64", "128 at the end"])
def test_keys_of_nan_reach_the_rows_that_see_them(case, where):
    """NaN in key head 0's keys of one place after the other: its query heads' rows from there on are NaN, all others as they were."""
    step = Step(*case[0], spare_width=1 + case[1])
    group = step.q_heads // step.kv_heads
    want, tol = step.oracle()
    hit = torch.zeros(step.q.shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(step.lens):
        lo, hi = {"first": (0, 1), "last": (n - 1, n), "64 of the middle": (n // 2 & -64, (n // 2 & -64) + 64), "all behind the first 64": (64, n),
                  "128 at the end": ((n - 1) & -128, n)}[where]
        step.k[b][0, lo:hi] = float("nan")
        step.put(b)
        row, positions = rows_of(step, b)
        hit[row:row + step.new[b], :group] = (positions >= lo)[:, None]
    got = matmul_op.attention_paged(*step.args())
    matmul_op.attention_paged_status(0)
    assert bool(hit.any()) and bool(got[hit].isnan().all())
    got[hit], want[hit] = 0, 0
    assert_close(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORMS[:7], ids=ids)
def test_a_key_of_nan_among_keys_of_no_weight(case):
    """All scores behind the first 64 keys lie some 260 powers of two below the largest, one of them is NaN."""
    (lens, _, _, _, d, page, dtype), spare = case
    step = Step(lens, 1, 2, 2, d, page, dtype, spare_width=1 + spare)
    row = 0
    for b, n in enumerate(step.lens):
        # scale x |q| |k| = +-130 ln 2: weights of 2^-260 of the first keys'
        q = step.q[row].float()
        far = q * (130 * 0.6931 * d ** 0.5 / q.square().sum(-1, keepdim=True))
        step.k[b][:] = torch.where(torch.arange(n, device="cuda")[None, :, None] < 64, far[:, None], -far[:, None]).to(dtype)
        step.k[b][0, 64 + (n - 64) // 2] = float("nan")
        step.put(b)
        row += step.new[b]
    got = matmul_op.attention_paged(*step.args())
    matmul_op.attention_paged_status(0)
    assert bool(got[:, 0].isnan().all()) and not bool(got[:, 1].isnan().any())
