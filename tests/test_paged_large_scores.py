"""Scores so large that one of them takes all the weight, up to those that fp32 does not hold."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op

from tests.helpers_paged import Step, assert_close

BF, FP = torch.bfloat16, torch.float16
CASES = [([40], 1, 8, 2, 128, 16, BF), ([14], 8, 8, 2, 64, 16, FP), ([33], [33], 8, 8, 64, 16, BF), ([65, 300], 1, 8, 2, 128, 16, FP),
         ([65, 9000], 1, 8, 2, 128, 1024, BF), ([300], 16, 8, 2, 64, 16, FP), ([500, 90], 4, 8, 1, 128, 32, BF), ([2500], [3], 8, 2, 128, 64, FP),
         ([700, 300] * 40, [200, 300] * 40, 8, 2, 64, 32, FP), ([400], [400], 4, 2, 128, 16, BF)]
ids = [f"{len(c[0])}x{max(c[0])}_{c[1] if isinstance(c[1], int) else max(c[1])}x{c[4]}" for c in CASES]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=ids)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [10, 20, 24, 26, 30, 60, 100, 110])
def test_the_largest_scores_take_all_the_weight(case, power, sign):
    """Whole numbers as queries and keys: scores are exact in fp32, differ by 2^power at least, and the result is the mean of the largest ones' values: their
    weights are equal, exact in 16 bits up to the maximum's lag, and every other one's is below 2^-1400; so what is left is the result's rounding and
    the sums' in fp32 (up to 2^-16 for 2^8 equal scores)."""
    step = Step(*case, seed=power)
    g = torch.Generator(device="cuda").manual_seed(power)
    step.q = (torch.randint(0, 3, step.q.shape, generator=g, device="cuda") * sign).to(step.dtype)
    for b, n in enumerate(step.lens):
        step.k[b] = torch.randint(0, 3, step.k[b].shape, generator=g, device="cuda").to(step.dtype)
        step.put(b)
    got = matmul_op.attention_paged(*step.args(), scale=2.0 ** power)
    matmul_op.attention_paged_status(0)
    group, row = step.q_heads // step.kv_heads, 0
    for b, (n, new) in enumerate(zip(step.lens, step.new)):
        q = step.q[row:row + new].double().view(new, step.kv_heads, group, step.d).permute(1, 2, 0, 3)
        s = q @ step.k[b].double()[:, None].transpose(-1, -2)
        sees = torch.arange(n, device="cuda")[None] <= torch.arange(n - new, n, device="cuda")[:, None]
        s = torch.where(sees, s, float("-inf"))
        w = (s == s.amax(-1, keepdim=True)).double()
        assert int(w.sum(-1).max()) <= 256
        v = step.v[b].double()[:, None]
        want, size = ((w @ x) / w.sum(-1, keepdim=True) for x in (v, v.abs()))
        want, size = (x.permute(2, 0, 1, 3).reshape(new, step.q_heads, step.d) for x in (want, size))
        # (bf16 and fp16 weights of equal scores are one number; sums of them and the values in fp32)
        tol = torch.finfo(step.dtype).eps / 2 * want.abs() + (torch.finfo(step.dtype).eps / 2 + 2.0 ** -16) * size + 2.0 ** -25
        assert_close(got[row:row + new], want, tol)
        row += new


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=ids)
def test_a_row_with_a_score_of_infinity_is_nan(case):
    """A row whose largest score is +inf in fp32 gives NaN (inf - inf), as where the product of the heads is infinite itself, and not the zeros of
    a row without keys; rows whose scores stay small are not touched by it."""
    step = Step(*case, seed=4)
    scale = 2.0 ** 122
    # head 0 and the first key of each sequence: a product of d, that is 2^128 times log2 e or more with the scale; the other heads' rows are zeros
    step.q[:] = 0
    step.q[:, 0] = 1
    for b in range(len(step.lens)):
        step.k[b][:, 0] = 1
        step.put(b)
    got = matmul_op.attention_paged(*step.args(), scale=scale)
    matmul_op.attention_paged_status(0)
    assert bool(got[:, 0].isnan().all())
    step.q[:] = 0
    want, tol = step.oracle(scale=scale)
    got[:, 0] = 0
    want[:, 0] = 0
    assert_close(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES[4:] + [([283, 163, 157], 70, 16, 4, 128, 64, BF)], ids=lambda c: f"{len(c[0])}x{max(c[0])}")
@pytest.mark.parametrize("power", [5, 6, 7, 12, 17, 18, 19, 20])
def test_equal_scores_weigh_the_same_wherever_they_lie(case, power):
    """Every other row has one score many times all over its sequence, its neighbours only late a large one: equal scores share the weight evenly, in the
    tiles before the neighbours' and after. (The two ways to a weight differ by 2^-13 of its exponent; the other terms as above.)"""
    step = Step(*case, seed=power)
    row, group, half_d = 0, step.q_heads // step.kv_heads, step.d // 2
    r = torch.arange(step.q.shape[0] * step.q_heads, device="cuda").view(step.q.shape[0], step.q_heads, 1)
    at = torch.arange(step.d, device="cuda")
    step.q = torch.where(r % 2 == 0, at < 3 + r * 7 % (half_d // 2), at >= half_d).to(step.dtype)
    for b, n in enumerate(step.lens):
        j = torch.arange(n, device="cuda")[:, None]
        step.k[b][:] = torch.where(at < half_d, j % 3 != 1, j >= n - n // 3).to(step.dtype)
        step.put(b)
    got = matmul_op.attention_paged(*step.args(), scale=2.0 ** power)
    matmul_op.attention_paged_status(0)
    half = torch.finfo(step.dtype).eps / 2
    for b, (n, new) in enumerate(zip(step.lens, step.new)):
        q = step.q[row:row + new].double().view(new, step.kv_heads, group, step.d).permute(1, 2, 0, 3)
        s = (q @ step.k[b].double()[:, None].transpose(-1, -2)) * 2.0 ** power
        sees = torch.arange(n, device="cuda")[None] <= torch.arange(n - new, n, device="cuda")[:, None]
        s = torch.where(sees, s, float("-inf"))
        w = torch.softmax(s, -1)
        v = step.v[b].double()[:, None]
        want, size = (x.permute(2, 0, 1, 3).reshape(new, step.q_heads, step.d) for x in (w @ v, w @ v.abs()))
        tol = half * want.abs() + (half + 2 * 2.0 ** -13 + 2.0 ** -16) * size + 2.0 ** -24
        assert_close(got[row:row + new], want, tol)
        row += new
