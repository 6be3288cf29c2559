"""What run_paged's check of a step's rows sees: queries and keys turned wrongly, rows in a wrong place."""
import os
import subprocess
import sys

import pytest
import torch

from codegendemo_b200.kcg.run_paged import append_errors

BF, FP = torch.bfloat16, torch.float16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def step(dtype, d=64, heads=4, kv=2, page=16, first=10, rows=20, interleaved=False, shift=0, slot_shift=0, head_shift=0, by=None):
    """A plain append of a sequence's rows, with mistakes: neighbours in pairs, positions off, places off, other heads' values, other angles' width."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(rows, h, d, generator=g).to(dtype) for h in (heads, kv, kv))
    a = torch.arange(64, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, by or d, 2, dtype=torch.float64) / (by or d))
    rotary = a.cos().float(), a.sin().float()
    k_cache, v_cache = (torch.randn(6, kv, page, d, generator=g).to(dtype) for _ in range(2))
    table = torch.tensor([4, 1, 3], dtype=torch.int32)
    p = torch.arange(first, first + rows)

    def turn(x):
        c, s = (t[p + shift][:, None].double() for t in rotary)
        y, n = x.double().clone(), 2 * c.shape[-1]
        lo, hi = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
        y[..., lo], y[..., hi] = x[..., lo].double() * c - x[..., hi].double() * s, x[..., hi].double() * c + x[..., lo].double() * s
        return y.to(dtype)
    to = p + slot_shift
    at, slot = table.long()[to // page], to % page
    k_cache[at, :, slot], v_cache[at, :, slot] = turn(k), v.roll(head_shift, 1)
    return q, k, v, turn(q), k_cache, v_cache, table, first, rotary


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("by", [None, 32])
def test_right_rows_are_right(dtype, by):
    off_q, off_k, same = append_errors(*step(dtype, by=by))
    most = torch.finfo(dtype).eps / 2 + 2.0 ** -20
    assert off_q <= most and off_k <= most and same


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
@pytest.mark.parametrize("wrong", [dict(interleaved=True), dict(shift=1), dict(slot_shift=1), dict(slot_shift=-1), dict(head_shift=1)], ids=str)
def test_wrong_rows_are_seen(dtype, wrong):
    off_q, off_k, same = append_errors(*step(dtype, **wrong))
    most = torch.finfo(dtype).eps / 2 + 2.0 ** -20
    assert not (max(off_q, off_k) <= most and same)


def test_queries_that_stayed_as_they_were_are_seen():
    q, *rest = step(BF)
    rest[2] = q
    assert append_errors(q, *rest)[0] > 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("args", ["--batch 3 --length 700", "--batch 2 --length 500 --tokens 300 --window 64 --sinks 4 --dtype fp16 --d 64 --page 16"])
def test_the_command(args):
    r = subprocess.run([sys.executable, "-m", "codegendemo_b200.kcg.run_paged", "--launches", "2", *args.split()], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.count("OK") == 2, r.stdout + r.stderr[-2000:]
