"""Caches, rows and the 64-bit oracle for the tests of the paged cache."""
import torch


class Step:
    """A cache of sequences and a step's rows. Every place of the pool that no live token has is NaN, pages lie anywhere in it."""

    def __init__(self, lengths, new, q_heads, kv_heads, d, page, dtype, seed=0, ragged=None, spare_width=1, spare_pages=2, extra_rows=0, device="cuda"):
        """``new``: rows of each sequence (a list), or one number for all (no row ranges unless ``ragged``)."""
        g = torch.Generator(device=device).manual_seed(seed)
        self.page, self.d, self.dtype, self.q_heads, self.kv_heads = page, d, dtype, q_heads, kv_heads
        self.lens = list(lengths)
        self.new = list(new) if isinstance(new, (list, tuple)) else [new] * len(self.lens)
        ragged = isinstance(new, (list, tuple)) if ragged is None else ragged
        used = [-(-n // page) for n in self.lens]
        pages = sum(used) + spare_pages
        order = torch.randperm(pages, generator=g, device=device).int()
        self.table = torch.full((len(used), max(used + [1]) + spare_width), -1, dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k_cache, self.v_cache = (torch.full((pages, kv_heads, page, d), float("nan"), dtype=dtype, device=device) for _ in range(2))
        self.k = [torch.randn(kv_heads, n, d, generator=g, device=device).to(dtype) for n in self.lens]
        self.v = [torch.randn(kv_heads, n, d, generator=g, device=device).to(dtype) for n in self.lens]
        for b in range(len(self.lens)):
            self.put(b)
        rows = sum(self.new) + extra_rows
        self.q = (2 * torch.randn(rows, q_heads, d, generator=g, device=device)).to(dtype)
        self.lengths = torch.tensor(self.lens, dtype=torch.int32, device=device)
        starts = [sum(self.new[:b]) for b in range(len(self.new) + 1)]
        self.starts = torch.tensor(starts, dtype=torch.int32, device=device) if ragged else None

    def places(self, b, positions):
        """(pages, slots) of positions of sequence b."""
        p = torch.as_tensor(positions, device=self.table.device)
        return self.table[b].long()[p // self.page], p % self.page

    def put(self, b):
        n = self.lens[b]
        if n:
            at, slot = self.places(b, torch.arange(n))
            self.k_cache[at, :, slot] = self.k[b].transpose(0, 1)
            self.v_cache[at, :, slot] = self.v[b].transpose(0, 1)

    def hide_unseen(self, window, sinks):
        """What no row of a sequence sees: NaN in the cache, and pages of nothing else out of the table."""
        for b, (n, new) in enumerate(zip(self.lens, self.new)):
            first = max(n - new, 0) - window + 1
            if first <= sinks:
                continue
            at, slot = self.places(b, torch.arange(sinks, first))
            self.k_cache[at, :, slot] = float("nan")
            self.v_cache[at, :, slot] = float("nan")
            lo, hi = -(-sinks // self.page), first // self.page
            if hi > lo:
                bad = torch.tensor([-1, self.k_cache.shape[0], 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=self.table.device)
                self.table[b, lo:hi] = bad.repeat(-(-(hi - lo) // 4))[:hi - lo]

    def args(self):
        return self.q, self.k_cache, self.v_cache, self.table, self.lengths, self.starts

    def oracle(self, scale=None, window=None, sinks=0):
        """(result, tolerance) in 64 bits, both (rows, heads, d); rows behind the last sequence: NaN.

        With A = sum of weights x |v| over the weights' sum, the result is off by: its own rounding, eps / 2 of it; the rounding of each
        weight to 16 bits, eps / 2 of A (fp16: and 2^-25 for each weight that is below its normal range, against the largest of 1); scores in
        fp32, of products summed 16 at a time, (d / 16 + 8) 2^-23 of the sum of |q k| each, twice (numerator and denominator), and the
        exponential's 2^-21; sums over the keys, 16 at a time, length / 16 + 64 roundings of 2^-23, twice.
        """
        scale = self.d ** -0.5 if scale is None else scale
        group = self.q_heads // self.kv_heads
        out = torch.full(self.q.shape, float("nan"), dtype=torch.float64, device=self.q.device)
        tol = torch.zeros_like(out)
        half = torch.finfo(self.dtype).eps / 2
        row = 0
        for b, (n, new) in enumerate(zip(self.lens, self.new)):
            out[row:row + new] = 0
            if n and new:
                q = self.q[row:row + new].double().view(new, self.kv_heads, group, self.d).permute(1, 2, 0, 3)
                k, v = self.k[b].double()[:, None], self.v[b].double()[:, None]
                p = torch.arange(n - new, n, device=q.device)[:, None]
                j = torch.arange(n, device=q.device)[None]
                sees = j <= p
                if window:
                    sees = sees & ((p - j < window) | (j < sinks))
                s = torch.where(sees, (q @ k.transpose(-1, -2)) * scale, float("-inf"))
                top = s.amax(-1, keepdim=True)
                w = torch.exp(s - torch.where(top.isinf(), 0.0, top))
                total = w.sum(-1, keepdim=True)
                w = torch.where(total > 0, w / total, 0.0)
                o, a = w @ v, w @ v.abs()
                score = (torch.where(sees, q.abs() @ k.abs().transpose(-1, -2), 0.0) * scale).amax(-1, keepdim=True)
                t = half * (o.abs() + a) + a * (2 * score * (self.d / 16 + 8) * 2.0 ** -23 + 2.0 ** -20 + 2 * (n / 16 + 64) * 2.0 ** -23)
                if self.dtype == torch.float16:
                    t = t + 2.0 ** -25 * torch.where(total > 0, sees.sum(-1, keepdim=True) / total.clamp(min=1.0), 0.0) * v.abs().amax() + 2.0 ** -25
                out[row:row + new] = o.permute(2, 0, 1, 3).reshape(new, self.q_heads, self.d)
                tol[row:row + new] = t.permute(2, 0, 1, 3).reshape(new, self.q_heads, self.d)
            row += new
        return out, tol


def assert_close(got, want, tol):
    behind = want.isnan()
    off = (got.double() - want).abs()
    bad = ~(off <= tol) & ~behind
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((off / tol.clamp(min=1e-30))[~behind].nan_to_num(float("inf")).max()))
