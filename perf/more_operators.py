"""The calls that a server's attention over a paged cache is measured on: rotating a step's queries and keys by their positions and
storing keys and values into the pages of their sequences, the attention of one or a few new tokens over such a cache, and that of
whole prompts (or pieces of them), each with an optional sliding window and first tokens that stay visible.

Every case goes through the entry points of ``codegendemo_b200.kcg.matmul_op`` on GPU tensors: the step's rows, the caches, the page
table, lengths and row ranges in hand, results allocated by the call.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BASE = 10000.0  # of the rotation's angles
MAX_TOKENS = 16384


def listed():
    return [
        # a decode step of 32 sequences: one token's rows each, latency is all of it
        {"name": "append_decode_bf16", "op": "append", "batch": 32, "tokens": 1, "length": 4096, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 16, "dtype": "bf16", "interleaved": False, "rotary": 128, "fused_qkv": True, "seed": 1},
        # a packed batch of four prompts behind the projection of all three
        {"name": "append_prompt_bf16", "op": "append", "batch": 4, "tokens": 4096, "length": 4096, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 64, "dtype": "bf16", "interleaved": False, "rotary": 128, "fused_qkv": True, "seed": 2},
        # pieces of prompts of no even length, half of each head rotated, neighbouring values in pairs
        {"name": "append_ragged_fp16", "op": "append", "batch": 7, "tokens": 611, "length": 2500, "q_heads": 14, "kv_heads": 2, "d": 64,
         "page": 32, "dtype": "fp16", "interleaved": True, "rotary": 32, "fused_qkv": False, "seed": 3},
        # one user's next token over a chat: nothing but the split of its keys fills the GPU
        {"name": "decode_one_bf16", "op": "decode", "batch": 1, "tokens": 1, "length": 4097, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 16, "dtype": "bf16", "window": 0, "sinks": 0, "seed": 4},
        # a server's step: 64 sequences of all lengths, some places of the batch empty
        {"name": "decode_batch_bf16", "op": "decode", "batch": 64, "tokens": 1, "length": 16384, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 64, "dtype": "bf16", "window": 0, "sinks": 0, "seed": 5},
        # as many key heads as query heads, short heads
        {"name": "decode_heads_fp16", "op": "decode", "batch": 16, "tokens": 1, "length": 2049, "q_heads": 32, "kv_heads": 32, "d": 64,
         "page": 32, "dtype": "fp16", "window": 0, "sinks": 0, "seed": 6},
        # long streams that keep four first tokens and the last 1024; four drafted tokens checked at once
        {"name": "decode_window_bf16", "op": "decode", "batch": 48, "tokens": 4, "length": 8192, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 16, "dtype": "bf16", "window": 1024, "sinks": 4, "seed": 7},
        # one long prompt
        {"name": "prompt_bf16", "op": "prompt", "batch": 1, "tokens": 8192, "length": 8192, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 64, "dtype": "bf16", "window": 0, "sinks": 0, "seed": 8},
        # one longer prompt of a model whose layers look back 1024 tokens, and at the first four
        {"name": "prompt_window_bf16", "op": "prompt", "batch": 1, "tokens": 16384, "length": 16384, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 16, "dtype": "bf16", "window": 1024, "sinks": 4, "seed": 9},
        # a batch of prompts of no even length, seven query heads to a key head
        {"name": "prompt_ragged_fp16", "op": "prompt", "batch": 6, "tokens": 1501, "length": 1501, "q_heads": 14, "kv_heads": 2, "d": 64,
         "page": 32, "dtype": "fp16", "window": 0, "sinks": 0, "seed": 10},
        # the next piece of a long prompt, over what the cache holds of it
        {"name": "prompt_piece_bf16", "op": "prompt", "batch": 1, "tokens": 512, "length": 16384, "q_heads": 32, "kv_heads": 8, "d": 128,
         "page": 64, "dtype": "bf16", "window": 0, "sinks": 0, "seed": 11},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    while True:
        kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
        group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        d = rng.choice([64, 128, 128])
        c = {"op": op, "batch": 1, "tokens": 1, "length": 1, "q_heads": kv * group, "kv_heads": kv, "d": d, "page": rng.choice([16, 16, 32, 64, 128]),
             "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        if op == "append":
            c["batch"], c["length"] = _log(rng, 1, 256), _log(rng, 1 if rng.random() < 0.1 else 64, MAX_TOKENS)
            c["tokens"] = 1 if rng.random() < 0.4 else _log(rng, 1, c["length"])
            c["interleaved"], c["rotary"] = rng.random() < 0.3, rng.choice([d, d, d // 2, d // 4])
            c["fused_qkv"] = rng.random() < 0.6
            fits = c["batch"] * c["tokens"] * (c["q_heads"] + 2 * kv) * d <= 16384 * 48 * 128 and c["batch"] * c["length"] * kv * d <= 16384 * 8 * 128 * 4
        else:
            if op == "decode":
                c["batch"], c["length"] = _log(rng, 1, 128), _log(rng, 1 if rng.random() < 0.1 else 128, 2 * MAX_TOKENS)
                c["tokens"] = min(c["length"], rng.choice([1, 1, 1, 1, 2, 3, 5]))
                fits = c["batch"] * c["length"] * kv * d <= 64 * 16384 * 8 * 128 and c["batch"] * c["length"] * kv * group * c["tokens"] <= 64 * 16384 * 32 * 4
            else:
                c["batch"], c["length"] = _log(rng, 1, 12), _log(rng, 16 if rng.random() < 0.1 else 256, MAX_TOKENS)
                c["tokens"] = c["length"] if rng.random() < 0.6 else _log(rng, min(16, c["length"]), c["length"])
                fits = (c["batch"] * kv * group * c["tokens"] * c["length"] * d <= 32 * 16384 * 16384 * 128 // 3 and
                        c["batch"] * c["tokens"] * kv * group * d <= MAX_TOKENS * 32 * 128)
            c["window"], c["sinks"] = (_log(rng, 16, 4096), rng.choice([0, 1, 4, 64])) if rng.random() < 0.4 else (0, 0)
        if kv * group <= 64 and fits:
            c["seed"] = rng.randrange(1 << 20)
            return c


def _sequences(case):
    """(new tokens, length with them) of each sequence: the case's largest first, the others shorter; now and then none (an empty place)."""
    rng = random.Random(case["seed"])

    def shorter():
        n, length = case["tokens"], _log(rng, max(1, case["length"] // 8), case["length"])
        if case["op"] == "decode":
            return n, 0 if rng.random() < 0.05 else length
        if n == 1:
            return n, length
        return length if n == case["length"] else min(length, _log(rng, max(1, n // 4), n)), length
    return [(case["tokens"], case["length"])] + [shorter() for _ in range(case["batch"] - 1)]


def _uniform(case):
    """Whether every sequence has the same number of new tokens: the calls that need no row ranges."""
    return case["op"] == "decode" or case["tokens"] == 1


def _angles(rows, dim, device):
    """cos and sin of the rotation's angles of each position, taken in 64 bits."""
    inv = BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    a = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, hq, hkv, page = DTYPES[case["dtype"]], case["d"], case["q_heads"], case["kv_heads"], case["page"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    found = _sequences(case)
    new, lengths = [n for n, _ in found], [l for _, l in found]
    used = [-(-l // page) for l in lengths]
    width = max(used) + 1  # (the next page's place)
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.zeros((case["batch"], width), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):  # pages of a sequence lie anywhere
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, hkv, page, d)
    state = {"case": case, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "starts": None,
             "k_cache": torch.randn(shape, generator=g, device="cuda", dtype=dt), "v_cache": torch.randn(shape, generator=g, device="cuda", dtype=dt)}
    rows = sum(new)
    if not _uniform(case):
        state["starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        if case["fused_qkv"]:  # parts of one projection's rows
            qkv = normal(rows, hq + 2 * hkv, d).to(dt)
            state["q"], state["k"], state["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            state["q"], state["k"], state["v"] = normal(rows, hq, d).to(dt), normal(rows, hkv, d).to(dt), normal(rows, hkv, d).to(dt)
        state["cos"], state["sin"] = _angles(max(lengths) + 8, case["rotary"], "cuda")
    else:
        # heads from almost even weights to weights on few keys
        state["q"] = (normal(rows, hq, d) * torch.exp(0.5 * normal(hq, 1) + 0.4)).to(dt)
    return state


def _rows(case, state):
    """Of each row its sequence, its place among the sequence's new tokens, and its position."""
    n = state["q"].shape[0]
    if state["starts"] is None:
        r = torch.arange(n, device="cuda")
        b, i, new = r // case["tokens"], r % case["tokens"], case["tokens"]
    else:
        counts = (state["starts"][1:] - state["starts"][:-1]).long()
        b = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), counts, output_size=n)
        i, new = torch.arange(n, device="cuda") - state["starts"].long()[b], counts[b]
    return b, i, state["lengths"].long()[b] - new + i


def _rotated(x, cos, sin, interleaved):
    """x (rows, heads, d) with its first values turned by the angles of its rows."""
    x = x.float()
    half = cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from codegendemo_b200.kcg import matmul_op
        if op == "append":
            q = matmul_op.append_kv(state["k"], state["v"], state["k_cache"], state["v_cache"], state["table"], state["lengths"],
                                    starts=state["starts"], q=state["q"], rotary=(state["cos"], state["sin"]), interleaved=case["interleaved"])
            return q, state["k_cache"], state["v_cache"]
        return matmul_op.attention_paged(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lengths"],
                                         starts=state["starts"], window=case["window"] or None, sinks=case["sinks"])
    dt, page, batch, d = state["q"].dtype, case["page"], case["batch"], case["d"]
    b, i, pos = _rows(case, state)
    if op == "append":
        cos, sin = state["cos"][pos], state["sin"][pos]
        at = state["table"].long()[b, pos // page]
        state["k_cache"][at, :, pos % page] = _rotated(state["k"], cos, sin, case["interleaved"]).to(dt)
        state["v_cache"][at, :, pos % page] = state["v"]
        return _rotated(state["q"], cos, sin, case["interleaved"]).to(dt), state["k_cache"], state["v_cache"]
    hq, hkv, new, longest = case["q_heads"], case["kv_heads"], case["tokens"], case["length"]
    group = hq // hkv
    # every sequence filled up to the longest: rows (batch, kv heads, tokens x group, d), keys (batch, kv heads, length, d)
    q = torch.zeros((batch, new, hq, d), device="cuda")
    q[b, i] = state["q"].float()
    q = q.view(batch, new, hkv, group, d).transpose(1, 2).reshape(batch, hkv, new * group, d)
    at = state["table"][:, :-(-longest // page)].long()

    def keys(cache):
        return cache[at].transpose(1, 2).reshape(batch, hkv, -1, d)[:, :, :longest].float()
    scores = q @ keys(state["k_cache"]).transpose(2, 3)
    position = torch.full((batch, new), -1, device="cuda")
    position[b, i] = pos
    key = torch.arange(longest, device="cuda")
    hidden = key > position[:, :, None]
    if case["window"]:
        hidden |= (key <= position[:, :, None] - case["window"]) & (key >= case["sinks"])
    scores = scores.mul_(1.0 / math.sqrt(d)).view(batch, hkv, new, group, longest)
    scores.masked_fill_(hidden[:, None, :, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weights = scores.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = weights.sum(dim=-1, keepdim=True)
    out = (weights.view(batch, hkv, new * group, longest) @ keys(state["v_cache"])).view(batch, hkv, new, group, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.transpose(1, 2).reshape(batch, new, hq, d)[b, i].to(dt)


def _visible(case):
    """Over all sequences: pairs of a new token and a key that it sees, and keys that some new token sees."""
    window, sinks = case["window"], case["sinks"]

    def up_to(n, most):
        """min(1, most) + ... + min(n, most)"""
        return n * (n + 1) // 2 if n <= most else most * (most + 1) // 2 + (n - most) * most

    def of(n, length):
        first = max(length - n, 0)
        if not window:
            return (up_to(length, length) - up_to(first, length), length) if length else (0, 0)
        near, back = min(length, length - first + window - 1), [max(0, p - window) for p in (length, first)]
        return up_to(length, window) - up_to(first, window) + up_to(back[0], sinks) - up_to(back[1], sinks), near + min(sinks, length - near)
    return [sum(both) for both in zip(*(of(*found) for found in _sequences(case)))]


def work(case):
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["d"]
    found = _sequences(case)
    rows = sum(n for n, _ in found)
    if case["op"] == "append":
        values = rows * (hq + 2 * hkv) * d
        return {"bytes": 2 * 2 * values + 4 * rows * case["rotary"], "flops": 3.0 * rows * (hq + hkv) * case["rotary"]}
    pairs, seen = _visible(case)
    pages = sum(-(-l // case["page"]) for _, l in found)
    return {"bytes": 2 * (2 * rows * hq * d + 2 * seen * hkv * d) + 4 * (pages if not case["window"] else 0), "flops": 4.0 * pairs * hq * d}


def exact(case, seed):
    """In 64 bits, sequence by sequence."""
    s = prepare(case, seed)
    d, page, hq, hkv = case["d"], case["page"], case["q_heads"], case["kv_heads"]
    group = hq // hkv
    table = s["table"].tolist()
    found = _sequences(case)
    if case["op"] == "append":
        out = s["q"].double()
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        half = case["rotary"] // 2
        pair = torch.arange(half, device="cuda")
        low, high = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + half)

        def turned(x, first):
            y = x.double()
            angle = torch.complex(s["cos"][first:first + x.shape[0]].double(), s["sin"][first:first + x.shape[0]].double())[:, None]
            z = torch.complex(y[..., low], y[..., high]) * angle
            y[..., low], y[..., high] = z.real, z.imag
            return y
        row = 0
        for b, (n, length) in enumerate(found):
            rows, first = slice(row, row + n), length - n
            out[rows] = turned(s["q"][rows], first)
            where = [(table[b][p // page], p % page) for p in range(first, length)]
            to, slot = (torch.tensor(w, device="cuda") for w in zip(*where))
            k_cache[to, :, slot] = turned(s["k"][rows], first)
            v_cache[to, :, slot] = s["v"][rows].double()
            row += n
        return out, k_cache, v_cache
    if 4.0 * _visible(dict(case, window=0))[0] * hq * d > 2e13:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, length) in enumerate(found):
        if length > 0:
            mine = torch.tensor(table[b][:-(-length // page)], device="cuda")
            for h in range(hkv):
                k, v = (c[mine, h].reshape(-1, d)[:length].double() for c in (s["k_cache"], s["v_cache"]))
                for r0 in range(0, n, 1024):
                    r1 = min(n, r0 + 1024)
                    p = torch.arange(length - n + r0, length - n + r1, device="cuda")[:, None]
                    j = torch.arange(length, device="cuda")[None]
                    sees = j <= p
                    if case["window"]:
                        sees = sees & ((p - j < case["window"]) | (j < case["sinks"]))
                    q = s["q"][row + r0:row + r1, h * group:(h + 1) * group].double()
                    logits = torch.einsum("rgd,jd->grj", q, k) / math.sqrt(d)
                    logits[:, ~sees] = -math.inf
                    weights = torch.softmax(logits, dim=-1).nan_to_num(0.0)  # (a row before the sequence's first token sees nothing)
                    out[row + r0:row + r1, h * group:(h + 1) * group] = torch.einsum("grj,jd->rgd", weights, v)
        row += n
    return out
