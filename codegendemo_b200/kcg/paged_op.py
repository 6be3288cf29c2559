"""Attention over a paged cache of keys and values, as a server that generates text runs it in each layer of each step.

``append_kv`` turns a step's queries and keys by their positions and stores keys and values in the pages of their sequences;
``attention_paged`` attends over what the pages hold: one or a few new tokens a sequence (a decode step, drafted tokens), or prompts and
pieces of prompts of any lengths, causal, optionally with a sliding window and first tokens that stay visible. The reference has no
operator of this kind (it lists the attention-shaped chain among its next ones, doc/结果汇总.md).

A cache is a pair of tensors, each (pages, key heads, page size, head dimension), contiguous or any view of that shape; which pages a
sequence has is a row of the page table, how many tokens an entry of ``lengths``::

    cos, sin = rotary_table(max_positions, 128)
    lengths += 1                                                            # the step's token counts
    q = append_kv(k, v, k_cache, v_cache, table, lengths, q=q, rotary=(cos, sin))
    o = attention_paged(q, k_cache, v_cache, table, lengths)                # one new token of each sequence

    q = append_kv(k, v, k_cache, v_cache, table, lengths, starts, q=q, rotary=(cos, sin))
    o = attention_paged(q, k_cache, v_cache, table, lengths, starts)        # rows starts[b] .. starts[b + 1] - 1 are sequence b's

``table`` (sequences x width), ``lengths`` and ``starts`` (sequences + 1) are int32 on the caches' device; they are read when the work runs, so a
captured graph follows what they say at its replay. The rows of a sequence are its last tokens: row i of n has position lengths[b] - n
+ i. Without ``starts`` every sequence has as many rows as every other. A length of 0 is an empty place of the batch.

All work on CUDA tensors of any device, fp16 or bf16, head dimension 64 or 128, on torch's current stream of that device; results come
from torch's allocator. No autograd functions: what they serve is inference. After the first call, calls with right arguments take one step in C++
(3 to 5 us of host time, where the way through Python takes 19 to 31), results into given places among them.
"""
import ctypes
import math

from codegendemo_b200 import _lib
from codegendemo_b200.kcg.Utils import DeviceInfo

_warm = None  # csrc/kcg_torchcall.cpp once something was launched, False where it was not built for this torch


def _launched(status):
    """The end of a call that went this way: its error, or the next call's shorter way."""
    global _warm
    if status:
        _lib.check(status)
    if _warm is None:
        from codegendemo_b200.kcg import matmul_op
        _warm = matmul_op._warm_calls()


def rotary_table(positions, dim, base=10000.0, device="cuda"):
    """(cos, sin) of the angles ``p * base ** (-2 i / dim)`` of positions p = 0 .. positions - 1, each (positions, dim / 2) in fp32; the
    angles are taken in 64 bits (in 32 they are off by 2^-8 of a radian at a position of 100 000)."""
    import torch
    if dim < 2 or dim % 2 or positions < 1:
        raise ValueError("a table of at least one position, of an even number of values")
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angles.cos().float(), angles.sin().float()


def _strides(t, what, dims):
    """Elements between the rows of a tensor's outer dimensions; its innermost one is contiguous and starts on a 16-byte boundary."""
    if t.dim() != dims:
        raise ValueError(f"{what} must have {dims} dimensions, not {t.dim()}")
    sizes, strides = t.shape, t.stride()
    d = sizes[-1]
    if strides[-1] != 1 or t.data_ptr() % 16:
        raise ValueError(f"{what}: heads must be contiguous values on 16-byte boundaries")
    found, inner = [], d
    for n, s in zip(reversed(sizes[:-1]), reversed(strides[:-1])):
        if n <= 1:
            s = inner  # (never taken)
        elif s < d or s % 8:
            raise ValueError(f"{what}: strides must be multiples of 8 values, at least a head's (no broadcast views)")
        found.append(s)
        inner = max(inner, s * max(n, 1))
    return found[::-1]


def _ints(t, what, device, *shape):
    import torch
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != shape or (shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{what} must be int32 {' x '.join(map(str, shape))} on {device}, contiguous")


def _cache(k_cache, v_cache, table, lengths, starts, rows):
    """The C view of a cache after its checks."""
    import torch
    if not k_cache.is_cuda:
        raise ValueError("k_cache must be a CUDA tensor")
    if k_cache.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"k_cache must be float16 or bfloat16, not {k_cache.dtype}")
    ks, vs = _strides(k_cache, "k_cache", 4), _strides(v_cache, "v_cache", 4)
    if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype or v_cache.device != k_cache.device:
        raise ValueError(f"v_cache must be {tuple(k_cache.shape)} {k_cache.dtype} on {k_cache.device}")
    pages, heads, page, d = k_cache.shape
    if d not in (64, 128):
        raise ValueError(f"the head dimension must be 64 or 128, not {d}")
    if page < 8 or page & (page - 1):
        raise ValueError(f"pages hold a power of two of tokens, at least 8, not {page}")
    if pages < 1 or heads < 1:
        raise ValueError("a cache without pages or heads")
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError("page_table must be sequences x pages")
    sequences, width = table.shape
    if sequences > 2 ** 24:
        raise ValueError(f"at most 2^24 sequences, not {sequences}")
    _ints(table, "page_table", k_cache.device, sequences, width)
    ld = table.stride(0) if sequences > 1 else width
    if ld < width:
        raise ValueError("page_table: rows overlap")
    _ints(lengths, "lengths", k_cache.device, sequences)
    if starts is not None:
        _ints(starts, "starts", k_cache.device, sequences + 1)
    elif rows % sequences:
        raise ValueError(f"{rows} rows of {sequences} sequences: without starts every sequence has as many")
    if width * page > 2 ** 31 - 256 or pages > 2 ** 31 - 1:
        raise ValueError("a sequence of more than 2^31 - 256 tokens")
    return _lib.PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), (ctypes.c_int64 * 3)(*ks), (ctypes.c_int64 * 3)(*vs), table.data_ptr(),
                           lengths.data_ptr(), 0 if starts is None else starts.data_ptr(), ld, pages, page, width, sequences, heads, d,
                           62 if k_cache.dtype == torch.bfloat16 else 2)


def _heads(t, what, cache, rows=None, heads=None):
    """(strides as C takes them, rows, heads) of a step's rows."""
    strides = _strides(t, what, 3)
    n, h, d = t.shape
    if d != cache.shape[3] or t.dtype != cache.dtype or t.device != cache.device or (rows is not None and n != rows) or (heads is not None and h != heads):
        raise ValueError(f"{what} must be {'rows' if rows is None else rows} x {'heads' if heads is None else heads} x {cache.shape[3]}, {cache.dtype} on "
                         f"{cache.device}, not {tuple(t.shape)} {t.dtype} on {t.device}")
    return (ctypes.c_int64 * 2)(*strides), n, h


def append_kv(k, v, k_cache, v_cache, page_table, lengths, starts=None, q=None, rotary=None, interleaved=False, positions=None, q_out=None):
    """Stores a step's keys and values, ``k`` and ``v`` (rows, key heads, d), in their sequences' pages; ``lengths`` counts the step's tokens
    already. With ``rotary``, a pair (cos, sin) as ``rotary_table`` makes it, keys are turned by their positions on the way, and so are the
    queries ``q`` (rows, heads, d): returned (in ``q_out``, which may be ``q``, or a new tensor), else None. (cos, sin) of (positions, r / 2)
    values turn the first r of a head's (r a multiple of 16), in pairs r / 2 apart or, ``interleaved``, of neighbours: (x, y) ->
    (x cos - y sin, y cos + x sin), rounded once. ``positions`` (rows, int32): angles of other positions than the cache's. k, v and q may be parts of
    one projection's result. Where two rows have one place in the cache, it holds values of either. A position without angles gives NaN.
    Rows of the queries whose position is negative become zeros, those behind the last sequence's are not written."""
    if _warm:
        turned = _warm.append_kv(k, v, k_cache, v_cache, page_table, lengths, starts, q, rotary, interleaved, positions, q_out)
        if turned is not None:
            return turned if q is not None else None
    import torch
    cache_rows = k.shape[0] if k.dim() == 3 else 0
    c = _cache(k_cache, v_cache, page_table, lengths, starts, cache_rows)
    r = _lib.NewRows()
    r.k_stride, r.rows, _ = _heads(k, "k", k_cache, None, k_cache.shape[1])
    r.v_stride, _, _ = _heads(v, "v", k_cache, r.rows, k_cache.shape[1])
    r.K, r.V = k.data_ptr(), v.data_ptr()
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
    else:
        r.q_stride, _, r.q_heads = _heads(q, "q", k_cache, r.rows)
        if r.q_heads < 1:
            raise ValueError("q has no heads")
        if q_out is None:
            q_out = q.new_empty(q.shape)
        r.qo_stride, _, _ = _heads(q_out, "q_out", k_cache, r.rows, r.q_heads)
        r.Q, r.QO = q.data_ptr(), q_out.data_ptr()
    if rotary is None:
        if positions is not None:
            raise ValueError("positions without rotary")
    else:
        cos, sin = rotary
        if cos.dim() != 2 or cos.shape[0] < 1 or cos.shape[1] % 8 or not 8 <= cos.shape[1] <= k_cache.shape[3] // 2:
            raise ValueError(f"cos must be positions x r / 2, r a multiple of 16 up to {k_cache.shape[3]}")
        for t, what in ((cos, "cos"), (sin, "sin")):
            if t.dtype != torch.float32 or t.device != k_cache.device or t.shape != cos.shape or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{what} must be float32 {tuple(cos.shape)} on {k_cache.device}, contiguous, on a 16-byte boundary")
        r.cos, r.sin, r.angles, r.rotary, r.interleaved = cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1], int(bool(interleaved))
        if positions is not None:
            _ints(positions, "positions", k_cache.device, r.rows)
            r.positions = positions.data_ptr()
    if r.rows > 0:
        dev = k_cache.device.index or 0
        _launched(_lib.get_lib().kcg_append_kv(dev, DeviceInfo.get_cuda_stream(dev), ctypes.byref(c), ctypes.byref(r)))
    return q_out


def attention_paged(q, k_cache, v_cache, page_table, lengths, starts=None, scale=None, window=None, sinks=0, out=None):
    """``softmax(scale * q k^T) v`` of a step's rows over their sequences' keys in the cache: ``q`` (rows, heads, d), the heads a multiple
    of the cache's (up to 64 share a key head), returns (rows, heads, d), in ``out`` if given (which may be ``q``). A row sees its sequence's keys up to its own position; with ``window`` only the
    last that many (itself among them), and the first ``sinks`` of the sequence. ``scale`` is 1 / sqrt(d) if not given. A row without
    any key gives zeros (a negative position: an empty place of the batch); rows behind the last sequence's are not written. Sums and
    softmax in fp32, the weights rounded to the inputs' type in front of their product with the values. Values of keys that no row of the
    sequence sees may be anything; those of keys that some row sees have to be finite. A row that sees a key whose score is NaN, or +inf (by the
    scale, too: products are held in fp32), is NaN."""
    if _warm:
        found = _warm.attention_paged(q, k_cache, v_cache, page_table, lengths, starts, scale, window, sinks, out)
        if found is not None:
            return found
    if q.dim() != 3:
        raise ValueError("q must be rows x heads x d")
    c = _cache(k_cache, v_cache, page_table, lengths, starts, q.shape[0])
    a = _lib.PagedQuery()
    a.q_stride, a.rows, a.q_heads = _heads(q, "q", k_cache)
    if a.q_heads < 1 or a.q_heads % c.kv_heads or a.q_heads // c.kv_heads > 64:
        raise ValueError(f"{a.q_heads} heads of queries over {c.kv_heads} of keys: 1 to 64 share one")
    if out is None:
        out = q.new_empty(q.shape)
    a.o_stride, _, _ = _heads(out, "out", k_cache, a.rows, a.q_heads)
    a.Q, a.O = q.data_ptr(), out.data_ptr()
    if scale is None:
        scale = 1.0 / math.sqrt(c.d)
    if not 0.0 < scale <= 2e38:
        raise ValueError("scale must be positive and finite")
    if window is not None and window < 1:
        raise ValueError("a window sees at least the row's own key")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    a.scale, a.window, a.sinks = scale, min(window or 0, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1)
    if a.rows == 0:
        return out
    dev, lib = k_cache.device.index or 0, _lib.get_lib()
    size = lib.kcg_attention_paged_workspace(dev, ctypes.byref(c), ctypes.byref(a))
    if size < 0:
        _lib.check(size)
    if size > 0:
        import torch
        workspace = q.new_empty(size, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    _launched(lib.kcg_attention_paged(dev, DeviceInfo.get_cuda_stream(dev), ctypes.byref(c), ctypes.byref(a)))
    return out


def attention_paged_status(device: int = 0) -> None:
    """Synchronises the device and raises if a bounded wait of ``attention_paged`` ran out."""
    out = (ctypes.c_uint32 * 4)()
    _lib.check(_lib.get_lib().kcg_attention_paged_status(int(device), out))
