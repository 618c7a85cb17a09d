"""Plain 64-bit forms of rope, append_paged and attend_paged, on the CPU, with the
error bounds their kernels have to meet, and the structures of their C entry points."""

import ctypes

import torch

class Paged(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p)
                 for n in ("k_pages", "v_pages", "page_table", "seq_lens", "cu_tokens")]
                + [(n, ctypes.c_int)
                   for n in ("dtype", "batch", "tokens", "kv_heads", "head_dim", "page_size",
                             "num_pages", "max_pages")])


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64)]


def half_step(dtype):
    """Largest relative rounding error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def turn(x, positions, inv_freq, interleaved, factor=1.0):
    """x [..., D] in 64 bits turned at `positions` (shape of x without D, or one
    that broadcasts to it); also sum |a| + |c| per element, the size its fp32
    products have."""
    x = x.double()
    r = 2 * inv_freq.numel()
    theta = positions.double()[..., None] * inv_freq.double()
    cos, sin = theta.cos() * factor, theta.sin() * factor
    out, size = x.clone(), x.abs()
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, c = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - c * sin, a * sin + c * cos
    size[..., first] = size[..., second] = (a.abs() + c.abs()) * abs(factor)
    return out, size


def turn_bound(out, size, dtype):
    """One rounding of the result; in fp32 the angle (2^-24 of up to half a turn,
    pi in radians), sine and cosine (2 ulp), factor and products: under
    8 * 2^-24 + pi * 2^-24 of |a| + |c|. Results under the type's least normal
    number round by half its least step."""
    return half_step(dtype) * out.abs() + 12 * 2.0 ** -24 * size + torch.finfo(dtype).tiny * 2.0 ** -8


def attend(q, k_pages, v_pages, page_table, seq_lens, cu_tokens, scale, wide=None):
    """(out, bound) in 64 bits for CPU tensors. Keys of page ids outside the pool
    and of positions outside the page table do not exist."""
    tokens, heads, dim = q.shape
    pages, kv_heads, size, _ = k_pages.shape
    group = heads // kv_heads
    dtype = q.dtype
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    u = half_step(dtype)
    for b in range(len(seq_lens)):
        lo, hi = int(cu_tokens[b]), int(cu_tokens[b + 1])
        length = int(seq_lens[b])
        keys = torch.arange(max(0, min(length, page_table.shape[1] * size)))
        ids = page_table[b].long()[keys // size]
        there = (ids >= 0) & (ids < pages)
        keys, ids = keys[there], ids[there]
        k = k_pages[ids, :, keys % size].double()  # [L, H_kv, D]
        v = v_pages[ids, :, keys % size].double()
        for t in range(lo, min(hi, tokens)):
            seen = keys <= length - hi + t
            n = int(seen.sum())
            if n == 0:
                continue
            ks = k[seen].repeat_interleave(group, 1)
            vs = v[seen].repeat_interleave(group, 1)
            qt = q[t].double()
            logits = torch.einsum("hd,lhd->hl", qt, ks) * scale
            p = torch.softmax(logits, -1)
            o = torch.einsum("hl,lhd->hd", p, vs)
            spread = torch.einsum("hl,lhd->hd", p, vs.abs())
            # Logits in fp32: D products and sums, the scale, the exponent's
            # product and bound, exp2: (D + 8) half steps of sum |q| |k| |scale|.
            mass = torch.einsum("hd,lhd->hl", qt.abs(), ks.abs()).amax(-1) * abs(scale)
            logit = (dim + 8) * 2.0 ** -24 * (mass + 8)
            # Weights rounded to the type once (numerator and sum), sums in fp32.
            weights = 2 * u + 2 * n * 2.0 ** -24 / max(1.0, n ** 0.5)
            # Weights under the type's least normal number (at a bound that is at
            # most the row's maximum: the weights' sum is at least 1).
            tiny = n * torch.finfo(dtype).tiny * 2.0 ** -10 * vs.abs().amax(0)
            out[t] = o
            bound[t] = (spread * (weights + 2 * logit[:, None]) + tiny + u * o.abs()
                        + torch.finfo(dtype).tiny * 2.0 ** -8)
    return out, bound


def batch(sequences, kv_heads, heads, dim, page, dtype, seed, pad=0, extra_columns=1, spare=2):
    """A paged batch on the CPU: `sequences` is a list of (cached, new) counts."""
    gen = torch.Generator().manual_seed(seed)
    lens = [p + n for p, n in sequences]
    used = [(n + page - 1) // page for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.zeros(len(lens), max(used) + extra_columns, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    bounds = [0]
    for _, n in sequences:
        bounds.append(bounds[-1] + n)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float32).to(dtype)

    total = bounds[-1] + pad
    return {"q": randn(total, heads, dim), "k": randn(total, kv_heads, dim),
            "v": randn(total, kv_heads, dim), "k_pages": randn(pages, kv_heads, page, dim),
            "v_pages": randn(pages, kv_heads, page, dim), "page_table": table,
            "seq_lens": torch.tensor(lens, dtype=torch.int32),
            "cu_tokens": torch.tensor(bounds, dtype=torch.int32)}
