"""Serving operators of flashattn_cuda around attention, as a model's layer calls them.

Three operators that follow one another in a decoder layer:

* ``rope`` / ``rope_backward``: rotary positions of a [B, H, N, D] query or key
  tensor, and the gradient through them.
* ``append_paged``: a ragged batch's new tokens, packed as [T, heads, D], into a
  paged K/V cache, with the queries and keys rotated on the way.
* ``attend_paged``: those tokens' queries against the paged cache: chunks of a
  prompt, single tokens, or both in one batch.

Formulas. Rotation of a pair (a, c) at position p with frequency w, theta = p w:
(a cos - c sin, a sin + c cos) * factor; pair i is dims (i, i + R/2) (halves) or
(2i, 2i + 1) (interleaved) of the first R dims, the others are copied; the
gradient is the rotation by -theta with the same factor. Attention: token t of
sequence b sits at position p = seq_len[b] - n_b + t and sees the keys 0..p of
its sequence; query head h reads K/V head h // (H / H_kv).
"""

import math
import os
import sys

import torch

own = False

# What the drawn cases stay within: the largest listed case of each operator.
MAX_ROPE_ELEMENTS = 8 * 32 * 4096 * 128
MAX_APPEND_TOKENS = 8000
MAX_ATTEND_FLOPS = 4.0 * 32 * 128 * 4 * 2048 * 5120
MAX_CACHE_ELEMENTS = 8 * 8 * 8192 * 128
HEADS = [(12, 12), (14, 14), (8, 8), (14, 2), (32, 8), (28, 4)]
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "flash-attention-cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flashattn_cuda

    return flashattn_cuda


# ---- cases --------------------------------------------------------------------


def _rope(name, op, batch, heads, seq, head_dim, rotary, interleaved, dtype, start, stretch, layout):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "seq": seq,
            "head_dim": head_dim, "rotary": rotary, "interleaved": interleaved, "dtype": dtype,
            "start": start, "stretch": stretch, "layout": layout}


def _paged(name, op, heads, kv_heads, head_dim, dtype, page, batch, context, prompts, chunk,
           pad=0, rotary=0, interleaved=False, stretch=1.0):
    return {"name": name, "op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "page": page, "batch": batch, "context": context, "prompts": prompts,
            "chunk": chunk, "pad": pad, "rotary": rotary, "interleaved": interleaved,
            "stretch": stretch}


def listed():
    return [
        # One token's query heads in a decode step: a launch and a round trip.
        _rope("rope_token", "rope", 1, 12, 1, 64, 64, False, "fp16", 511, 1.0, "heads"),
        # The query heads of a training or prompt batch, straight from the
        # projection's token-major rows (the result is head-major for prefill).
        _rope("rope_batch", "rope", 8, 32, 4096, 128, 128, False, "bf16", 0, 1.0, "tokens"),
        # Gradient of a partly rotated head, adjacent pairs, a length no tile
        # divides, far positions stretched for a long context.
        _rope("rope_backward_ragged", "rope_backward", 2, 14, 1733, 64, 32, True, "fp16", 100000,
              4.0, "heads"),
        # Gradient of a training batch's key heads.
        _rope("rope_backward_batch", "rope_backward", 4, 12, 4096, 64, 64, False, "bf16", 0, 1.0,
              "heads"),
        # A decode step of a serving batch: one token per sequence into its page.
        _paged("append_step", "append", 14, 2, 64, "fp16", 16, 32, 4095, 0, 1, rotary=64),
        # Prompts of several users at once, cut into chunks, into 64-row pages.
        _paged("append_chunks", "append", 32, 8, 128, "bf16", 64, 5, 4096, 5, 2048, pad=7,
               rotary=128, stretch=8.0),
        # One token of a young chat: latency.
        _paged("attend_token_small", "attend", 12, 12, 64, "fp16", 16, 1, 511, 0, 1),
        # One token for each of a serving batch's ragged sequences.
        _paged("attend_token_batch", "attend", 14, 2, 64, "fp16", 16, 32, 4095, 0, 1),
        # One token each over a few long documents.
        _paged("attend_token_long", "attend", 32, 8, 128, "bf16", 64, 8, 8190, 0, 1),
        # A whole prompt as one chunk into an empty cache.
        _paged("attend_prompt", "attend", 14, 14, 64, "fp16", 16, 1, 0, 1, 4096),
        # Continuous batching: three chunks of prompts among sequences that decode.
        _paged("attend_mixed", "attend", 28, 4, 128, "fp16", 32, 24, 4001, 3, 777, pad=5),
        # The largest: long prompts' later chunks over what is cached already.
        _paged("attend_chunks", "attend", 32, 8, 128, "bf16", 64, 4, 6144, 4, 2048),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["rope", "rope_backward", "append", "append", "attend", "attend", "attend",
                     "attend", "attend"])
    dtype = rng.choice(["fp16", "bf16"])
    head_dim = rng.choice([64, 128])
    heads, kv_heads = rng.choice(HEADS)
    rotary = head_dim if rng.random() < 0.6 else 16 * rng.randint(1, head_dim // 16)
    interleaved = rng.random() < 0.4
    stretch = rng.choice([1.0, 1.0, 2.5, 8.0])
    if op in ("rope", "rope_backward"):
        seq = _log_int(rng, 1, 8192)
        limit = MAX_ROPE_ELEMENTS / (heads * seq * head_dim)
        batch = _log_int(rng, 1, max(1.0, min(32.0, limit)))
        return {"op": op, "batch": batch, "heads": heads, "seq": seq, "head_dim": head_dim,
                "rotary": rotary, "interleaved": interleaved, "dtype": dtype,
                "start": rng.choice([0, _log_int(rng, 1, 500000)]), "stretch": stretch,
                "layout": rng.choice(["heads", "tokens"])}
    page = rng.choice([16, 16, 32, 64, 128])
    pad = rng.choice([0, 0, rng.randint(1, 40)])
    kind = rng.choice(["tokens", "few", "chunks", "mixed"])
    if op == "append":
        batch = _log_int(rng, 1, 64)
        prompts = 0 if kind == "tokens" else batch if kind != "mixed" else (batch + 1) // 2
        chunk = _log_int(rng, 2, max(2, MAX_APPEND_TOKENS // max(1, prompts))) if prompts else 1
        limit = MAX_CACHE_ELEMENTS / (batch * kv_heads * head_dim)
        context = _log_int(rng, 1, max(1.0, min(16384.0, limit)))
        rotary = rotary if rng.random() < 0.8 else 0
    else:
        rotary, interleaved, stretch = 0, False, 1.0
        if kind == "tokens":
            batch, prompts, chunk = _log_int(rng, 1, 64), 0, 1
        elif kind == "few":  # a few drafted tokens per sequence, checked at once
            batch = _log_int(rng, 1, 32)
            prompts, chunk = batch, rng.randint(2, 8)
        elif kind == "chunks":
            batch = rng.randint(1, 4)
            prompts, chunk = batch, _log_int(rng, 16, 2048)
        else:
            batch = rng.randint(2, 32)
            prompts, chunk = rng.randint(1, min(4, batch - 1)), _log_int(rng, 16, 1024)
        limit = MAX_CACHE_ELEMENTS / (batch * kv_heads * head_dim)
        context = _log_int(rng, 1, max(1.0, min(16384.0, limit)))
        context = 0 if kind == "chunks" and rng.random() < 0.3 else context
    return {"op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "page": page, "batch": batch, "context": context, "prompts": prompts, "chunk": chunk,
            "pad": pad, "rotary": rotary, "interleaved": interleaved, "stretch": stretch}


def _tokens(case):
    """New tokens of each sequence: the first `prompts` bring chunks of spread
    lengths (the last the whole `chunk`), the others one token each."""
    prompts, chunk = case["prompts"], case["chunk"]
    return [max(1, (i + 1) * chunk // prompts) if i < prompts else 1
            for i in range(case["batch"])]


def _contexts(case):
    """Rows cached before this call, spread evenly over (0, context]."""
    return [(i + 1) * case["context"] // case["batch"] for i in range(case["batch"])]


def work(case):
    size = 2
    if case["op"] in ("rope", "rope_backward"):
        rows = case["batch"] * case["heads"] * case["seq"]
        return {"bytes": 2 * size * rows * case["head_dim"] + 4 * case["batch"] * case["seq"],
                "flops": 3.0 * rows * case["rotary"]}
    new, past = _tokens(case), _contexts(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    table = 4 * sum((p + n + case["page"] - 1) // case["page"] for p, n in zip(past, new))
    lengths = 4 * (2 * case["batch"] + 1)
    if case["op"] == "append":
        moved = 2 * kv_heads + (heads if case["rotary"] else 0)
        return {"bytes": 2 * size * sum(new) * moved * dim + 4 * sum(new) + lengths,
                "flops": 3.0 * sum(new) * (heads + kv_heads) * case["rotary"]}
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
    return {"bytes": 2 * size * sum(new) * heads * dim + table + lengths
            + 2 * size * sum(p + n for p, n in zip(past, new)) * kv_heads * dim,
            "flops": 4.0 * pairs * heads * dim}


# ---- inputs -------------------------------------------------------------------


class State:
    """What a program holds before the call."""


def _inv_freq(rotary, stretch):
    """Frequencies of the pairs, positions pressed together by `stretch`."""
    pair = torch.arange(0, rotary, 2, dtype=torch.float64)
    return (10000.0 ** (-pair / max(rotary, 1)) / stretch).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    s = State()
    s.case = case
    s.inv_freq = _inv_freq(case["rotary"], case["stretch"])
    # Temperature factor that goes with a stretched context.
    s.factor = 1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0
    if case["op"] in ("rope", "rope_backward"):
        batch, heads, seq, dim = case["batch"], case["heads"], case["seq"], case["head_dim"]
        if case["layout"] == "tokens":
            s.x = randn(batch, seq, heads, dim).transpose(1, 2)
        else:
            s.x = randn(batch, heads, seq, dim)
        first = torch.arange(batch, dtype=torch.int32)[:, None] * 3 + case["start"]
        s.positions = (first + torch.arange(seq, dtype=torch.int32)[None]).cuda()
        return s
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    s.new, s.past = _tokens(case), _contexts(case)
    total = sum(s.new) + case["pad"]
    lens = [p + n for p, n in zip(s.past, s.new)]
    used = [(n + page - 1) // page for n in lens]
    pages = sum(used) + 3
    s.k_pages = randn(pages, kv_heads, page, dim)
    s.v_pages = randn(pages, kv_heads, page, dim)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.zeros(case["batch"], max(used) + 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    s.page_table = table.cuda()
    s.seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    bounds = [0]
    for n in s.new:
        bounds.append(bounds[-1] + n)
    s.cu_tokens = torch.tensor(bounds, dtype=torch.int32).cuda()
    # Queries, keys and values as one projection leaves them.
    qkv = randn(total, heads + 2 * kv_heads, dim)
    s.q, s.k, s.v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    s.scale = 1.0 / math.sqrt(dim)
    return s


# ---- plain forms --------------------------------------------------------------


def _rotated(x, cos, sin, rotary, interleaved):
    """x [..., D] rotated by angles whose cos / sin are [..., R / 2]."""
    rot, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, c = rot[..., 0::2], rot[..., 1::2]
    else:
        a, c = rot[..., :rotary // 2], rot[..., rotary // 2:]
    first, second = a * cos - c * sin, a * sin + c * cos
    if interleaved:
        turned = torch.stack((first, second), dim=-1).flatten(-2)
    else:
        turned = torch.cat((first, second), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_rope(s, sign):
    # Angles of far positions need 64 bits; their sines do not.
    angle = s.positions.double()[..., None] * s.inv_freq * sign
    cos = (angle.cos() * s.factor).float()[:, None]
    sin = (angle.sin() * s.factor).float()[:, None]
    out = _rotated(s.x.float(), cos, sin, s.case["rotary"], s.case["interleaved"])
    return out.to(s.x.dtype)


def _plain_append(s):
    total, bounds = sum(s.new), s.cu_tokens
    token = torch.arange(total, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(bounds[1:], token, right=True)
    pos = s.seq_lens[b] - bounds[b + 1] + token
    page = s.page_table[b, (pos // s.case["page"]).long()].long()
    row = (pos % s.case["page"]).long()
    q, k, v = s.q[:total], s.k[:total], s.v[:total]
    out = None
    if s.case["rotary"]:
        angle = pos.double()[:, None] * s.inv_freq
        cos, sin = ((angle.cos() * s.factor).float()[:, None],
                    (angle.sin() * s.factor).float()[:, None])
        k = _rotated(k.float(), cos, sin, s.case["rotary"], s.case["interleaved"]).to(k.dtype)
        out = torch.zeros(s.q.shape, dtype=q.dtype, device="cuda")
        out[:total] = _rotated(q.float(), cos, sin, s.case["rotary"], s.case["interleaved"])
    s.k_pages[page, :, row] = k
    s.v_pages[page, :, row] = v
    return [s.k_pages, s.v_pages] + ([out] if out is not None else [])


def _softmax_products(q, k, v, scale, hidden):
    """softmax(scale q k^T, without the hidden pairs) v of contiguous operands."""
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    scores.masked_fill_(hidden, float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    return torch.matmul(weights, v) / weights.sum(-1, keepdim=True)


def _gathered(pages, table, kv_heads, dim):
    """Rows of the tables' pages, [..., H_kv, rows, D] in 32 bits."""
    return pages[table.long()].transpose(-4, -3).flatten(-3, -2).float().contiguous()


def _plain_attend(s):
    case = s.case
    heads, kv_heads, dim, batch = case["heads"], case["kv_heads"], case["head_dim"], case["batch"]
    group = heads // kv_heads
    out = torch.zeros(s.q.shape, dtype=s.q.dtype, device="cuda")
    if case["prompts"] == 0:  # one token each: one padded batch
        k = _gathered(s.k_pages, s.page_table, kv_heads, dim)
        v = _gathered(s.v_pages, s.page_table, kv_heads, dim)
        q = s.q[:batch].float().reshape(batch, kv_heads, group, dim)
        hidden = torch.arange(k.shape[2], device="cuda") >= s.seq_lens[:, None, None, None]
        out[:batch] = _softmax_products(q, k, v, s.scale, hidden).reshape(batch, heads, dim)
        return out
    at = 0
    for b, (n, past) in enumerate(zip(s.new, s.past)):
        used = (past + n + case["page"] - 1) // case["page"]
        k = _gathered(s.k_pages, s.page_table[b, :used], kv_heads, dim)[:, :past + n].contiguous()
        v = _gathered(s.v_pages, s.page_table[b, :used], kv_heads, dim)[:, :past + n].contiguous()
        q = s.q[at:at + n].float().reshape(n, kv_heads, group, dim).permute(1, 2, 0, 3)
        q = q.reshape(kv_heads, group * n, dim)
        hidden = (torch.arange(past + n, device="cuda")
                  > torch.arange(past, past + n, device="cuda")[:, None]).repeat(group, 1)
        o = _softmax_products(q, k, v, s.scale, hidden).reshape(kv_heads, group, n, dim)
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, heads, dim)
        at += n
    return out


def run(s):
    op = s.case["op"]
    if not own:
        if op == "attend":
            return _plain_attend(s)
        if op == "append":
            return _plain_append(s)
        return _plain_rope(s, 1.0 if op == "rope" else -1.0)
    fa = _package()
    if op == "attend":
        return fa.attend_paged(s.q, s.k_pages, s.v_pages, s.page_table, s.seq_lens, s.cu_tokens,
                               s.scale)
    if op == "append":
        if not s.case["rotary"]:
            fa.append_paged(s.k_pages, s.v_pages, s.k, s.v, s.page_table, s.seq_lens, s.cu_tokens)
            return [s.k_pages, s.v_pages]
        out = fa.append_paged(s.k_pages, s.v_pages, s.k, s.v, s.page_table, s.seq_lens,
                              s.cu_tokens, s.q, s.inv_freq, s.case["interleaved"], s.factor)
        return [s.k_pages, s.v_pages, out]
    call = fa.rope if op == "rope" else fa.rope_backward
    return call(s.x, s.positions, s.inv_freq, s.case["interleaved"], s.factor)


# ---- definitions in 64 bits ---------------------------------------------------


def _turn64(x, positions, s):
    """Row-by-row rotation in 64 bits as a complex product; x [..., R or more]."""
    r = s.case["rotary"]
    theta = positions.double()[..., None] * s.inv_freq
    phase = torch.polar(torch.full_like(theta, s.factor), theta)
    x = x.double()
    out = x.clone()
    if s.case["interleaved"]:
        z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * phase
        out[..., 0:r:2], out[..., 1:r:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * phase
        out[..., :r // 2], out[..., r // 2:r] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rope", "rope_backward"):
        positions = s.positions if case["op"] == "rope" else -s.positions
        return _turn64(s.x, positions[:, None], s)
    table = s.page_table.cpu()
    page, heads, kv_heads = case["page"], case["heads"], case["kv_heads"]
    if case["op"] == "append":
        k_pages, v_pages = s.k_pages.double(), s.v_pages.double()
        out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
        at = 0
        for b, (n, past) in enumerate(zip(s.new, s.past)):
            pos = torch.arange(past, past + n)
            where = table[b][pos // page].long().cuda(), slice(None), (pos % page).cuda()
            rows = slice(at, at + n)
            k = s.k[rows].double()
            if case["rotary"]:
                k = _turn64(s.k[rows], pos.cuda()[:, None], s)
                out[rows] = _turn64(s.q[rows], pos.cuda()[:, None], s)
            k_pages[where] = k
            v_pages[where] = s.v[rows].double()
            at += n
        return [k_pages, v_pages] + ([out] if case["rotary"] else [])
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, past) in enumerate(zip(s.new, s.past)):
        used = (past + n + page - 1) // page
        ids = table[b, :used].long().cuda()
        for h in range(kv_heads):
            k = s.k_pages[ids, h].reshape(used * page, -1)[:past + n].double()
            v = s.v_pages[ids, h].reshape(used * page, -1)[:past + n].double()
            for head in range(h * (heads // kv_heads), (h + 1) * (heads // kv_heads)):
                logits = s.q[at:at + n, head].double() @ k.t().contiguous() * s.scale
                logits = logits + torch.full_like(logits, float("-inf")).triu(past + 1)
                out[at:at + n, head] = torch.softmax(logits, -1) @ v
        at += n
    return out
