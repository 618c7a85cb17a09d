"""append_paged and attend_paged over random batches: head counts, page sizes, ragged and
empty sequences, rows outside them, absent pages, wide tables, strided inputs."""

import random

import pytest
import torch

import flashattn_cuda
import paged_reference as ref

pytestmark = pytest.mark.gpu
CACHE = ("k_pages", "v_pages", "page_table", "seq_lens", "cu_tokens")


def _draw(seed):
    rng = random.Random(seed)
    dtype = rng.choice([torch.float16, torch.bfloat16])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 1, 2, 3, 5])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 11, 16, 17, 31, 33])
    page = rng.choice([16, 32, 64, 128, 256])
    sequences = []
    for _ in range(rng.choice([1, 2, 3, 5, 9, 70, 140])):
        cached = int(10 ** rng.uniform(0, 3.2)) - 1
        new = rng.choice([0, 1, 1, 1, 2, 3, rng.randint(4, 40), rng.randint(1, 170)])
        sequences.append((cached, new))
    if len(sequences) > 9:
        sequences = [(p % 300, min(n, rng.choice([0, 1, 6]))) for p, n in sequences]
    front, back = (rng.choice([0, 0, rng.randint(1, 30)]) for _ in range(2))
    s = ref.batch(sequences, kv_heads, heads, dim, page, dtype, seed, pad=front + back,
                  extra_columns=rng.choice([0, 1, 40, 2 ** 26 // page]) or 1)
    s["cu_tokens"] += front
    if rng.random() < 0.3:  # absent pages
        for _ in range(rng.randint(1, 4)):
            b = rng.randrange(len(sequences))
            s["page_table"][b, rng.randrange(min(s["page_table"].shape[1], 12))] = rng.choice(
                [-1, s["k_pages"].shape[0], 2 ** 31 - 1, -2 ** 31])
    if rng.random() < 0.3:  # lengths under their new tokens
        for _ in range(2):
            b = rng.randrange(len(sequences))
            s["seq_lens"][b] = rng.choice([0, -7, int(s["seq_lens"][b]) // 2])
    rotary = rng.choice([0, dim, 16, dim // 2])
    return s, rotary, rng.random() < 0.5, rng.choice([dim ** -0.5, 0.3, -0.2])


def _strided(x, seed):
    """`x` with the strides of a slice of a projection, or with heads first in memory."""
    if seed % 3 == 0:
        return x.cuda()
    if seed % 3 == 1:
        wide = torch.zeros(x.shape[0], x.shape[1] + 3, x.shape[2], dtype=x.dtype, device="cuda")
        wide[:, 2:-1] = x.cuda()
        return wide[:, 2:-1]
    return x.cuda().transpose(0, 1).contiguous().transpose(0, 1)


@pytest.mark.parametrize("seed", range(60))
def test_random_batches(seed):
    s, rotary, interleaved, scale = _draw(seed)
    cache = {n: s[n].cuda() for n in CACHE}
    q, k, v = (_strided(s[n], seed) for n in ("q", "k", "v"))
    args = {}
    if rotary:
        inv_freq = flashattn_cuda.rope_frequencies(rotary)[0]
        args = {"q": q, "inv_freq": inv_freq.cuda(), "interleaved": interleaved}
    out = flashattn_cuda.append_paged(cache["k_pages"], cache["v_pages"], k, v,
                                      *(cache[n] for n in CACHE[2:]), **args)
    # The pages and q_out by the definition.
    page, pages = s["k_pages"].shape[2], s["k_pages"].shape[0]
    want_k, want_v = s["k_pages"].clone(), s["v_pages"].clone()
    new_k, new_q = k.cpu(), q.cpu()
    bounds, where = s["cu_tokens"].tolist(), []
    outside = torch.ones(new_k.shape[0], dtype=torch.bool)
    positions = torch.zeros(new_k.shape[0], dtype=torch.long)
    for b, n in enumerate(s["seq_lens"].tolist()):
        for t in range(bounds[b], bounds[b + 1]):
            pos = n - bounds[b + 1] + t
            outside[t], positions[t] = False, pos
            if 0 <= pos < s["page_table"].shape[1] * page:
                at = int(s["page_table"][b, pos // page])
                if 0 <= at < pages:
                    where.append((t, at, pos % page))
                    want_v[at, :, pos % page] = s["v"][t]
    got_k, got_v = cache["k_pages"].cpu(), cache["v_pages"].cpu()
    assert torch.equal(got_v, want_v)
    turned, bound = new_k.double(), torch.zeros(new_k.shape, dtype=torch.float64)
    if rotary:
        turned, size = ref.turn(new_k, positions[:, None], inv_freq, interleaved)
        bound = ref.turn_bound(turned, size, new_k.dtype)
        turned_q, size = ref.turn(new_q, positions[:, None], inv_freq, interleaved)
        assert (out[outside.cuda()] == 0).all()
        assert ((out.cpu().double() - turned_q).abs()
                <= ref.turn_bound(turned_q, size, new_q.dtype))[~outside].all()
        q = out
    for t, at, row in where:
        assert ((got_k[at, :, row].double() - turned[t]).abs() <= bound[t]).all()
        want_k[at, :, row] = got_k[at, :, row]
    assert torch.equal(got_k, want_k)

    got = flashattn_cuda.attend_paged(q, *(cache[n] for n in CACHE), scale)
    want, bound = ref.attend(q.cpu(), got_k, got_v, *(s[n] for n in CACHE[2:]), scale)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert (got[outside.cuda()] == 0).all()
    assert torch.equal(flashattn_cuda.attend_paged(q, *(cache[n] for n in CACHE), scale), got)


@pytest.mark.parametrize("sequences", [
    [(5000, 1), (40, 1)], [(3001, 40), (10, 1), (4100, 1)], [(0, 600)], [(9000, 3)] * 3,
    [(100, 1)] * 300, [(20000, 1)]])
@pytest.mark.parametrize("columns", [2 ** 17 - 400, 2 ** 14])
def test_tables_much_wider_than_the_lengths(sequences, columns):
    """The weights' unit is chosen for the table's width: up to 2^27 keys for each sequence, a
    share's border then counts thousands of keys."""
    s = ref.batch(sequences, 2, 6, 64, 1024, torch.float16, 90, extra_columns=columns)
    got = flashattn_cuda.attend_paged(s["q"].cuda(), *(s[n].cuda() for n in CACHE), 0.125)
    want, bound = ref.attend(s["q"], *(s[n] for n in CACHE), 0.125)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    # Borders elsewhere, partials joined in another order: the same within the sums' rounding.
    narrow = s["page_table"][:, :-columns + 1].contiguous()
    assert (got - flashattn_cuda.attend_paged(
        s["q"].cuda(), s["k_pages"].cuda(), s["v_pages"].cuda(), narrow.cuda(),
        s["seq_lens"].cuda(), s["cu_tokens"].cuda(), 0.125)).abs().max() <= 2 * bound.max()
