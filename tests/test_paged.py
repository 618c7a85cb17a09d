"""The paged cache: ``append_paged`` and ``attend_paged`` against plain forms in
64 bits, at the sizes, lengths and contents where they can go wrong."""

import ctypes
import os
import threading

import pytest
import torch

import flashattn_cuda
import paged_reference as ref
from paged_reference import Paged, Rows

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
CACHE = ("k_pages", "v_pages", "page_table", "seq_lens", "cu_tokens")


def _attend(s, scale, q=None):
    return flashattn_cuda.attend_paged((s["q"] if q is None else q).cuda(),
                                       *(s[name].cuda() for name in CACHE), scale)


def _check(s, scale=0.125):
    got = _attend(s, scale).cpu()
    want, bound = ref.attend(s["q"], *(s[name] for name in CACHE), scale)
    error = (got.double() - want).abs()
    assert got.dtype == s["q"].dtype and got.shape == s["q"].shape
    assert torch.isfinite(got).all()
    assert (error <= bound).all(), f"{(error - bound).max()} over the bound"
    return got


SEQUENCES = {
    "one_token_first": [(0, 1)],
    "one_token": [(1, 1)],
    "tokens": [(15, 1), (16, 1), (63, 1), (64, 1), (127, 1), (300, 1)],
    "drafts": [(40, 5), (0, 3), (129, 2)],
    "empty_among": [(0, 0), (7, 1), (50, 0), (0, 2), (3, 0)],
    "prompt": [(0, 150)],
    "chunks": [(33, 70), (0, 129), (200, 64)],
    "mixed": [(90, 1), (5, 77), (0, 1), (250, 1), (64, 31)],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(3, 3, 16), (14, 2, 32), (8, 1, 128)])
@pytest.mark.parametrize("name", SEQUENCES)
def test_attend_matches_the_definition(dtype, dim, heads, kv_heads, page, name):
    s = ref.batch(SEQUENCES[name], kv_heads, heads, dim, page, dtype, 1, pad=3)
    got = _check(s, dim ** -0.5)
    assert (got[int(s["cu_tokens"][-1]):] == 0).all()


@pytest.mark.parametrize("heads,kv_heads", [(32, 1), (33, 1), (128, 1), (66, 2), (20, 4)])
def test_attend_takes_every_group_size(heads, kv_heads):
    s = ref.batch([(20, 1), (70, 3), (0, 40)], kv_heads, heads, 64, 16, torch.float16, 2)
    _check(s)


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128)])
def test_attend_splits_long_contexts(dtype, dim):
    """Few sequences with long contexts: items are cut into several shares."""
    _check(ref.batch([(6000, 1)], 2, 4, dim, 16, dtype, 3), dim ** -0.5)
    _check(ref.batch([(3001, 40), (10, 1), (4100, 1)], 1, 4, dim, 64, dtype, 4), dim ** -0.5)


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("cached", [7900, 8300, 9000, 9600, 17000, 30000])
def test_attend_joins_many_pieces(dtype, dim, new, cached):
    """One long sequence: about 15 to 60 pieces of an item, 17 and 33 among them."""
    _check(ref.batch([(cached, new)], 1, 5, dim, 64, dtype, cached % 89))


def test_items_cut_anywhere_join_alike():
    """Lengths that move every border, beside a neighbour in the same shares."""
    for cached in range(9000, 12000, 131):
        _check(ref.batch([(200, 2), (cached, 1), (150, 1), (cached - 2000, 33)], 1, 4, 64, 32,
                         torch.float16, cached % 97))


def test_joins_of_groups_of_pieces():
    """Counts of pieces from under 48 to over 65: joined at once, or by 16 with a last group
    of any size, one piece among them."""
    for cached in range(24000, 35000, 509):
        _check(ref.batch([(cached, 1 + cached % 2)], 1, 3, 64, 128, torch.float16, cached % 83))


def test_attend_many_sequences():
    """More sequences than threads of a block."""
    gen = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 40, (600, 2), generator=gen).tolist()
    _check(ref.batch([(p, min(n, 3)) for p, n in lens], 1, 2, 64, 16, torch.float16, 5, pad=1))


@pytest.mark.parametrize("scale", [-0.125, 0.0, 1.0, 1e-30])
@pytest.mark.parametrize("name", ["tokens", "chunks"])
def test_attend_scales(scale, name):
    _check(ref.batch(SEQUENCES[name], 2, 6, 64, 16, torch.float16, 6), scale)


@pytest.mark.parametrize("name", ["tokens", "mixed", "drafts"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -65504.0])
def test_rows_that_hold_no_key_do_not_matter(name, junk):
    """Unused pages, and rows of the last page past the length, hold anything."""
    s = ref.batch(SEQUENCES[name], 2, 6, 64, 32, torch.float16, 7)
    want = _attend(s, 0.125)
    used = torch.zeros(s["k_pages"].shape[0], 32, dtype=torch.bool)
    for b, n in enumerate(s["seq_lens"].tolist()):
        for j in range(n):
            used[s["page_table"][b, j // 32], j % 32] = True
    for pages in ("k_pages", "v_pages"):
        s[pages].transpose(1, 2)[~used] = junk
    assert torch.equal(_attend(s, 0.125), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(6, 2), (14, 1)])
@pytest.mark.parametrize("where", [(1, 2, 3), (0, 5, 40), (130, 131, 149)])
def test_later_tokens_that_are_not_finite_do_not_matter(dtype, dim, heads, kv_heads, where):
    """A token's NaN or infinity reaches the queries at and after it, and no other:
    not through a weight of zero (0 * inf) of a query before it."""
    s = ref.batch([(9, 150), (33, 4), (60, 8)], kv_heads, heads, dim, 16, dtype, 40)
    want = _attend(s, 0.125).cpu()
    at = [w for w in where], [33 + 1, 33 + 2], [60 + 3]
    for b, tokens in enumerate(at):
        for i, token in enumerate(tokens):
            pos = token + (9 if b == 0 else 0)
            page = s["page_table"][b, pos // 16]
            s["v_pages"][page, :, pos % 16, i::5] = [float("inf"), float("nan"), -float("inf")][i % 3]
            s["k_pages"][page, :, pos % 16, 0] = float("nan")
    got = _attend(s, 0.125).cpu()
    bounds = s["cu_tokens"].tolist()
    for b, first in enumerate([min(where), 1, 3]):
        assert torch.equal(got[bounds[b]:bounds[b] + first], want[bounds[b]:bounds[b] + first])
        assert not torch.isfinite(got[bounds[b] + first:bounds[b + 1]]).any()


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("name", ["drafts", "chunks"])
def test_infinite_values_reach_only_their_dims(value, name):
    """With finite keys, a value dim that is not finite leaves that dim not finite for
    the queries that see it, and changes no other. (Items of few rows, also the last
    ones of a chunk, split each weight into hi + lo with |lo| <= hi / 2048 of either
    sign, so an infinity may come out as inf hi + inf lo = NaN.)"""
    s = ref.batch(SEQUENCES[name], 2, 6, 64, 16, torch.float16, 41)
    want = _attend(s, 0.125).cpu()
    bounds, lens = s["cu_tokens"].tolist(), s["seq_lens"].tolist()
    for b, n in enumerate(lens):
        pos = n - 2
        s["v_pages"][s["page_table"][b, pos // 16], :, pos % 16, 7] = value
    got = _attend(s, 0.125).cpu()
    for b in range(len(lens)):
        before, after = slice(bounds[b], bounds[b + 1] - 2), slice(bounds[b + 1] - 2, bounds[b + 1])
        assert torch.equal(got[before], want[before])
        rest = [d for d in range(64) if d != 7]
        assert torch.equal(got[after][..., rest], want[after][..., rest])
        assert not torch.isfinite(got[after][..., 7]).any()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("name", ["tokens", "mixed", "chunks"])
def test_page_ids_outside_the_pool_have_no_keys(page, name):
    s = ref.batch(SEQUENCES[name], 2, 6, 64, page, torch.float16, 8)
    pages = s["k_pages"].shape[0]
    for b, bad in enumerate([-1, pages, 2 ** 31 - 1, -2 ** 31, pages + 7, -5][:len(s["seq_lens"])]):
        s["page_table"][b, (b * 7) % s["page_table"].shape[1]] = bad
    s["page_table"][-1, :] = -1  # a sequence with no page at all
    got = _check(s)
    assert (got[int(s["cu_tokens"][-2]):] == 0).all()


def test_lengths_that_do_not_fit_the_tokens():
    """A length under the token count (the first tokens have no position), zero,
    negative, and one past the page table (keys end there)."""
    s = ref.batch([(20, 5), (0, 40), (30, 2), (40, 50), (60, 1)], 1, 4, 64, 16, torch.float16, 9)
    s["seq_lens"] = torch.tensor([3, 0, -4, 20, 10 ** 6], dtype=torch.int32)
    got = _check(s)
    assert (got[:2] == 0).all() and (got[5:47] == 0).all()
    s["seq_lens"] = torch.full((5,), -2 ** 31, dtype=torch.int32)
    assert (_check(s) == 0).all()


def test_token_bounds_that_do_not_fit_the_tensor():
    """cu_tokens past the packed rows ends with them; rows before the first
    sequence are zero."""
    s = ref.batch([(20, 5), (9, 40)], 1, 4, 64, 16, torch.float16, 10)
    s["q"] = s["q"][:30]
    got = _attend(s, 0.125).cpu()
    want, bound = ref.attend(s["q"], *(s[name] for name in CACHE), 0.125)
    assert ((got.double() - want).abs() <= bound).all()
    s["cu_tokens"] = torch.tensor([4, 9, 9], dtype=torch.int32)
    got = _attend(s, 0.125).cpu()
    assert (got[:4] == 0).all() and (got[9:] == 0).all() and (got[4:9] != 0).any()


@pytest.mark.parametrize("repeats", [3, 200])
def test_bounds_that_fall_have_no_sequences(repeats):
    """Bounds that go up and down claim more rows than there are: the outputs are
    zero, and the next call is as if nothing had been."""
    s = ref.batch([(40, 20)] * repeats, 1, 4, 64, 16, torch.float16, 42)
    want = _attend(s, 0.125)
    good = s["cu_tokens"].clone()
    s["cu_tokens"][0::2], s["cu_tokens"][1::2] = 0, s["q"].shape[0]
    assert (_attend(s, 0.125) == 0).all()
    s["cu_tokens"] = good
    assert torch.equal(_attend(s, 0.125), want)


def test_attend_takes_slices_of_a_projection():
    s = ref.batch(SEQUENCES["mixed"], 2, 6, 64, 16, torch.float16, 11)
    total = s["q"].shape[0]
    projected = torch.randn(total, 10, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    q = projected[:, 1:7]
    assert not q.is_contiguous()
    assert torch.equal(_attend(s, 0.125, q), _attend(s, 0.125, q.contiguous()))
    token_last = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(_attend(s, 0.125, token_last), _attend(s, 0.125, q))


def test_results_do_not_depend_on_timing():
    s = ref.batch([(3001, 40), (10, 1), (6100, 1)], 1, 4, 64, 16, torch.float16, 12)
    first = _attend(s, 0.125)
    for _ in range(5):
        assert torch.equal(_attend(s, 0.125), first)


def test_peaky_rows():
    """One key carries its row: its weight's rounding cancels against the sum."""
    s = ref.batch([(500, 1), (100, 60)], 1, 2, 64, 16, torch.float16, 13)
    s["q"] *= 4
    s["k_pages"] *= 4
    got = _attend(s, 0.125).cpu()
    want, _ = ref.attend(s["q"], *(s[name] for name in CACHE), 0.125)
    # Everything in range, most rows settled by one key: 2 roundings of |v| <= ~4.5.
    assert (got.double() - want).abs().max() <= 4.5 * (4 * 2.0 ** -11)


def test_offsets_past_32_bits():
    """A pool of over 2^32 elements; the sequence's pages lie at its ends."""
    page, kv_heads, dim = 1024, 8, 128
    pages = 2 ** 32 // (page * kv_heads * dim) + 3
    pool = torch.empty(pages, kv_heads, page, dim, dtype=torch.float16, device="cuda")
    small = ref.batch([(2100, 3), (1500, 1)], kv_heads, 8, dim, page, torch.float16, 14, spare=0)
    where = torch.tensor([pages - 1, 0, pages - 2, 1, pages - 3], dtype=torch.int64)
    pool[where.cuda()] = small["k_pages"].cuda()
    cache = [small[n].cuda() for n in CACHE]
    want = flashattn_cuda.attend_paged(small["q"].cuda(), cache[0], cache[0], *cache[2:], 0.1)
    table = where[small["page_table"].long()].to(torch.int32).cuda()
    got = flashattn_cuda.attend_paged(small["q"].cuda(), pool, pool, table, *cache[3:], 0.1)
    assert torch.equal(got, want)
    # The append's last rows land in the last page.
    flashattn_cuda.append_paged(pool, pool, small["k"].cuda(), small["k"].cuda(), table,
                                *cache[3:])
    new = pool[where[small["page_table"][0, 2].long()]].cpu()
    assert torch.equal(new[:, 2100 - 2048:2103 - 2048].transpose(0, 1), small["k"][:3])
    del pool
    torch.cuda.empty_cache()


# ---- append ----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary,interleaved", [
    (64, 0, False), (64, 64, False), (64, 32, True), (128, 128, True), (128, 48, False)])
@pytest.mark.parametrize("name", SEQUENCES)
def test_append_writes_the_new_rows_only(dtype, dim, rotary, interleaved, name):
    s = ref.batch(SEQUENCES[name], 2, 6, dim, 32, dtype, 15, pad=4)
    cache = {n: s[n].cuda() for n in CACHE}
    inv_freq = None
    if rotary:
        inv_freq, _ = flashattn_cuda.rope_frequencies(rotary)
        out = flashattn_cuda.append_paged(
            *(cache[n] for n in CACHE[:2]), s["k"].cuda(), s["v"].cuda(),
            *(cache[n] for n in CACHE[2:]), q=s["q"].cuda(), inv_freq=inv_freq.cuda(),
            interleaved=interleaved, factor=1.5).cpu()
    else:
        assert flashattn_cuda.append_paged(*(cache[n] for n in CACHE[:2]), s["k"].cuda(),
                                           s["v"].cuda(), *(cache[n] for n in CACHE[2:])) is None
    k_pages, v_pages = cache["k_pages"].cpu(), cache["v_pages"].cpu()
    untouched = torch.ones(k_pages.shape[0], 32, dtype=torch.bool)
    bounds = s["cu_tokens"].tolist()
    for b, n in enumerate(s["seq_lens"].tolist()):
        for t in range(bounds[b], bounds[b + 1]):
            pos = n - bounds[b + 1] + t
            page, row = int(s["page_table"][b, pos // 32]), pos % 32
            untouched[page, row] = False
            assert torch.equal(v_pages[page, :, row], s["v"][t])
            if not rotary:
                assert torch.equal(k_pages[page, :, row], s["k"][t])
                continue
            for got, x in ((k_pages[page, :, row], s["k"][t]), (out[t], s["q"][t])):
                want, size = ref.turn(x, torch.tensor([pos]), inv_freq, interleaved, 1.5)
                assert ((got.double() - want).abs() <= ref.turn_bound(want, size, dtype)).all()
    for got, before in ((k_pages, s["k_pages"]), (v_pages, s["v_pages"])):
        assert torch.equal(got.transpose(1, 2)[untouched], before.transpose(1, 2)[untouched])
    if rotary:
        assert (out[bounds[-1]:] == 0).all()


def test_append_skips_tokens_without_a_place():
    s = ref.batch([(20, 5), (0, 4), (30, 3), (14, 4)], 2, 4, 64, 16, torch.float16, 16)
    s["seq_lens"] = torch.tensor([3, -4, 10 ** 6, 18], dtype=torch.int32)
    s["page_table"][3, 1] = s["k_pages"].shape[0]  # rows 16, 17 of the last sequence
    cache = [s[n].cuda() for n in CACHE]
    inv_freq = flashattn_cuda.rope_frequencies(64)[0].cuda()
    flashattn_cuda.append_paged(*cache[:2], s["k"].cuda(), s["v"].cuda(), *cache[2:],
                                q=s["q"].cuda(), inv_freq=inv_freq)
    want = s["v_pages"].clone()
    want[s["page_table"][0, 0], :, 0:3] = s["v"][2:5].transpose(0, 1)
    want[s["page_table"][3, 0], :, 14:16] = s["v"][12:14].transpose(0, 1)
    assert torch.equal(cache[1].cpu(), want)
    changed = (cache[0].cpu() != s["k_pages"]).any(-1).any(1).nonzero().tolist()
    first, last = int(s["page_table"][0, 0]), int(s["page_table"][3, 0])
    assert set(map(tuple, changed)) <= {(first, 0), (first, 1), (first, 2), (last, 14), (last, 15)}


# ---- together --------------------------------------------------------------------


@pytest.mark.parametrize("heads,kv_heads,dim,chunk", [(6, 2, 64, 48), (8, 8, 64, 100),
                                                      (8, 2, 128, 33)])
def test_chunked_prompt_equals_rope_and_prefill(heads, kv_heads, dim, chunk):
    """A prompt cut into chunks through append_paged and attend_paged, then single
    tokens, gives the rows of rope + prefill_gqa over the whole sequence."""
    total, tail, page = 200, 6, 16
    scale = dim ** -0.5
    gen = torch.Generator().manual_seed(17)
    q, k, v = (torch.randn(total, h, dim, generator=gen).half().cuda()
               for h in (heads, kv_heads, kv_heads))
    inv_freq = flashattn_cuda.rope_frequencies(dim)[0].cuda()
    positions = torch.arange(total, dtype=torch.int32, device="cuda")
    turned = [flashattn_cuda.rope(x.transpose(0, 1)[None], positions, inv_freq) for x in (q, k)]
    whole = flashattn_cuda.prefill_gqa(*turned, v.transpose(0, 1)[None].contiguous(), True, scale)
    pages = (total + page - 1) // page
    table = torch.randperm(pages, generator=gen).to(torch.int32)[None].cuda()
    k_pages = torch.zeros(pages, kv_heads, page, dim, dtype=torch.float16, device="cuda")
    v_pages = torch.zeros_like(k_pages)
    steps = list(range(0, total - tail, chunk)) + list(range(total - tail, total))
    outs = []
    for at, stop in zip(steps, steps[1:] + [total]):
        lens = torch.tensor([stop], dtype=torch.int32, device="cuda")
        bounds = torch.tensor([0, stop - at], dtype=torch.int32, device="cuda")
        qt = flashattn_cuda.append_paged(k_pages, v_pages, k[at:stop], v[at:stop], table, lens,
                                         bounds, q[at:stop], inv_freq)
        assert torch.equal(qt, turned[0][0, :, at:stop].transpose(0, 1))
        outs.append(flashattn_cuda.attend_paged(qt, k_pages, v_pages, table, lens, bounds, scale))
    got = torch.cat(outs).float()
    # Two fp16 results of one row: a rounding of |o| each and of the weights each;
    # rows of few keys have |o| up to max |v|.
    bound = 4 * 2.0 ** -11 * v.float().abs().max()
    assert (got - whole[0].transpose(0, 1).float()).abs().max() <= bound


def test_decode_steps_equal_the_contiguous_cache():
    """append_kv + decode_gqa and append_paged + attend_paged, token by token."""
    batch, heads, kv_heads, dim, page, length, steps = 5, 8, 2, 64, 16, 80, 12
    gen = torch.Generator().manual_seed(18)
    lens = torch.tensor([0, 15, 16, 33, 60], dtype=torch.int32)
    k_cache = torch.randn(batch, kv_heads, length, dim, generator=gen).half().cuda()
    v_cache = torch.randn(batch, kv_heads, length, dim, generator=gen).half().cuda()
    table = torch.randperm(batch * length // page, generator=gen).to(torch.int32)
    table = table.reshape(batch, -1).cuda()
    paged = []
    for cache in (k_cache, v_cache):
        pages = torch.empty(batch * length // page, kv_heads, page, dim, dtype=torch.float16,
                            device="cuda")
        pages[table.flatten().long()] = cache.reshape(batch, kv_heads, -1, page, dim).transpose(
            1, 2).flatten(0, 1)
        paged.append(pages)
    lens_c, lens_p = lens.cuda(), lens.cuda()
    bounds = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        q, k, v = (torch.randn(batch, h, dim, generator=gen).half().cuda()
                   for h in (heads, kv_heads, kv_heads))
        flashattn_cuda.append_kv(k_cache, v_cache, k[:, :, None], v[:, :, None], lens_c)
        want = flashattn_cuda.decode_gqa(q[:, :, None], k_cache, v_cache, lens_c, 0.125)
        lens_p += 1
        flashattn_cuda.append_paged(*paged, k, v, table, lens_p, bounds)
        got = flashattn_cuda.attend_paged(q, *paged, table, lens_p, bounds, 0.125)
        # Both split the weights, so each output is its own rounding of nearly one value.
        spread = 2.0 ** -10 * want[:, :, 0].float().abs() + 2e-5
        assert ((got.float() - want[:, :, 0].float()).abs() <= spread).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step_replays(dtype):
    """Length, append and attention of a padded step in one graph, replayed with
    eager work and synchronisation between, against the eager calls."""
    s = ref.batch([(40, 1), (3000, 1), (0, 3)], 2, 6, 64, 16, dtype, 19, pad=2, extra_columns=3)
    cache = [s[n].cuda() for n in CACHE]
    q, k, v = s["q"].cuda(), s["k"].cuda(), s["v"].cuda()
    inv_freq = flashattn_cuda.rope_frequencies(64)[0].cuda()
    grow = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")

    def step(c):
        c[3].add_(grow)
        turned = flashattn_cuda.append_paged(*c[:2], k, v, *c[2:], q, inv_freq)
        return flashattn_cuda.attend_paged(turned, *c, 0.125)

    step([x.clone() for x in cache])
    torch.cuda.synchronize()
    eager = [x.clone() for x in cache]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(50 + i)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(eager))
        for a, b in zip(cache, eager):
            assert torch.equal(a, b)


def test_many_empty_sequences():
    """Thousands of sequences without tokens around a few with them."""
    sequences = [(0, 0)] * 3000 + [(2900, 3), (40, 1)] + [(0, 0)] * 2000 + [(700, 40)] + [(0, 0)] * 999
    _check(ref.batch(sequences, 1, 4, 64, 16, torch.float16, 21))


@pytest.mark.parametrize("before,between,after", [(0, 62, 0), (1, 63, 5), (64, 64, 64),
                                                  (3, 127, 1), (70, 200, 130)])
def test_runs_of_empty_sequences(before, between, after):
    """Slots without tokens, cached lengths kept, before, between and behind those in use."""
    idle = [(33, 0)]
    _check(ref.batch(idle * before + [(90, 1)] + idle * between + [(20, 40)] + idle * between
                     + [(700, 3)] + idle * after, 2, 4, 64, 16, torch.float16, 27))


def test_a_stream_without_arrival_counters():
    """hipStreamPerThread names another stream in every thread, so the library keeps no
    counters for it and zeroes some in the workspace: same results, call after call."""
    s = ref.batch([(3001, 40), (10, 1), (6100, 1)], 1, 4, 64, 16, torch.float16, 24)
    want = _attend(s, 0.125)
    t = {n: x.cuda() for n, x in s.items()}
    lib = ctypes.CDLL(os.path.join(os.path.dirname(flashattn_cuda.__file__), "libflashattn_hip.so"))
    lib.fa_attend_paged_workspace_bytes.restype = ctypes.c_size_t
    tokens, heads, dim = t["q"].shape
    cache = Paged(*(t[n].data_ptr() for n in CACHE), 0, len(t["seq_lens"]), tokens, 1, dim, 16,
                  t["k_pages"].shape[0], t["page_table"].shape[1])
    rows = Rows(t["q"].data_ptr(), t["q"].stride(0), t["q"].stride(1))
    need = lib.fa_attend_paged_workspace_bytes(tokens, heads, 1, dim)
    workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    out = [torch.empty_like(t["q"]) for _ in range(3)]
    torch.cuda.synchronize()
    for o in out:
        assert lib.fa_attend_paged(ctypes.byref(cache), ctypes.byref(rows),
                                   ctypes.c_void_p(o.data_ptr()), heads, ctypes.c_float(0.125),
                                   ctypes.c_void_p(workspace.data_ptr()), ctypes.c_size_t(need),
                                   ctypes.c_void_p(2)) == 0
    torch.cuda.synchronize()  # every stream, the per-thread one included
    assert all(torch.equal(o, want) for o in out)
    # A workspace one byte short is refused.
    assert lib.fa_attend_paged(ctypes.byref(cache), ctypes.byref(rows),
                               ctypes.c_void_p(out[0].data_ptr()), heads, ctypes.c_float(0.125),
                               ctypes.c_void_p(workspace.data_ptr()), ctypes.c_size_t(need - 1),
                               None) == 2


def test_more_captures_than_counter_slots():
    """Every capture takes a slot of arrival counters until none is left; the graphs
    captured after that zero counters in their workspace. All replay to the same bits."""
    s = {n: t.cuda() for n, t in ref.batch([(2000, 40), (10, 1)], 1, 4, 64, 16, torch.float16,
                                           26).items()}
    want = _attend(s, 0.125)
    graphs, outs = [], []
    for _ in range(70):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_attend(s, 0.125))
        graphs.append(graph)
    for _ in range(3):
        for out in outs:
            out.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)
        assert torch.equal(_attend(s, 0.125), want)


def test_two_streams_at_once():
    batches = [ref.batch([(3001, 40), (10, 1)], 2, 4, 64, 16, torch.float16, 20 + i)
               for i in range(2)]
    want = [_attend(s, 0.125) for s in batches]
    on_gpu = [(s["q"].cuda(), *(s[n].cuda() for n in CACHE)) for s in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(flashattn_cuda.attend_paged(*on_gpu[i], 0.125))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_host_threads_at_once():
    """Threads on streams of their own, attending and appending to caches of their own."""
    batches = [ref.batch([(3001 + i, 1), (100, 40), (10, 1)], 2, 4, 64, 16, torch.float16, 30 + i)
               for i in range(4)]
    want = [_attend(s, 0.125) for s in batches]
    on_gpu = [{n: x.cuda() for n, x in s.items()} for s in batches]
    torch.cuda.synchronize()
    got = [[] for _ in batches]

    def work(i):
        s = on_gpu[i]
        cache = [s[n] for n in CACHE]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i].append(flashattn_cuda.attend_paged(s["q"], *cache, 0.125))
            flashattn_cuda.append_paged(*cache[:2], s["k"], s["v"], *cache[2:])
            got[i].append(flashattn_cuda.attend_paged(s["q"], *cache, 0.125))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(batches))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    for i, s in enumerate(on_gpu):
        assert len(got[i]) == 11 and all(torch.equal(x, want[i]) for x in got[i][:10])
        assert torch.equal(got[i][10], flashattn_cuda.attend_paged(
            s["q"], *(s[n] for n in CACHE), 0.125))


@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences_that_share_pages(dtype):
    """A common prefix is stored once, and one page stands twice in a table."""
    s = ref.batch([(160, 1), (160, 33), (500, 3)], 2, 6, 128, 32, dtype, 25)
    s["page_table"][1, :5] = s["page_table"][0, :5]
    s["page_table"][2, 3] = s["page_table"][2, 9]
    _check(s, 0.09)


def test_no_tokens():
    s = ref.batch([(5, 0), (0, 0)], 2, 4, 64, 16, torch.float16, 22)
    assert _attend(s, 0.125).shape == (0, 4, 64)
    cache = [s[n].cuda() for n in CACHE]
    flashattn_cuda.append_paged(*cache[:2], s["k"].cuda(), s["v"].cuda(), *cache[2:])
    assert torch.equal(cache[0].cpu(), s["k_pages"])


def test_refusals():
    s = {n: x.cuda() for n, x in
         ref.batch([(20, 1), (3, 2)], 2, 4, 64, 16, torch.float16, 23).items()}
    inv_freq = flashattn_cuda.rope_frequencies(64)[0].cuda()

    def attend(scale=0.125, **new):
        t = {**s, **new}
        return flashattn_cuda.attend_paged(t["q"], *(t[n] for n in CACHE), scale)

    def append(q=None, w=None, **new):
        t = {**s, **new}
        return flashattn_cuda.append_paged(t["k_pages"], t["v_pages"], t["k"], t["v"],
                                           *(t[n] for n in CACHE[2:]), q=q, inv_freq=w)

    odd = torch.zeros(4, 2, 24, 64, dtype=torch.float16, device="cuda")
    bad = [
        (lambda: attend(q=s["q"].float()), "must be fp16 or bf16"),
        (lambda: attend(q=s["q"].bfloat16()), "same type"),
        (lambda: attend(q=s["q"][0]), "must be 3-D"),
        (lambda: attend(q=s["q"].cpu()), "must be a CUDA tensor"),
        (lambda: attend(q=s["q"][:, :3]), "divide the query head count"),
        (lambda: attend(q=s["q"][..., :32]), "same type and head_dim"),
        (lambda: attend(q=torch.zeros(3, 258, 64, dtype=torch.float16, device="cuda")), "at most 128"),
        (lambda: attend(q=s["q"].transpose(1, 2).contiguous().transpose(1, 2)), "16 bytes"),
        (lambda: attend(k_pages=odd, v_pages=odd), "page_size must be a power of two"),
        (lambda: attend(k_pages=s["k_pages"][:1]), "identical shapes"),
        (lambda: attend(k_pages=s["k_pages"][:, :, ::2], v_pages=s["v_pages"][:, :, ::2]),
         "contiguous"),
        (lambda: attend(k_pages=s["k_pages"][:0], v_pages=s["v_pages"][:0]), "at least one page"),
        (lambda: attend(page_table=s["page_table"].long()), "page_table must be int32"),
        (lambda: attend(page_table=s["page_table"][:1]), "must be \\[B, max_pages\\]"),
        (lambda: attend(page_table=s["page_table"][:, :0]), "at least one sequence and one page"),
        (lambda: attend(seq_lens=s["seq_lens"].cpu()), "seq_lens must be a CUDA tensor"),
        (lambda: attend(seq_lens=s["seq_lens"][None]), "seq_lens must be 1-D"),
        (lambda: attend(cu_tokens=s["cu_tokens"][:2]), "cu_tokens \\[B \\+ 1\\]"),
        (lambda: attend(scale=float("inf")), "scale must be finite"),
        (lambda: append(k=s["k"][:1]), "append_paged expects"),
        (lambda: append(k=s["q"], v=s["q"]), "append_paged expects"),
        (lambda: append(q=s["q"]), "together or neither"),
        (lambda: append(w=inv_freq), "together or neither"),
        (lambda: append(q=s["q"][:1], w=inv_freq), "same number of tokens"),
        (lambda: append(q=s["q"], w=inv_freq.float()), "float64"),
        (lambda: append(v=s["v"].bfloat16()), "same type"),
    ]
    for make, message in bad:
        with pytest.raises(RuntimeError, match=message):
            make()
