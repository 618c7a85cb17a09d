"""Packed rows that belong to no sequence: ``append_paged`` writes none of them and
``attend_paged`` gives zeros for them."""

import pytest
import torch

import flashattn_cuda
import paged_reference as ref

pytestmark = pytest.mark.gpu
CACHE = ("k_pages", "v_pages", "page_table", "seq_lens", "cu_tokens")


def _append(s, inv_freq):
    """(q_out, k_pages, v_pages) after the append, on the CPU."""
    cache = [s[n].cuda() for n in CACHE]
    with_q = {} if inv_freq is None else {"q": s["q"].cuda(), "inv_freq": inv_freq.cuda()}
    out = flashattn_cuda.append_paged(*cache[:2], s["k"].cuda(), s["v"].cuda(), *cache[2:], **with_q)
    return None if out is None else out.cpu(), cache[0].cpu(), cache[1].cpu()


def _check_append(s, rotary):
    """Tokens t in [cu_tokens[b], cu_tokens[b + 1]) lie at seq_lens[b] - cu_tokens[b + 1] + t;
    every other row of the pages is as it was, every other row of q_out zero."""
    inv_freq = flashattn_cuda.rope_frequencies(rotary)[0] if rotary else None
    out, k_pages, v_pages = _append(s, inv_freq)
    page = k_pages.shape[2]
    untouched = torch.ones(k_pages.shape[0], page, dtype=torch.bool)
    outside = torch.ones(s["k"].shape[0], dtype=torch.bool)
    bounds = s["cu_tokens"].tolist()
    for b, n in enumerate(s["seq_lens"].tolist()):
        for t in range(max(bounds[b], 0), min(bounds[b + 1], len(outside))):
            pos = n - bounds[b + 1] + t
            at, row = int(s["page_table"][b, pos // page]), pos % page
            untouched[at, row] = outside[t] = False
            assert torch.equal(v_pages[at, :, row], s["v"][t])
            if not rotary:
                assert torch.equal(k_pages[at, :, row], s["k"][t])
                continue
            for got, x in ((k_pages[at, :, row], s["k"][t]), (out[t], s["q"][t])):
                want, size = ref.turn(x, torch.tensor([pos]), inv_freq, False)
                assert ((got.double() - want).abs() <= ref.turn_bound(want, size, x.dtype)).all()
    for got, before in ((k_pages, s["k_pages"]), (v_pages, s["v_pages"])):
        assert torch.equal(got.transpose(1, 2)[untouched], before.transpose(1, 2)[untouched])
    if rotary:
        assert outside.any() and (out[outside] == 0).all()


def _shifted(sequences, front, back, dtype=torch.float16, dim=64, page=16):
    """A batch with `front` packed rows before its first sequence and `back` behind its last."""
    s = ref.batch(sequences, 2, 4, dim, page, dtype, 60, pad=front + back)
    s["cu_tokens"] += front
    return s


@pytest.mark.parametrize("dtype,dim,rotary", [(torch.float16, 64, 64), (torch.bfloat16, 128, 48),
                                              (torch.float16, 64, 0)])
@pytest.mark.parametrize("sequences,front", [
    ([(20, 5), (9, 0)], 4),          # cu_tokens [4, 9, 9]
    ([(20, 5), (9, 3)], 1),
    ([(40, 1), (17, 1), (90, 1)], 1),  # single tokens, one row on
    ([(40, 1), (17, 1), (90, 1)], 2),
    ([(300, 0), (200, 40)], 70),     # an empty sequence first
    ([(500, 30)], 200)])
def test_append_leaves_rows_before_the_first_sequence(dtype, dim, rotary, sequences, front):
    for back in (0, 3):
        _check_append(_shifted(sequences, front, back, dtype, dim), rotary)


def test_append_of_a_part_of_a_batch():
    """The bounds of sequences i.. of a batch, with all of its packed rows."""
    whole = ref.batch([(33, 6), (50, 1), (0, 20), (70, 4)], 2, 4, 64, 16, torch.float16, 61)
    for i in range(1, 4):
        s = dict(whole)
        for name in ("page_table", "seq_lens", "cu_tokens"):
            s[name] = whole[name][i:].clone()
        _check_append(s, 64)


def test_append_with_bounds_that_start_below_zero():
    """A first bound below 0: tokens before row 0 are not in the tensors, the others keep
    their places."""
    s = ref.batch([(20, 9), (5, 3)], 2, 4, 64, 16, torch.float16, 62, pad=2)
    s["q"], s["k"], s["v"] = (s[n][4:] for n in ("q", "k", "v"))
    s["cu_tokens"] -= 4
    _check_append(s, 64)


@pytest.mark.parametrize("front", [1, 4, 129])
def test_both_calls_agree_on_what_is_outside(front):
    """append_paged + attend_paged of a batch behind `front` foreign rows are the ones of the
    batch alone, with zeros for those rows."""
    sequences = [(33, 70), (40, 1), (0, 3)]
    alone, s = (_shifted(sequences, n, 0) for n in (0, front))
    for name in ("q", "k", "v"):
        s[name] = torch.cat([s[name][-front:], alone[name]])
    for name in CACHE[:3]:
        s[name] = alone[name]
    inv_freq = flashattn_cuda.rope_frequencies(64)[0]
    outs = []
    for t in (alone, s):
        q, k_pages, v_pages = _append(t, inv_freq)
        o = flashattn_cuda.attend_paged(q.cuda(), k_pages.cuda(), v_pages.cuda(),
                                        *(t[n].cuda() for n in CACHE[2:]), 0.125).cpu()
        outs.append((q, k_pages, v_pages, o))
    for i in (0, 3):
        assert (outs[1][i][:front] == 0).all()
        assert torch.equal(outs[1][i][front:], outs[0][i])
    for i in (1, 2):
        assert torch.equal(outs[1][i], outs[0][i])


def _attend(s):
    return flashattn_cuda.attend_paged(s["q"].cuda(), *(s[n].cuda() for n in CACHE), 0.125).cpu()


@pytest.mark.parametrize("dtype,kv_heads,heads", [(torch.float16, 2, 4), (torch.bfloat16, 1, 40)])
def test_bounds_that_fall_give_no_row_to_two_sequences(dtype, kv_heads, heads):
    """A fall by one row or more, first, last or among many, also where the sequences claim no
    more rows than there are: zeros, and the next call is as if nothing had been."""
    for bounds, tokens in (([0, 5, 3, 4], 8), ([0, 5, 4, 4], 9), ([3, 2, 8, 8], 8),
                           ([0, 2, 4, 6, 8, 7], 8), ([0, 70, 60, 65], 200),
                           (list(range(150)) + [140] + [141] * 49, 150)):
        s = ref.batch([(40, 1)] * (len(bounds) - 1), kv_heads, heads, 64, 16, dtype, 63)
        s["q"] = torch.randn(tokens, heads, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
        s["cu_tokens"] = torch.tensor(bounds, dtype=torch.int32)
        assert (_attend(s) == 0).all(), bounds
        s["cu_tokens"] = torch.tensor(bounds, dtype=torch.int32).cummax(0)[0].to(torch.int32)
        want, bound = ref.attend(s["q"], *(s[n] for n in CACHE), 0.125)
        assert ((_attend(s).double() - want).abs() <= bound).all(), bounds


def test_bounds_that_fall_outside_the_rows_are_those_of_its_ends():
    """Bounds past the packed rows, or below them, end there; falls among them claim nothing."""
    s = ref.batch([(40, 5), (20, 3), (30, 0), (9, 0)], 2, 4, 64, 16, torch.float16, 64)
    want = _attend(s)
    s["cu_tokens"] = torch.tensor([0, 5, 8, 30, 12], dtype=torch.int32)
    assert torch.equal(_attend(s), want)
    # The first two sequences have no rows; the third's bounds are [-1, 5).
    s["cu_tokens"] = torch.tensor([-1, -9, -1, 5, 8], dtype=torch.int32)
    want, bound = ref.attend(s["q"], s["k_pages"], s["v_pages"], s["page_table"],
                             s["seq_lens"], s["cu_tokens"].clamp(min=0), 0.125)
    assert ((_attend(s).double() - want).abs() <= bound).all()


def test_append_with_bounds_that_fall():
    """A token goes to its place in a sequence whose bounds hold it, or nowhere; nothing but
    such places changes."""
    s = ref.batch([(40, 5), (20, 3), (30, 2)], 2, 4, 64, 16, torch.float16, 65)
    s["cu_tokens"] = torch.tensor([0, 5, 3, 6], dtype=torch.int32)
    cache = [s[n].cuda() for n in CACHE]
    flashattn_cuda.append_paged(*cache[:2], s["k"].cuda(), s["v"].cuda(), *cache[2:])
    changed = (cache[1].cpu() != s["v_pages"]).any(-1).any(1).nonzero().tolist()
    bounds, tokens = s["cu_tokens"].tolist(), set()
    for page, row in changed:
        places = [(b, t) for b, n in enumerate(s["seq_lens"].tolist())
                  for t in range(bounds[b], bounds[b + 1])
                  if int(s["page_table"][b, (n - bounds[b + 1] + t) // 16]) == page
                  and (n - bounds[b + 1] + t) % 16 == row]
        held = [t for _, t in places if torch.equal(cache[1][page, :, row].cpu(), s["v"][t])]
        assert len(held) == 1 and held[0] not in tokens
        tokens.add(held[0])


@pytest.mark.parametrize("tokens", [0, 7])
@pytest.mark.parametrize("columns", [0, 3])
def test_a_batch_of_no_sequences(tokens, columns):
    """No packed row belongs to one: nothing is written, and the outputs are zero."""
    s = ref.batch([(20, 5)], 2, 4, 64, 16, torch.float16, 66, pad=2)
    s["q"], s["k"], s["v"] = (s[n][:tokens] for n in ("q", "k", "v"))
    s["page_table"] = torch.zeros(0, columns, dtype=torch.int32)
    s["seq_lens"] = torch.zeros(0, dtype=torch.int32)
    s["cu_tokens"] = torch.zeros(1, dtype=torch.int32)
    for inv_freq in (None, flashattn_cuda.rope_frequencies(64)[0]):
        out, k_pages, v_pages = _append(s, inv_freq)
        assert torch.equal(k_pages, s["k_pages"]) and torch.equal(v_pages, s["v_pages"])
        assert out is None if inv_freq is None else torch.equal(out, torch.zeros_like(s["q"]))
    assert torch.equal(_attend(s), torch.zeros_like(s["q"]))
