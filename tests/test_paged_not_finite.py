"""NaN and infinities that a query does see reach its row of ``attend_paged``, however
its keys are cut into pieces, and no other row."""

import pytest
import torch

import flashattn_cuda
import paged_reference as ref

pytestmark = pytest.mark.gpu
CACHE = ("k_pages", "v_pages", "page_table", "seq_lens", "cu_tokens")
# Keys of the one long sequence: an item that is not cut, of a few pieces, of up to 48, of more.
CACHED = [300, 3000, 9000, 20000, 31000]


def _attend(s):
    return flashattn_cuda.attend_paged(s["q"].cuda(), *(s[n].cuda() for n in CACHE), 0.125).cpu()


def _rows(s, b, first, last):
    """Index of the page rows of positions [first, last) of sequence b, over (page, row)."""
    page = s["k_pages"].shape[2]
    pos = torch.arange(first, last)
    return s["page_table"][b, pos // page].long(), pos % page


def _check_rest(s, got, spoiled):
    """Rows that are not spoiled are the definition's."""
    want, bound = ref.attend(s["q"], *(s[n] for n in CACHE), 0.125)
    rest = ~spoiled
    assert torch.isfinite(got[rest]).all()
    assert ((got.double() - want).abs()[rest] <= bound[rest]).all()


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("new,token", [(1, 0), (3, 2), (40, 7), (40, 39)])
@pytest.mark.parametrize("cached", CACHED)
def test_a_query_that_is_not_a_number(dtype, dim, new, token, cached):
    """Narrow items (also the last 8 of the 40 tokens) and wide ones."""
    s = ref.batch([(cached, new), (50, 2)], 1, 4, dim, 64, dtype, 70)
    s["q"][token, 1, 5] = float("nan")
    got = _attend(s)
    spoiled = torch.zeros(got.shape[:2], dtype=torch.bool)
    spoiled[token, 1] = True
    assert torch.isnan(got[spoiled]).all()
    s["q"][token, 1, 5] = 0.0
    _check_rest(s, got, spoiled)


@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("where", ["first", "middle", "last", "all"])
@pytest.mark.parametrize("cached", CACHED)
def test_keys_that_are_not_numbers(new, where, cached):
    """600 keys (more than a piece of the least size) or all of them."""
    s = ref.batch([(cached, new), (50, 2)], 2, 4, 64, 64, torch.float16, 71)
    span = min(600, cached)
    first = {"first": 0, "middle": (cached - span) // 2, "last": cached - span, "all": 0}[where]
    pages, rows = _rows(s, 0, first, cached + 1 if where == "all" else first + span)
    s["k_pages"][pages, 1, rows, 3] = float("nan")
    got = _attend(s)
    spoiled = torch.zeros(got.shape[:2], dtype=torch.bool)
    spoiled[:new, 2:] = True  # the query heads of K/V head 1
    assert torch.isnan(got[spoiled]).all()
    s["k_pages"][pages, 1, rows, 3] = 0.0
    _check_rest(s, got, spoiled)


@pytest.mark.parametrize("cached", [9000, 31000])
def test_pieces_of_keys_that_are_not_numbers(cached):
    """NaN in the keys up to anywhere that a first piece may end."""
    s = ref.batch([(cached, 1)], 1, 4, 64, 64, torch.float16, 73)
    cache = {n: s[n].cuda() for n in CACHE}
    pages, rows = (x.cuda() for x in _rows(s, 0, 0, cached))
    for stop in range(64, 1600, 64):
        k_pages = cache["k_pages"].clone()
        k_pages[pages[:stop], 0, rows[:stop], 3] = float("nan")
        got = flashattn_cuda.attend_paged(s["q"].cuda(), k_pages,
                                          *(cache[n] for n in CACHE[1:]), 0.125)
        assert torch.isnan(got).all(), stop


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("cached", CACHED)
def test_spoiled_keys_and_values_of_weight_zero(new, what, cached):
    """Keys whose weights come out as zero in 32 bits beside key 0's, one of them with a score
    or a value that is not finite: 0 * NaN and 0 * inf are NaN, in one piece or in many."""
    gone = ref.batch([(cached, new)], 1, 2, 64, 64, torch.float16, 72)
    gone["q"].zero_()
    gone["q"][..., 0] = 40.0
    gone["k_pages"][..., 0] = -20.0  # scores of -100 and 200: 433 powers of two apart
    pages, rows = _rows(gone, 0, 0, 1)
    gone["k_pages"][pages, :, rows, 0] = 40.0
    at = _rows(gone, 0, cached - 40, cached - 39)
    got = []
    for name in ("k_pages", "v_pages"):
        s = {n: x.clone() for n, x in gone.items()}
        s[name][at[0], :, at[1], 0] = what
        got.append(_attend(s))
    assert not torch.isfinite(got[0]).any()  # the score is NaN or inf
    assert not torch.isfinite(got[1][..., 0]).any()
    assert torch.equal(got[1][..., 1:], _attend(gone)[..., 1:])
