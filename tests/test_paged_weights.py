"""``attend_paged`` where nearly all keys weigh next to nothing beside a few."""

import pytest
import torch

import flashattn_cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("top", [16.0, 17.0, 18.0, 20.0])
def test_many_keys_of_small_weight(dtype, dim, new, top):
    """16384 keys at 2^-23 to 2^-29 of the weight of four: 96 sequences on the same pages, so
    that an item's keys are one block's."""
    length, page, kv_heads, sequences = 16384, 128, 8, 96
    gen = torch.Generator().manual_seed(80)
    k = torch.zeros(length // page, kv_heads, page, dim, dtype=dtype)
    v = (1 + 0.25 * torch.randn(length // page, kv_heads, page, dim, generator=gen)).to(dtype)
    k[0, :, 0:128:32, 0] = top  # one in each wave's keys
    v[0, :, 0:128:32] = 0
    q = torch.zeros(sequences * new, kv_heads, dim, dtype=dtype)
    q[..., 0] = 1.0
    table = torch.arange(length // page, dtype=torch.int32).repeat(sequences, 1)
    lens = torch.full((sequences,), length, dtype=torch.int32)
    bounds = torch.arange(sequences + 1, dtype=torch.int32) * new
    got = flashattn_cuda.attend_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(),
                                      bounds.cuda(), 1.0).cpu().double()

    keys = k.transpose(0, 1).reshape(kv_heads, length, dim)[..., 0].double()
    values = v.transpose(0, 1).reshape(kv_heads, length, dim).double()
    p = (keys - top).exp()
    want = torch.stack([(p[:, :length - new + 1 + t, None] * values[:, :length - new + 1 + t]).sum(1)
                        / p[:, :length - new + 1 + t].sum(1)[:, None] for t in range(new)])
    u = torch.finfo(dtype).eps / 2
    # Weights and output rounded once each (the row sum takes the rounded weights); scores exact
    # but for the product with log2 e and the bound: 4 roundings of up to 32 powers of two, 2^-24
    # each; sums of 2^14 terms in fp32. A weight whose place is under the type's least normal
    # number is off by half its least step, relative to the row's largest weight 2^-32 at
    # most in fp16 (that one is held at 2^7 or more), in the numerator and in the sum.
    spread = 3 * u + 4 * 32 * 2.0 ** -24 + 2 * 2.0 ** 14 * 2.0 ** -24
    tiny = 2 * length * 2.0 ** -32 * values.abs().max() / 4 if dtype == torch.float16 else 0.0
    bound = want.abs() * spread + tiny + torch.finfo(dtype).tiny * 2.0 ** -8
    error = (got.reshape(sequences, new, kv_heads, dim) - want).abs()
    assert (error <= bound).all(), f"{(error / want.abs()).max():.3g} of the value off"
