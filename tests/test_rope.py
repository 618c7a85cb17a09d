"""Rotary positions (``rope``, ``rope_backward``, ``rope_frequencies``) against
their formula in 64 bits."""

import math

import pytest
import torch

import flashattn_cuda
import paged_reference as ref

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _rand(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen, dtype=torch.float32).to(dtype)


def _check(got, x, positions, inv_freq, interleaved, factor, sign=1):
    out, size = ref.turn(x, sign * positions[:, None], inv_freq, interleaved, factor)
    error = (got.cpu().double() - out).abs()
    assert got.dtype == x.dtype and got.is_contiguous()
    assert (error <= ref.turn_bound(out, size, x.dtype)).all(), error.max()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,heads,seq,dim,rotary,start", [
    (1, 1, 1, 64, 64, 0),
    (1, 12, 1, 64, 64, 511),
    (2, 3, 17, 64, 16, 5),
    (3, 14, 129, 64, 48, 100000),
    (2, 32, 65, 128, 128, 1000003),
    (2, 5, 33, 128, 32, 2000000000),
    (1, 300, 3, 128, 112, -7),
])
def test_rope_matches_the_formula(dtype, interleaved, batch, heads, seq, dim, rotary, start):
    x = _rand((batch, heads, seq, dim), dtype, 1)
    positions = (torch.arange(seq, dtype=torch.int32)[None] + start
                 + 3 * torch.arange(batch, dtype=torch.int32)[:, None])
    inv_freq, _ = flashattn_cuda.rope_frequencies(rotary)
    args = positions.cuda(), inv_freq.cuda(), interleaved, 1.25
    _check(flashattn_cuda.rope(x.cuda(), *args), x, positions, inv_freq, interleaved, 1.25)
    _check(flashattn_cuda.rope_backward(x.cuda(), *args), x, positions, inv_freq, interleaved,
           1.25, -1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rope_takes_views_and_shared_positions(dtype):
    batch, heads, seq, dim = 3, 6, 37, 64
    inv_freq, _ = flashattn_cuda.rope_frequencies(dim)
    positions = torch.arange(seq, dtype=torch.int32)
    projected = _rand((batch, seq, 3 * heads, dim), dtype, 2)
    x = projected[:, :, heads:2 * heads].transpose(1, 2)
    on_gpu = projected.cuda()[:, :, heads:2 * heads].transpose(1, 2)
    got = flashattn_cuda.rope(on_gpu, positions.cuda(), inv_freq.cuda())
    _check(got, x, positions[None].expand(batch, seq), inv_freq, False, 1.0)
    # One head's row shared by all heads (stride 0), every second position.
    one = _rand((batch, 1, 2 * seq, dim), dtype, 3)
    got = flashattn_cuda.rope(one.cuda()[:, :, ::2].expand(batch, heads, seq, dim),
                              positions.cuda(), inv_freq.cuda())
    _check(got, one[:, :, ::2].expand(batch, heads, seq, dim),
           positions[None].expand(batch, seq), inv_freq, False, 1.0)


@gpu
def test_rope_past_2_to_the_31_elements():
    """The last heads of a tensor of 2^31 and more elements, and of a token-major view of it."""
    inv_freq, _ = flashattn_cuda.rope_frequencies(128, device="cuda")
    positions = torch.arange(1 << 19, dtype=torch.int32, device="cuda")
    x = torch.empty((1, 33, 1 << 19, 128), dtype=torch.float16, device="cuda")
    x[:, :31] = 0
    x[:, 31:] = torch.randn((1, 2, 1 << 19, 128), device="cuda", dtype=torch.float16)
    want = flashattn_cuda.rope(x[:, 31:].contiguous(), positions, inv_freq)
    assert torch.equal(flashattn_cuda.rope(x, positions, inv_freq)[:, 31:], want)
    tokens = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(flashattn_cuda.rope(tokens, positions, inv_freq)[:, 31:], want)


@gpu
def test_rope_of_no_rows_is_empty():
    inv_freq = flashattn_cuda.rope_frequencies(64)[0].cuda()
    for shape in [(0, 2, 5, 64), (2, 0, 5, 64), (2, 2, 0, 64)]:
        x = torch.zeros(shape, dtype=torch.float16, device="cuda")
        positions = torch.zeros(shape[0], shape[2], dtype=torch.int32, device="cuda")
        assert flashattn_cuda.rope(x, positions, inv_freq).shape == shape


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_backward_is_the_gradient_of_forward(interleaved):
    """rope is linear, so the central difference of <rope(x), g> along d is its
    derivative: it has to be <rope_backward(g), d>. x +- d are exact in fp16
    (multiples of 1/8 up to 4), each product sum is taken in 64 bits."""
    shape, rotary = (2, 4, 19, 64), 32
    gen = torch.Generator().manual_seed(4)
    x, d = (torch.randint(-16, 17, shape, generator=gen).double() / 8 for _ in range(2))
    g = _rand(shape, torch.float16, 5)
    positions = torch.randint(0, 50000, shape[::2], generator=gen, dtype=torch.int32).cuda()
    inv_freq, factor = flashattn_cuda.rope_frequencies(
        rotary, scaling="parts", stretch=4.0, trained_length=2048)
    inv_freq = inv_freq.cuda()

    def loss(y):
        out = flashattn_cuda.rope(y.half().cuda(), positions, inv_freq, interleaved, factor)
        return (out.cpu().double() * g.double()).sum()

    slope = (loss(x + d) - loss(x - d)) / 2
    grad = flashattn_cuda.rope_backward(g.cuda(), positions, inv_freq, interleaved, factor)
    # Each side rounds its outputs once: half a step of |value| per element.
    u = ref.half_step(torch.float16) * 1.01
    reach = math.sqrt(2) * factor
    slack = u * reach * (((x + d).abs() + (x - d).abs()).amax() / 2 * g.double().abs().sum()
                         + g.double().abs().amax() * d.abs().sum())
    assert abs(slope - (grad.cpu().double() * d).sum()) <= slack


@gpu
def test_gradient_of_shared_heads_sums_over_them():
    """The gradient of a key head that several query heads read is the sum of
    theirs; rope_backward is linear, so it may be taken before or after the sum."""
    inv_freq = flashattn_cuda.rope_frequencies(64)[0].cuda()
    positions = torch.arange(23, dtype=torch.int32).cuda()
    g = _rand((2, 8, 23, 64), torch.float16, 6)
    one = torch.ones(64, dtype=torch.float64)
    each = flashattn_cuda.rope_backward(g.cuda(), positions, inv_freq).cpu().double()
    exact, size = ref.turn(g, -positions.cpu()[None, None], inv_freq.cpu(), False)
    want = exact.reshape(2, 2, 4, 23, 64).sum(2)
    got = each.reshape(2, 2, 4, 23, 64).sum(2)
    bound = ref.turn_bound(exact, size, torch.float16).reshape(2, 2, 4, 23, 64).sum(2) * one
    assert ((got - want).abs() <= bound).all()


@gpu
def test_rope_on_another_stream_and_in_a_graph():
    x = _rand((2, 4, 40, 128), torch.bfloat16, 7).cuda()
    positions = torch.arange(40, dtype=torch.int32).cuda()
    inv_freq = flashattn_cuda.rope_frequencies(128)[0].cuda()
    want = flashattn_cuda.rope(x, positions, inv_freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = flashattn_cuda.rope(x, positions, inv_freq)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flashattn_cuda.rope(x, positions, inv_freq)
    for step in range(3):
        x.copy_(_rand(x.shape, torch.bfloat16, 20 + step))
        positions.add_(11)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, flashattn_cuda.rope(x, positions, inv_freq))


@gpu
def test_rope_refuses():
    x = torch.zeros(1, 2, 8, 64, dtype=torch.float16, device="cuda")
    positions = torch.zeros(8, dtype=torch.int32, device="cuda")
    inv_freq = flashattn_cuda.rope_frequencies(64)[0].cuda()
    call = flashattn_cuda.rope
    bad = [
        (lambda: call(x.float(), positions, inv_freq), "must be fp16 or bf16"),
        (lambda: call(x.cpu(), positions, inv_freq), "must be a CUDA tensor"),
        (lambda: call(x[0], positions, inv_freq), "must be 4-D"),
        (lambda: call(x[..., :32], positions, inv_freq), "head_dim"),
        (lambda: call(x, positions.long(), inv_freq), "positions must be int32"),
        (lambda: call(x, positions[:7], inv_freq), "positions must be"),
        (lambda: call(x, positions, inv_freq.float()), "float64"),
        (lambda: call(x, positions, inv_freq.cpu()), "inv_freq must be a CUDA tensor"),
        (lambda: call(x, positions, inv_freq[:7]), "multiple of 8"),
        (lambda: call(x, positions, inv_freq[:0]), "multiple of 8"),
        (lambda: call(x, positions, inv_freq.repeat(2)), "multiple of 8"),
        (lambda: call(x, positions, inv_freq, False, float("nan")), "factor must be finite"),
        (lambda: call(torch.zeros(1, 2, 8, 65, dtype=torch.float16, device="cuda")[..., 1:],
                      positions, inv_freq), "start on 16 bytes"),
        (lambda: call(x.transpose(2, 3).contiguous().transpose(2, 3), positions, inv_freq),
         "start on 16 bytes"),
        (lambda: flashattn_cuda.rope_backward(x.float(), positions, inv_freq), "grad must be fp16"),
    ]
    for make, message in bad:
        with pytest.raises(RuntimeError, match=message):
            make()


# ---- frequencies (CPU) ---------------------------------------------------------


def test_frequencies_follow_their_formulas():
    w, factor = flashattn_cuda.rope_frequencies(64)
    assert w.dtype == torch.float64 and w.shape == (32,) and factor == 1.0
    assert w[0] == 1.0 and math.isclose(w[-1], 10000.0 ** (-62 / 64))
    linear, factor = flashattn_cuda.rope_frequencies(64, scaling="linear", stretch=4.0)
    assert torch.equal(linear, w / 4) and factor == 1.0
    base, factor = flashattn_cuda.rope_frequencies(64, scaling="base", stretch=4.0)
    assert base[0] == 1.0 and math.isclose(base[-1], w[-1] / 4, rel_tol=1e-12) and factor == 1.0
    parts, factor = flashattn_cuda.rope_frequencies(128, scaling="parts", stretch=8.0,
                                                    trained_length=4096)
    plain, _ = flashattn_cuda.rope_frequencies(128)
    turns = 4096 * plain / (2 * math.pi)
    ratio = parts / plain
    assert torch.allclose(ratio[turns > 40], torch.ones(()).double())
    assert torch.allclose(ratio[turns < 0.8], torch.full((), 1 / 8).double())
    assert (ratio[1:] <= ratio[:-1] + 1e-12).all()
    assert math.isclose(factor, 0.1 * math.log(8) + 1)


@pytest.mark.parametrize("kwargs,message", [
    (dict(rotary_dim=24), "multiple of 16"), (dict(rotary_dim=0), "multiple of 16"),
    (dict(rotary_dim=64, base=1.0), "base"), (dict(rotary_dim=64, base=float("inf")), "base"),
    (dict(rotary_dim=64, scaling="other"), "scaling"),
    (dict(rotary_dim=64, scaling="linear", stretch=0.5), "stretch"),
    (dict(rotary_dim=64, scaling="parts", stretch=2.0), "trained_length"),
    (dict(rotary_dim=64, scaling="parts", trained_length=10, fast_turns=1.0), "fast_turns"),
])
def test_frequencies_refuse(kwargs, message):
    with pytest.raises(ValueError, match=message):
        flashattn_cuda.rope_frequencies(**kwargs)
