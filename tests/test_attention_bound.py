"""What the checks of fp32 attention would let pass, on the CPU: the sound form does, one with a product of parts left out or an operand in half
the bits does not."""
import pytest
import torch

import attention_bound as A

SHAPES = [(64, 64), (197, 64), (300, 128), (100, 8)]


def _inputs(n, d):
    gen = torch.Generator().manual_seed(n + d)
    return [torch.randn(n, d, generator=gen) for _ in range(3)]


def _passes(n, d, **kw):
    q, k, v = _inputs(n, d)
    want, bound = A.attention(*(t[None, :, None] for t in (q, k, v)))
    got = A.emulated(q, k, v, d ** -0.5, **kw)
    try:
        A.check(got[None, :, None], want, bound)
    except AssertionError:
        return False
    return A.rms(got, want[0, :, 0]) <= A.RMS


@pytest.mark.parametrize("n,d", SHAPES)
def test_the_sound_form_passes(n, d):
    assert _passes(n, d)
    assert A.rms(A.emulated(*_inputs(n, d), d ** -0.5), A.attention(*(t[None, :, None] for t in _inputs(n, d)))[0][0, :, 0]) < A.RMS / 8


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("term", A.TERMS)
@pytest.mark.parametrize("which", ["terms_qk", "terms_pv"])
def test_a_missing_product_does_not(n, d, which, term):
    assert not _passes(n, d, **{which: [t for t in A.TERMS if t != term]})


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("operand", "qkvp")
def test_an_operand_in_half_the_bits_does_not(n, d, operand):
    assert not _passes(n, d, halved=operand)


def test_parts_are_the_number():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(100000, generator=gen) * torch.exp2(torch.randint(-80, 120, (100000,), generator=gen).float())
    x = torch.cat([x, torch.tensor([0.0, torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max])])
    assert torch.equal(sum(p.double() for p in A.parts(x)), x.double())
