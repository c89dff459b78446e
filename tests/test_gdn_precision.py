"""The bounds of the chunked delta rule reject an operand that has lost its low half: a model of the chunks' products on the CPU."""
import pytest

import gdn_chunks as G

SIZES = [(1, 1, 2, 64), (33, 1, 2, 128), (100, 2, 4, 64), (257, 1, 3, 128), (600, 1, 2, 64)]


@pytest.fixture(scope="module", params=SIZES, ids=lambda s: "x".join(map(str, s)))
def prompt(request):
    x = G.inputs(*request.param, seed=request.param[0])
    return (request.param[0], x, *G.reference(*x))


def test_two_halves_are_well_within_the_bounds(prompt):
    n, x, want, limits = prompt
    o, s = G.share(G.chunks(*x), want, limits)
    assert o < 0.2 and s < 0.2, (o, s)


@pytest.mark.parametrize("name", G.OPERANDS)
def test_a_single_half_is_far_outside(prompt, name):
    """In the outputs (the rows before the state enter those of later chunks only), and in the state where it enters that."""
    n, x, want, limits = prompt
    o, s = G.share(G.chunks(*x, single=(name,)), want, limits)
    if name != "y" or n > G.N:
        assert o > 3, o
    if name in ("r", "T", "y", "K"):
        assert s > 3, s


@pytest.mark.parametrize("kind", ["2", "1.5", "one", "spread"])
def test_betas_above_one(kind):
    """The model's operands stay below f16's largest value, and the errors within the wider bounds."""
    for n, H, D in ((16 * G.N + 20, 2, 64), (75, 1, 128)):
        x, wider = G.long_betas(kind, n, H, D, n)
        want, limits = G.reference(*x, **wider)
        o, s = G.share(G.chunks(*x), want, limits)
        assert o < 0.5 and s < 0.5, (o, s)


def test_small_betas():
    """A state of small betas alone keeps the bits that others do; without a scale it would not."""
    x = G.small_betas(200, 6, 64, 1)
    want, limits = G.reference(*x)
    o, s = G.share(G.chunks(*x), want, limits)
    assert o < 0.2 and s < 0.2, (o, s)
    o, s = G.share(G.chunks(*x, scaled=False), want, limits)
    assert o > 3 and s > 3, (o, s)
