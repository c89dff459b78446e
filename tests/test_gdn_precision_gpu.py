"""How precise the chunked delta rule and the log probabilities are on the GPU."""
import pytest

import gdn_chunks as G

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def env():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cwen_amd import gpu
    ctx = gpu.Context(0)
    yield gpu, ctx
    torch.cuda.synchronize()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def borders(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


# Sequences and heads for launches of two, four and eight (f32: four) waves a workgroup.
WIDTHS = [([70, 33, 1, 257], 2, 6, 128), ([70, 33, 1, 257], 1, 3, 64), ([33, 64, 5, 97, 1], 8, 16, 128),
          ([40, 31, 32, 1, 0, 65, 96, 7, 64, 33], 8, 16, 128), ([40, 31, 32, 1, 0, 65, 96, 7, 64, 33], 7, 28, 64)]


def prompt(env, lens, nkh, nvh, D, tx, to, seed):
    """One call on sequences that each go on behind their slot: inputs, the states before, outputs, the states behind."""
    gpu, ctx = env
    g, T = gen(seed), sum(lens)
    pool = gpu.GdnPool.empty(1, len(lens), nkh, nvh, D)
    pool.state.normal_(generator=g).mul_(0.2)
    before = pool.state[0].clone()
    q, k, v = (randn(g, T, n, D, dtype=tx) for n in (nkh, nkh, nvh))
    a, b = -torch.exp(1.5 * randn(g, T, nvh) - 3), torch.sigmoid(randn(g, T, nvh))
    o, slots = torch.empty(T, nvh, D, device="cuda", dtype=to), ints(list(range(len(lens))))
    gpu.gdn_prompt(ctx, pool, 0, q, k, v, a, b, o, ints(borders(lens)), slots, slots)
    assert pool.take_status(ctx) == 0
    return (q, k, v, a, b), before, o, pool.state[0]


@pytest.mark.parametrize("tx", [F32, F16, BF16])
def test_every_operand_keeps_both_halves(env, tx):
    """Outputs and states within bounds that a single f16 value in any operand exceeds by far."""
    for i, (lens, nkh, nvh, D) in enumerate(WIDTHS + [([1025], 1, 2, 128), ([700, 3], 2, 2, 64)]):
        inputs, before, o, after = prompt(env, lens, nkh, nvh, D, tx, F32, 40 + i)
        inputs, before, o, after = [t.cpu() for t in inputs], before.cpu(), o.cpu(), after.cpu()
        at = 0
        for j, n in enumerate(lens):
            if n:
                want, limits = G.reference(*(t[at:at + n] for t in inputs), before[j])
                worst = G.share((o[at:at + n], after[j]), want, limits)
                print(tx, lens[j], nvh, D, "share of the bounds: outputs %.3f, state %.3f" % worst, flush=True)
                assert max(worst) < 1, (lens, j, nvh, D, worst)
            at += n


@pytest.mark.parametrize("to", [BF16, F16])
@pytest.mark.parametrize("tx", [F32, F16, BF16])
def test_the_outputs_type_only_rounds_them(env, tx, to):
    """Outputs of 16 bits are the f32 outputs of the same call, rounded once: half a step from them (f16: from them before
    their own rounding, 2^-24 more; 2^-25 for subnormals), and the states are the same bits."""
    for i, (lens, nkh, nvh, D) in enumerate(WIDTHS):
        _, _, o, s = prompt(env, lens, nkh, nvh, D, tx, F32, 20 + i)
        _, _, p, t = prompt(env, lens, nkh, nvh, D, tx, to, 20 + i)
        assert torch.equal(s, t), (lens, nvh, D)
        far = (p.double() - o.double()).abs() - o.double().abs() * (torch.finfo(to).eps / 2 + 2.0 ** -24)
        assert far.max() <= (2.0 ** -25 if to == F16 else 0), (lens, nvh, D, far.max(), int((far > 0).sum()), "of", far.numel())
