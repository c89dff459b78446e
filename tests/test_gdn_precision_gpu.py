"""How precise the chunked delta rule and the log probabilities are on the GPU."""
import math

import pytest

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
          ([40, 31, 32, 1, 0, 65, 96, 7, 64, 33], 8, 48, 128)]


def prompt(env, lens, nkh, nvh, D, tx, to, seed):
    gpu, ctx = env
    g, T = gen(seed), sum(lens)
    pool = gpu.GdnPool.empty(1, len(lens), nkh, nvh, D)
    pool.state.normal_(generator=g).mul_(0.2)
    q, k, v = (randn(g, T, n, D, dtype=tx) for n in (nkh, nkh, nvh))
    a, b = -torch.exp(2 * randn(g, T, nvh) - 2), torch.sigmoid(randn(g, T, nvh))
    o, slots = torch.empty(T, nvh, D, device="cuda", dtype=to), ints(list(range(len(lens))))
    gpu.gdn_prompt(ctx, pool, 0, q, k, v, a, b, o, ints(borders(lens)), slots, slots)
    return o, pool.state


@pytest.mark.parametrize("to", [BF16, F16])
@pytest.mark.parametrize("tx", [F32, F16, BF16])
def test_the_outputs_type_only_rounds_them(env, tx, to):
    """Outputs of 16 bits are the f32 outputs of the same call, rounded once: half a step from them (f16: from them before
    their own rounding, 2^-24 more; 2^-25 for subnormals), and the states are the same bits."""
    for i, (lens, nkh, nvh, D) in enumerate(WIDTHS):
        o, s = prompt(env, lens, nkh, nvh, D, tx, F32, 20 + i)
        p, t = prompt(env, lens, nkh, nvh, D, tx, to, 20 + i)
        assert torch.equal(s, t), (lens, nvh, D)
        far = (p.double() - o.double()).abs() - o.double().abs() * (torch.finfo(to).eps / 2 + 2.0 ** -24)
        assert far.max() <= (2.0 ** -25 if to == F16 else 0), (lens, nvh, D, far.max(), int((far > 0).sum()), "of", far.numel())
