"""How precise the chunked delta rule and the log probabilities are on the GPU."""
import pytest

import gdn_chunks as G
import gdn_ref as R

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


@pytest.mark.parametrize("tx", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["2", "1.5", "one", "spread"])
def test_betas_above_one(env, kind, tx):
    """Betas to 2, where the state grows by two values a row: prompts in every launch width, and steps."""
    gpu, ctx = env
    for n, S, H, D in ((16 * G.N + 20, 1, 2, 128), (16 * G.N + 20, 3, 20, 64), (16 * G.N + 20, 40, 2, 128), (16 * G.N + 20, 70, 2, 128),
                       (10 * G.N, 70, 2, 64)):
        x, wider = G.long_betas(kind, n, H, D, n + D, tx)
        want, limits = G.reference(*x, **wider)
        _, _, M = R.rule(*x[:3], x[3].double(), x[4].double(), x[5])
        q, k, v, a, b = (t.cuda().repeat(S, *[1] * (t.dim() - 1)) for t in x[:5])
        cu, slots = ints(borders([n] * S)), ints(list(range(S)))
        for call in (gpu.gdn_prompt, gpu.gdn_step):
            pool = gpu.GdnPool.empty(1, S, H, H, D)
            pool.state[0] = x[5].cuda()
            o = torch.empty(S * n, H, D, device="cuda")
            call(ctx, pool, 0, q, k, v, a, b, o, cu, slots, slots)
            assert pool.take_status(ctx) == 0
            for i in range(S):
                got = o[i * n:(i + 1) * n], pool.state[0, i]
                assert i == 0 or all(torch.equal(x, y) for x, y in zip(got, first)), (call.__name__, i)
                first = got
            got = [t.cpu() for t in first]
            worst = G.share(got, want, limits)
            print(call.__name__, kind, tx, n, H, D, worst, flush=True)
            if call is gpu.gdn_prompt:
                assert max(worst) < 1, (n, D, worst)
            else:
                eo, es = R.step_bounds(n, D, M, F32)
                assert bool(((got[0] - want[0]).abs() <= eo).all()) and bool(((got[1] - want[1]).abs() <= es[:, None]).all()), (n, D)


@pytest.mark.parametrize("tx", [F32, F16, BF16])
def test_small_betas(env, tx):
    """A prompt whose state is far below its values keeps as many bits of the state, in every launch width."""
    gpu, ctx = env
    for n, S, H, D in ((200, 1, 6, 128), (333, 2, 6, 64), (200, 16, 6, 128), (200, 24, 6, 128), (161, 24, 6, 64)):
        x = G.small_betas(n, H, D, n + D, tx)
        want, limits = G.reference(*x)
        q, k, v, a, b = (t.cuda().repeat(S, *[1] * (t.dim() - 1)) for t in x[:5])
        pool = gpu.GdnPool.empty(1, S, H, H, D)
        o, slots = torch.empty(S * n, H, D, device="cuda"), ints(list(range(S)))
        gpu.gdn_prompt(ctx, pool, 0, q, k, v, a, b, o, ints(borders([n] * S)), None, slots)
        for i in range(0, S, max(1, S - 1)):
            worst = G.share((o[i * n:(i + 1) * n].cpu(), pool.state[0, i].cpu()), want, limits)
            print(tx, n, S, D, worst, flush=True)
            assert max(worst) < 1, (n, S, D, worst)


def test_silu_of_the_convolution(env):
    """Taps that pass the input on: silu alone, to the stated share of itself."""
    gpu, ctx = env
    pool = gpu.GdnPool(1, 2, 64, hist=torch.zeros(1, 1, 256, 3, device="cuda"))
    kw = torch.zeros(256, 4, device="cuda")
    kw[:, 3] = 1
    span = torch.linspace(-86.5, 90, 39000, device="cuda"), torch.logspace(-30, 4, 1000, device="cuda"), -torch.logspace(-30, 1, 960, device="cuda")
    x = torch.cat(span).view(160, 256)
    low = torch.linspace(-3e38, -87.5, 256, device="cuda")[None]
    y = torch.empty(161, 256, device="cuda")
    gpu.gdn_conv(ctx, pool, 0, torch.cat([x, low]), kw, y, ints([0, 161]))
    z = x.double()
    want = z * torch.sigmoid(z)
    # the exponent's product 1.22 |z|, exp2 2, the sum 1, the reciprocal 2, the product 1, each 2^-24
    assert ((y[:160].double() - want).abs() <= (6 + 2 * z.abs()) * 2.0 ** -24 * want.abs() + 2.0 ** -126).all()
    assert y[160].abs().max() < 2e-36
