"""The serving operators of the GatedDeltaNet layers and the log probabilities on
the GPU against plain 64-bit references, and a request through all of them.  The
bounds are those of gdn_ref.py, derived from the roundings that the kernels make."""
import math
import random

import pytest

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


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def close(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    both = (torch.isnan(got) & torch.isnan(want)) | (got == want)
    off = torch.where(both, torch.zeros_like(want), (got - want).abs())
    bad = ~(both | (off <= bound))
    assert not bool(bad.any()), (what, int(bad.sum()), "of", bad.numel(), "first", bad.nonzero()[0].tolist(),
                                 got[bad][:4].tolist(), want[bad][:4].tolist(), bound.expand_as(want)[bad][:4].tolist())


def borders(lens, first=0):
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


# ---------------------------------------------------------------- convolution
LENS = [[1], [3, 1, 0, 2], [33, 5, 64, 31, 32, 0, 1], [200], [2, 96, 95, 97]]


@pytest.mark.parametrize("tx,ty", [(F32, F32), (BF16, BF16), (F16, F32), (F32, F16), (BF16, F16), (F16, BF16)])
def test_conv_values(env, tx, ty):
    gpu, ctx = env
    for i, lens in enumerate(LENS):
        for nkh, nvh, D in ((1, 3, 64), (16, 48, 128)):
            g, S, first, extra = gen(10 * i + nkh), len(lens), 3 * (i % 2), 2
            pool = gpu.GdnPool.empty(2, S + 3, nkh, nvh, D)
            C = pool.channels
            pool.hist.normal_(generator=g)
            before = pool.hist.clone()
            T = first + sum(lens) + extra
            x, kw = randn(g, T, C + 16, dtype=tx)[:, 8:-8], randn(g, C, 4) * 0.5
            y = torch.full((T, C + 8), 7.0, device="cuda", dtype=ty)
            r = random.Random(i)
            slots = r.sample(range(S + 3), S)
            src = [s if j % 3 else -1 for j, s in enumerate(slots)]
            count = [max(0, n - (j % 2)) for j, n in enumerate(lens)] if i % 2 else None
            gpu.gdn_conv(ctx, pool, 1, x, kw, y[:, :C], ints(borders(lens, first)), ints(src), ints(slots), None if count is None else ints(count))
            assert pool.take_status(ctx) == 0
            want_y, want_h = torch.full((T, C), 7.0, dtype=torch.float64), before.double().cpu()
            bound = torch.zeros(T, C, dtype=torch.float64)
            xc, kc = x.cpu(), kw.cpu()
            at = first
            for j, n in enumerate(lens):
                m = n if count is None else count[j]
                h = before[1, src[j]].cpu() if src[j] >= 0 else torch.zeros(C, 3)
                yy, hh, b = R.conv(xc[at:at + m], h, kc)
                want_y[at:at + m], want_h[1, slots[j]], bound[at:at + m] = yy, hh, R.rounded(yy, b, ty)
                at += n
            close(y[:, :C], want_y, bound, ("conv", lens, tx, ty))
            assert bool((y[:, C:] == 7).all())
            assert torch.equal(pool.hist.double().cpu(), want_h)           # inputs are kept as they are; other slots and layers untouched


def test_conv_in_pieces(env):
    """Rows in one call, in pieces and one by one: the same bits, the history carried by the slot; y None moves it alone."""
    gpu, ctx = env
    g, n = gen(3), 71
    whole, parts = gpu.GdnPool.empty(1, 2, 2, 4, 64), gpu.GdnPool.empty(1, 2, 2, 4, 64)
    x, kw = randn(g, n, whole.channels, dtype=BF16), randn(g, whole.channels, 4)
    y, z = (torch.empty(n, whole.channels, device="cuda", dtype=F32) for _ in range(2))
    gpu.gdn_conv(ctx, whole, 0, x, kw, y, ints([0, n]), None, ints([1]))
    at = 0
    for m in (1, 1, 2, 33, 0, 5, 29):
        gpu.gdn_conv(ctx, parts, 0, x[at:at + m], kw, z[at:at + m], ints([0, m]), ints([0]), ints([0]))
        at += m
    assert at == n and torch.equal(y, z) and torch.equal(whole.hist[0, 1], parts.hist[0, 0])
    gpu.gdn_conv(ctx, parts, 0, x, kw, None, ints([0, n]), None, ints([1]))
    assert torch.equal(parts.hist[0, 1], whole.hist[0, 1])
    for m in (0, 1, 2):                                                     # a fork with few rows keeps the older inputs
        gpu.gdn_conv(ctx, parts, 0, x[:m], kw, None, ints([0, m]), ints([1]), ints([0]))
        assert torch.equal(parts.hist[0, 0], torch.cat([parts.hist[0, 1].t(), x[:m].float()])[m:].t())


# ---------------------------------------------------------------- delta rule
def rule_inputs(g, T, nkh, nvh, D, dtype, raw=True, pad=0):
    x = randn(g, T, (2 * nkh + nvh) * D + pad, dtype=dtype)
    q, k, v = x[:, :nkh * D].unflatten(1, (nkh, D)), x[:, nkh * D:2 * nkh * D].unflatten(1, (nkh, D)), x[:, 2 * nkh * D:(2 * nkh + nvh) * D].unflatten(1, (nvh, D))
    a, b = randn(g, T, nvh + 3)[:, :nvh], randn(g, T, nvh + 3)[:, :nvh]
    if raw:
        return q, k, v, a, b, -torch.exp(randn(g, nvh)), 2 * randn(g, nvh) - 3
    return q, k, v, -torch.exp(2 * a - 2), torch.sigmoid(b), None, None


def check_rule(env, name, lens, nkh, nvh, D, tx, to, seed, raw=True, key_head="mod", count=None, first=0, change=None, fork=False, emit=True):
    """One call against the reference; returns what it ran on."""
    gpu, ctx = env
    g, S = gen(seed), len(lens)
    pool = gpu.GdnPool.empty(2, S + 3, nkh, nvh, D, key_head)
    pool.state.normal_(generator=g).mul_(0.2)
    T = first + sum(lens) + 2
    q, k, v, a, b, A, dt = rule_inputs(g, T, nkh, nvh, D, tx, raw, 8)
    if change:
        q, k, v, a, b = change(q, k, v, a, b)
    before = pool.state.clone()
    o = torch.full((T, nvh, D), 7.0, device="cuda", dtype=to)
    r = random.Random(seed)
    slots = r.sample(range(S + 3), S)
    src = [slots[j] if j % 3 else -1 for j in range(S)]
    if fork:
        free = [s for s in range(S + 3) if s not in slots]
        src = [free[j % len(free)] for j in range(S)]
    call = gpu.gdn_step if name == "step" else gpu.gdn_prompt
    call(ctx, pool, 1, q, k, v, a, b, o if emit else None, ints(borders(lens, first)), ints(src), ints(slots), A=A, dt=dt,
         count=None if count is None else ints(count))
    assert pool.take_status(ctx) == 0
    cpu = lambda t: None if t is None else t.cpu()
    lg, beta = R.gates(cpu(a), cpu(b), cpu(A), cpu(dt))
    want_o, want_s = torch.full((T, nvh, D), 7.0, dtype=torch.float64), before.double().cpu()
    bo, bs = torch.zeros_like(want_o), torch.zeros_like(want_s)
    at = first
    full = F32 in (tx, to)
    for j, n in enumerate(lens):
        m = n if count is None else count[j]
        s0 = before[1, src[j]].cpu() if src[j] >= 0 else None
        oo, ss, M = R.rule(q[at:at + m].cpu(), k[at:at + m].cpu(), v[at:at + m].cpu(), lg[at:at + m], beta[at:at + m], s0, key_head)
        eo, es = R.step_bounds(m, D, M, to) if name == "step" else R.prompt_bounds(m, D, M, to, full)
        want_s[1, slots[j]] = ss
        bs[1, slots[j]] = es[:, None, :] + 2.0 ** -149
        if emit:
            want_o[at:at + m] = oo
            bo[at:at + m] = R.rounded(oo, eo[None].expand_as(oo), to)
        at += n
    close(pool.state, want_s, bs, (name, "state", lens, D, tx, to))
    close(o, want_o, bo, (name, "o", lens, D, tx, to))
    return pool, q, k, v, a, b, A, dt, o


STEP_LENS = [[1], [1, 1, 1], [5, 0, 16, 1, 2], [40]]


@pytest.mark.parametrize("tx,to", [(F32, F32), (BF16, BF16), (F16, F16), (F32, F16), (F16, BF16), (BF16, F32)])
def test_step_values(env, tx, to):
    for i, lens in enumerate(STEP_LENS):
        check_rule(env, "step", lens, 16, 48, 128, tx, to, 50 + i, raw=i % 2 == 0)
        check_rule(env, "step", lens, 1, 3, 64, tx, to, 60 + i, key_head="group", first=i, fork=i == 2)
        check_rule(env, "step", lens, 4, 8, 64, tx, to, 70 + i, key_head="group", count=[n // 2 for n in lens], emit=i != 1)


PROMPT_LENS = [[1], [31, 32, 33, 0, 64, 2], [100], [257, 5], [7, 129, 65, 96, 1, 1, 40]]


@pytest.mark.parametrize("tx,to", [(F32, F32), (BF16, BF16), (F16, F16), (F32, F16), (F16, BF16), (BF16, F32), (F32, BF16), (F16, F32), (BF16, F16)])
def test_prompt_values(env, tx, to):
    for i, lens in enumerate(PROMPT_LENS):
        check_rule(env, "prompt", lens, 2, 6, 128, tx, to, 150 + i, raw=i % 2 == 0)
        check_rule(env, "prompt", lens, 1, 3, 64, tx, to, 160 + i, key_head="group", first=i, fork=i == 2)
        check_rule(env, "prompt", lens, 4, 8, 64, tx, to, 170 + i, key_head="group", count=[n - n // 3 for n in lens], emit=i != 1)
        check_rule(env, "prompt", lens, 5, 5, 128, tx, to, 180 + i)


def _decays(values):
    def change(q, k, v, a, b):
        pick = torch.tensor(values, device="cuda")
        a.copy_(pick[torch.arange(a.numel(), device="cuda").view(a.shape) * 7 % len(values)])
        return q, k, v, a, b
    return change


def _betas(value):
    def change(q, k, v, a, b):
        b.fill_(value)
        return q, k, v, a, b
    return change


def _keys(kind):
    def change(q, k, v, a, b):
        if kind == "same":                  # one key for all rows: the solve's hardest
            k.copy_(k[:1].clone().expand_as(k))
        elif kind == "zero":
            k[::3] = 0
            q[::5] = 0
        elif kind == "alternate":
            k.copy_(k[:1].clone() * torch.where(torch.arange(k.shape[0], device="cuda") % 2 == 0, 1.0, -1.0).to(k.dtype)[:, None, None])
        elif kind == "tiny":                # lengths far below the 1e-6 under the root
            k.mul_(2.0 ** -14)
            q.mul_(2.0 ** -12)
        elif kind == "long":                # f16's upper range
            k.mul_(2.0 ** 11)
            q.mul_(2.0 ** 10)
        elif kind == "one":                 # all of a key's length in one dim
            k.zero_()
            k[:, :, 5] = 3
        return q, k, v, a, b
    return change


def _values(scale):
    def change(q, k, v, a, b):
        v.mul_(scale)
        return q, k, v, a, b
    return change


HARD = {"none": _decays([0.0]), "slow": _decays([-1e-5, 0.0, -3e-4]), "fast": _decays([-30.0, -0.5, -1e-3, -90.0]),
        "cut": _decays([-math.inf, -0.1, 0.0, -0.01, -200.0, -0.3, -5.0]), "beta0": _betas(0.0), "beta1": _betas(1.0), "same": _keys("same"),
        "zero": _keys("zero"), "alternate": _keys("alternate"), "tiny": _keys("tiny"), "long": _keys("long"), "one": _keys("one"),
        "large": _values(2.0 ** 13), "small": _values(2.0 ** -13)}


@pytest.mark.parametrize("kind", HARD)
@pytest.mark.parametrize("name", ["step", "prompt"])
def test_rule_hard_inputs(env, name, kind):
    for i, (tx, to) in enumerate(((F32, F32), (BF16, BF16), (F16, F16))):
        check_rule(env, name, [70, 33], 2, 4, (64, 128)[i % 2], tx, to, 300 + i, raw=False, change=HARD[kind])


# Sequences and heads for launches of two, four and eight (f32: four) waves a workgroup.
WIDE = [([33, 64, 5, 97, 1], 4, 12, 128), ([33, 64, 5, 97, 1], 8, 16, 128), ([40, 31, 32, 1, 0, 65, 96, 7, 64, 33], 8, 16, 128),
        ([40, 31, 32, 1, 0, 65, 96, 7, 64, 33], 8, 16, 64), ([40, 31, 32, 1, 0, 65, 96, 7, 64, 33], 28, 28, 64)]


@pytest.mark.parametrize("tx,to", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32)])
def test_prompt_of_many_heads(env, tx, to):
    for i, (lens, nkh, nvh, D) in enumerate(WIDE):
        check_rule(env, "prompt", lens, nkh, nvh, D, tx, to, 700 + i, key_head="mod" if i % 2 else "group")
        check_rule(env, "prompt", lens, nkh, nvh, D, tx, to, 710 + i, raw=False, count=[n - n // 4 for n in lens],
                   change=list(HARD.values())[i % len(HARD)])


@pytest.mark.parametrize("tx,to", [(F32, F32), (BF16, BF16), (F16, F16)])
def test_prompt_of_many_heads_with_values_that_are_not_finite(env, tx, to):
    """In one column of every head of a sequence: rows before, other columns and other sequences stay as they are."""
    gpu, ctx = env
    for i, (lens, nkh, nvh, D) in enumerate(WIDE):
        T, at, n = sum(lens), sum(lens[:3]), lens[3] if lens[3] > 70 else 0
        if not n:
            at, n = sum(lens[:6]), lens[6]
        q, k, v, a, b, _, _ = rule_inputs(gen(720 + i), T, nkh, nvh, D, tx, raw=False)
        cu, dst = ints(borders(lens, 0)), ints(list(range(len(lens))))

        def run():
            pool = gpu.GdnPool.empty(1, len(lens), nkh, nvh, D)
            o = torch.full((T, nvh, D), 7.0, device="cuda", dtype=to)
            gpu.gdn_prompt(ctx, pool, 0, q, k, v, a, b, o, cu, None, dst)
            return o, pool.state[0].clone()

        clean, state = run()
        seq = lens.index(n)
        for row, bad in ((0, math.nan), (33, math.inf), (63, -math.inf), (70, math.nan)):
            keep = v[at + row].clone()
            v[at + row, :, 9] = bad
            o, s = run()
            v[at + row] = keep
            cols, rest = [c for c in range(D) if c != 9], [r for r in range(len(lens)) if r != seq]
            tell = (lens, nvh, D, row, bad, tx)
            assert torch.equal(o[:, :, cols], clean[:, :, cols]) and torch.equal(s[:, :, :, cols], state[:, :, :, cols]), tell
            assert torch.equal(o[:at + row], clean[:at + row]) and torch.equal(o[at + n:], clean[at + n:]), tell
            assert torch.equal(s[rest], state[rest]), tell
            assert not bool(torch.isfinite(o[at + row:at + n, :, 9]).any()) and not bool(torch.isfinite(s[seq, :, :, 9]).any()), tell


def test_rule_wide_range(env):
    """Values of f32's and bf16's range, beside columns of small ones: each column by its own size."""
    def change(q, k, v, a, b):
        v.mul_(torch.logspace(-24, 24, v.shape[2], device="cuda").to(v.dtype))
        return q, k, v, a, b
    for name in ("step", "prompt"):
        check_rule(env, name, [70, 3], 2, 4, 64, F32, F32, 5, raw=False, change=change)
        check_rule(env, name, [70, 3], 2, 4, 128, BF16, BF16, 6, raw=False, change=change)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("name", ["step", "prompt"])
def test_rule_values_that_are_not_finite(env, name, bad):
    """They reach their own column, head or row, never an earlier row, another sequence or the rows of no sequence."""
    gpu, ctx = env
    for i, (tx, to, nkh, nvh, D) in enumerate(((F32, F32, 2, 4, 64), (BF16, BF16, 2, 4, 128), (F16, F16, 1, 3, 128))):
        lens, first = [75, 40], 1
        T = first + sum(lens) + 3
        call = gpu.gdn_step if name == "step" else gpu.gdn_prompt
        q, k, v, a, b, _, _ = rule_inputs(gen(500 + i), T, nkh, nvh, D, tx, raw=False)
        cu, dst = ints(borders(lens, first)), ints([0, 1])

        def run():
            pool = gpu.GdnPool.empty(1, 2, nkh, nvh, D)
            o = torch.full((T, nvh, D), 7.0, device="cuda", dtype=to)
            call(ctx, pool, 0, q, k, v, a, b, o, cu, None, dst)
            return o, pool.state[0].clone()

        for t in (q, k, v, a, b):                                # rows of no sequence hold anything
            t[0], t[-3:] = bad, math.nan
        clean, state = run()
        assert bool(torch.isfinite(clean).all()) and bool(torch.isfinite(state).all())
        for what, row in (("v", 0), ("v", 45), ("v", 31), ("k", 13), ("k", 64), ("q", 20), ("a", 33), ("b", 50), ("b", 7)):
            if what == "a" and bad == -math.inf:
                continue                                          # a decay to nothing: a number like others
            t = {"q": q, "k": k, "v": v, "a": a, "b": b}[what]
            at = first + row
            keep = t[at].clone()
            if what == "v":
                t[at, 1, 5] = bad
            elif what in "kq":
                t[at, 0, 3] = bad
            else:
                t[at, 1] = bad
            o, s = run()
            t[at] = keep
            heads = [h for h in range(nvh) if h % nkh == 0] if what in "kq" else [1]
            others = [h for h in range(nvh) if h not in heads]
            tell = (name, what, row, tx)
            assert torch.equal(o[:, others], clean[:, others]) and torch.equal(s[:, others], state[:, others]), tell
            assert torch.equal(o[:at, heads], clean[:at, heads]), tell                       # earlier rows
            assert torch.equal(o[first + 75:], clean[first + 75:]) and torch.equal(s[1], state[1]), tell
            end = first + 75
            if what == "v":
                cols = [c for c in range(D) if c != 5]
                assert torch.equal(o[:, 1, cols], clean[:, 1, cols]) and torch.equal(s[0, 1][:, cols], state[0, 1][:, cols]), tell
                assert not bool(torch.isfinite(o[at:end, 1, 5]).any()) and not bool(torch.isfinite(s[0, 1, :, 5]).any()), tell
            elif what == "q":                                     # (an infinite one: over its length, NaN)
                assert torch.equal(o[at + 1:end], clean[at + 1:end]) and torch.equal(s, state), tell
                assert not bool(torch.isfinite(o[at, heads]).any()), tell
            else:
                assert not bool(torch.isfinite(o[at:end, heads]).any()) and not bool(torch.isfinite(s[0, heads]).any()), tell


def test_step_rows_do_not_depend_on_the_call(env):
    """A block's rows are the bits of single ones, alone or among other sequences; scored rows leave the slots alone, the
    accepted counts move them."""
    gpu, ctx = env
    g = gen(4)
    lens = [9, 3, 16]
    T = sum(lens)
    pool = gpu.GdnPool.empty(1, 7, 16, 48)
    pool.state.normal_(generator=g)
    start = pool.state.clone()
    q, k, v, a, b, A, dt = rule_inputs(g, T, 16, 48, 128, BF16)
    o, one = torch.empty(T, 48, 128, device="cuda", dtype=BF16), torch.empty(T, 48, 128, device="cuda", dtype=BF16)
    cu, src = ints(borders(lens)), ints([5, 0, 2])
    gpu.gdn_step(ctx, pool, 0, q, k, v, a, b, o, cu, src, None, A=A, dt=dt)
    assert torch.equal(pool.state, start)
    gpu.gdn_step(ctx, pool, 0, q, k, v, a, b, o, cu, src, ints([-1, -1, -1]), A=A, dt=dt)
    assert torch.equal(pool.state, start)
    accepted = [4, 3, 1]
    gpu.gdn_step(ctx, pool, 0, q, k, v, a, b, None, cu, src, ints([6, 0, 3]), A=A, dt=dt, count=ints(accepted))
    moved = pool.state.clone()
    pool.state.copy_(start)
    for s, slot in enumerate((5, 0, 2)):
        for t in range(borders(lens)[s], borders(lens)[s + 1]):
            r = slice(t, t + 1)
            gpu.gdn_step(ctx, pool, 0, q[r], k[r], v[r], a[r], b[r], one[r], ints([0, 1]), ints([slot]), ints([slot]), A=A, dt=dt)
            if t - borders(lens)[s] + 1 == accepted[s]:
                assert torch.equal(pool.state[0, slot], moved[0, (6, 0, 3)[s]])
    assert torch.equal(o, one)
    assert torch.equal(moved[0, 1], start[0, 1]) and torch.equal(moved[0, 5], start[0, 5])


def test_prompt_goes_on_behind_a_prefix(env):
    """A prompt in two calls, the second behind the slot, agrees with one call within the bound; steps behind it too."""
    gpu, ctx = env
    g, n = gen(8), 150
    pool = gpu.GdnPool.empty(1, 3, 4, 8, 128)
    q, k, v, a, b, A, dt = rule_inputs(g, n, 4, 8, 128, BF16)
    o = torch.empty(n, 8, 128, device="cuda", dtype=F32)
    for call, cuts in ((gpu.gdn_prompt, (0, 37, 101, 150)), (gpu.gdn_prompt, (0, 64, 150)), (gpu.gdn_step, (0, 3, 150))):
        for x, y in zip(cuts, cuts[1:]):
            f = gpu.gdn_prompt if x == 0 else call
            f(ctx, pool, 0, q[x:y], k[x:y], v[x:y], a[x:y], b[x:y], o[x:y], ints([0, y - x]), None if x == 0 else ints([2]), ints([2]), A=A, dt=dt)
        lg, beta = R.gates(a.cpu(), b.cpu(), A.cpu(), dt.cpu())
        wo, ws, M = R.rule(q.cpu(), k.cpu(), v.cpu(), lg, beta, None)
        eo, es = R.prompt_bounds(n + 64, 128, M, F32, True)
        close(pool.state[0, 2], ws, es[:, None].expand_as(ws), "state")
        close(o, wo, R.rounded(wo, eo[None].expand_as(wo), F32), "o")


def test_forks_and_cleared_slots(env):
    gpu, ctx = env
    g = gen(9)
    pool = gpu.GdnPool.empty(1, 6, 1, 3, 64)
    pool.state.normal_(generator=g)
    pool.hist.normal_(generator=g)
    s0, h0 = pool.state.clone(), pool.hist.clone()
    q, k, v, a, b, A, dt = rule_inputs(g, 4, 1, 3, 64, F32)
    x, kw = randn(g, 4, pool.channels), randn(g, pool.channels, 4)
    o = torch.empty(4, 3, 64, device="cuda")
    for f in (gpu.gdn_step, gpu.gdn_prompt):
        pool.state.copy_(s0)
        f(ctx, pool, 0, q, k, v, a, b, o, ints([4, 4, 4, 4, 4]), ints([0, 0, -1, 5]), ints([1, 2, 3, 5]), A=A, dt=dt)
        assert torch.equal(pool.state[0, 1], s0[0, 0]) and torch.equal(pool.state[0, 2], s0[0, 0])
        assert not bool(pool.state[0, 3].any()) and torch.equal(pool.state[0, 4:], s0[0, 4:]) and torch.equal(pool.state[0, 0], s0[0, 0])
        f(ctx, pool, 0, q[:0], k[:0], v[:0], a[:0], b[:0], o[:0], ints([0, 0]), ints([4]), ints([0]), A=A, dt=dt)      # no rows at all
        assert torch.equal(pool.state[0, 0], s0[0, 4])
        f(ctx, pool, 0, q, k, v, a, b, o, ints([0]), A=A, dt=dt)                                                      # no sequences
    gpu.gdn_conv(ctx, pool, 0, x, kw, None, ints([0, 0, 0]), ints([4, -1]), ints([1, 2]))
    assert torch.equal(pool.hist[0, 1], h0[0, 4]) and not bool(pool.hist[0, 2].any()) and torch.equal(pool.hist[0, 3:], h0[0, 3:])
    assert pool.take_status(ctx) == 0


def test_sequences_that_are_left_out(env):
    """Bad slots and counts, and slots named twice: those sequences are left out whole, the others done."""
    gpu, ctx = env
    g, n = gen(11), 12
    pool = gpu.GdnPool.empty(1, 8, 2, 4, 64)
    q, k, v, a, b, A, dt = rule_inputs(g, 2 * n, 2, 4, 64, F32)
    x, kw = randn(g, 2 * n, pool.channels), randn(g, pool.channels, 4)
    cu = ints(borders([2] * n))
    src = [0, 8, -2, 3, 4, 5, 5, 7, 1, -1, 2 ** 31 - 1, -1]
    dst = [0, -1, -1, 8, -2, 6, 6, 1, -1, 2, -1, 4]
    count = [2, 2, 2, 2, 2, 2, 2, 2, 2, 3, 2, -1]
    # 5 and 6 end in one slot, 7 ends in what 8 reads; 8 itself only reads; the others have a bad slot or count
    left = {1, 2, 3, 4, 5, 6, 7, 9, 10, 11}
    state, hist = torch.randn(pool.state.shape, device="cuda", generator=g), torch.randn(pool.hist.shape, device="cuda", generator=g)
    for f in (gpu.gdn_step, gpu.gdn_prompt, gpu.gdn_conv):
        good = [i for i in range(n) if i not in left]
        res = []
        for seqs in (list(range(n)), good):
            pool.state.copy_(state)
            pool.hist.copy_(hist)
            s, d, c = (ints([w[i] for i in seqs]) for w in (src, dst, count))
            if len(seqs) < n:      # the good ones alone: the rows of the others between no borders, by one call each
                outs = torch.full((2 * n, 4 * 64 if f != gpu.gdn_conv else pool.channels), 7.0, device="cuda")
                for i in seqs:
                    r, one = slice(2 * i, 2 * i + 2), (ints([0, 2]), ints([src[i]]), ints([dst[i]]))
                    if f is gpu.gdn_conv:
                        f(ctx, pool, 0, x[r], kw, outs[r], *one)
                    else:
                        f(ctx, pool, 0, q[r], k[r], v[r], a[r], b[r], outs[r].view(2, 4, 64), *one, A=A, dt=dt)
                assert pool.take_status(ctx) == 0
            else:
                outs = torch.full((2 * n, 4 * 64 if f != gpu.gdn_conv else pool.channels), 7.0, device="cuda")
                if f is gpu.gdn_conv:
                    f(ctx, pool, 0, x, kw, outs, cu, s, d, count=c)
                else:
                    f(ctx, pool, 0, q, k, v, a, b, outs.view(2 * n, 4, 64), cu, s, d, A=A, dt=dt, count=c)
                assert pool.take_status(ctx) == gpu.GDN_ARG and pool.take_status(ctx) == 0
            res.append((outs, pool.state.clone(), pool.hist.clone()))
        for one, other in zip(*res):
            assert torch.equal(one, other), f.__name__


def test_refusals_of_the_python_layer(env):
    gpu, ctx = env
    pool = gpu.GdnPool.empty(1, 2, 2, 4, 64)
    q, k, v, a, b, A, dt = rule_inputs(gen(1), 3, 2, 4, 64, F16)
    o, cu = torch.empty(3, 4, 64, device="cuda"), ints([0, 3])
    ok = dict(q=q, k=k, v=v, a=a, b=b, o=o, cu=cu, A=A, dt=dt)
    for f in (gpu.gdn_step, gpu.gdn_prompt):
        f(ctx, pool, 0, **ok)
        for bad in (dict(q=q[:, :1]), dict(k=k[:2]), dict(v=v.float()), dict(a=a.half()), dict(a=a[:, :3]), dict(o=o[:, :, :32]), dict(A=None),
                    dict(dt=dt[:3]), dict(cu=cu.long()), dict(cu=ints([])), dict(src=ints([0, 1])), dict(dst=torch.zeros(1)), dict(b=b.contiguous()),
                    dict(q=q.cpu()), dict(q=q.double(), k=k.double(), v=v.double()), dict(count=ints([1, 1])), dict(q=q.transpose(1, 2))):
            with pytest.raises(ValueError):
                f(ctx, pool, 0, **{**ok, **bad})
        with pytest.raises(gpu.CwenError):
            f(ctx, pool, 1, **ok)
    for bad in (dict(state=None, hist=None), dict(state=pool.state[:, :, :2], hist=None), dict(state=pool.state.half(), hist=None),
                dict(state=pool.state, hist=pool.hist[:, :1])):
        with pytest.raises(ValueError):
            gpu.GdnPool(2, 4, 64, **bad)
    only = gpu.GdnPool(2, 4, 64, pool.state)
    with pytest.raises(gpu.CwenError):
        gpu.gdn_conv(ctx, only, 0, torch.zeros(1, only.channels, device="cuda"), torch.zeros(only.channels, 4, device="cuda"), None, ints([0, 1]))
    x = torch.zeros(2, 9, device="cuda")
    for bad in (dict(tokens=ints([1, 2], torch.int64)), dict(lse=torch.zeros(3, device="cuda")), dict(top_ids=ints([[1], [2], [3]])),
                dict(top_ids=ints([[1, 1], [2, 2]]), top_logprobs=torch.zeros(2, 3, device="cuda")), dict(rank=torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            gpu.logprobs(ctx, x, **bad)
    with pytest.raises(gpu.CwenError):
        gpu.logprobs(ctx, x, logprob=torch.zeros(2, device="cuda"))


# ---------------------------------------------------------------- log probabilities
def check_logprobs(env, x, tokens, top, what):
    gpu, ctx = env
    rows, V = x.shape
    f = lambda *s: torch.full(s, 7.0, device="cuda")
    i = lambda *s: torch.full(s, 7, device="cuda", dtype=torch.int32)
    lp, H, lse, rank, ids, tlp = f(rows), f(rows), f(rows), i(rows), i(rows, top), f(rows, top)
    tok = None if tokens is None else ints(tokens)
    gpu.logprobs(ctx, x, tok, lp if tokens else None, rank if tokens else None, H, lse, ids, tlp)
    wlp, wrank, wH, wlse, wids, wtlp = R.logprobs(x.cpu(), tokens, top)
    per = V // 256 + 32
    if tokens:
        close(lp, wlp, R.logprobs_bound(V, per, wlp), (what, "logprob"))
        assert torch.equal(rank.cpu(), wrank), (what, "rank", rank.tolist()[:8], wrank.tolist()[:8])
    close(H, wH, R.logprobs_bound(V, per, wH), (what, "entropy"))
    close(lse, wlse, R.logprobs_bound(V, per, wlse), (what, "lse"))
    assert torch.equal(ids.cpu(), wids), (what, "ids", ids[0].tolist(), wids[0].tolist())
    close(tlp, wtlp, R.logprobs_bound(V, per, wtlp), (what, "top"))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_logprobs_values(env, dtype):
    g = gen(21)
    for V in (1, 2, 63, 64, 65, 257, 1000, 4095, 4099):
        for rows, top, gap in ((1, 1, 0), (3, 5, 1), (5, 64, 3)):
            x = (randn(g, rows, V + gap) * 4).to(dtype)[:, :V]
            check_logprobs(env, x, [(7 * r) % V for r in range(rows)], top, (V, rows, top, dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_logprobs_large(env, dtype):
    g = gen(22)
    for rows, V, top in ((2, 248320, 20), (1, 131073, 64), (300, 8200, 3), (1500, 257, 2)):
        x = (randn(g, rows, V) * 3).to(dtype)
        hot = torch.randint(0, V, (rows,), device="cuda", generator=g)
        x[torch.arange(rows), hot] += 9
        few = x[:4]
        check_logprobs(env, few, hot[:4].tolist(), top, (V, dtype))
        if rows > 4:                                       # all rows at once against the few: sums split otherwise
            gpu, ctx = env
            lp, ids = torch.empty(rows, device="cuda"), torch.empty(rows, top, device="cuda", dtype=torch.int32)
            gpu.logprobs(ctx, x, hot.int(), lp, top_ids=ids)
            z = torch.log_softmax(x.double(), 1)
            close(lp, z[torch.arange(rows), hot], R.logprobs_bound(V, V // 256 + 32, z[torch.arange(rows), hot]).cpu(), "rows")
            want = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
            assert torch.equal(ids.long(), want)


def test_logprobs_orders(env):
    """Ties, sorted and constant rows, masks: the queue's hardest inputs."""
    V = 9000
    up = torch.arange(V, device="cuda").float() / 100
    rows = {"up": up, "down": -up, "same": torch.zeros(V, device="cuda"), "steps": torch.floor(up), "zeros": torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0),
            "lowest": torch.full((V,), torch.finfo(F32).min, device="cuda"), "few": torch.full((V,), -math.inf, device="cuda"),
            "none": torch.full((V,), -math.inf, device="cuda"), "high": torch.full((V,), 3e38, device="cuda"), "wide": up * 1e35}
    rows["few"][[8999, 17, 4100]] = torch.tensor([1.0, 1.0, -3.0], device="cuda")
    rows["lowest"][77] = 2.0
    for name, x in rows.items():
        for off in (0, 1):
            check_logprobs(env, x[None, off:], [V // 2], 64, name)
    check_logprobs(env, torch.stack(list(rows.values())), [0, 1, 8999, 4500, 7, 77, 17, 5, 6, 8998], 20, "all")
    low = torch.full((2, 5000), torch.finfo(F16).min, device="cuda", dtype=F16)
    check_logprobs(env, low, [3, 4999], 64, "f16 lowest")


def test_logprobs_bad_values(env):
    g = gen(23)
    x = randn(g, 6, 5000) * 3
    x[0, 100] = math.nan
    x[1, 4999] = math.inf
    x[2, :] = math.nan
    x[3, 0], x[3, 1] = math.nan, math.inf
    x[4, 7] = -math.inf
    check_logprobs(env, x, [5, 6, 7, 0, 7, 4], 20, "bad values")
    check_logprobs(env, x, [100, 4999, 7, 1, -1, 5000], 64, "bad tokens")
    check_logprobs(env, x, [-2 ** 31, 2 ** 31 - 1, 7, 1, 0, 4999], 1, "bad tokens")
    check_logprobs(env, x[:, :40], None, 64, "no tokens, fewer than top")


# ---------------------------------------------------------------- together
def layer_weights(g, gpu, nkh, nvh, D, H):
    C = (2 * nkh + nvh) * D
    w = lambda *s: randn(g, *s) / math.sqrt(s[0])
    return {"in": w(H, C), "a": w(H, nvh), "b": w(H, nvh), "kw": randn(g, C, 4) * 0.4, "A": -torch.exp(randn(g, nvh)), "dt": 2 * randn(g, nvh) - 3,
            "out": w(nvh * D, H)}


def model_step(gpu, ctx, pool, ws, h, cu, src, dst, rule, count=None, emit=True, stream=None):
    """h [T, H] through the pool's layers: projections, convolution, delta rule, residual."""
    nk, D = pool.nkh * pool.dk, pool.dk
    for l, w in enumerate(ws):
        x = h @ w["in"]
        y = torch.empty_like(x, dtype=BF16)
        gpu.gdn_conv(ctx, pool, l, x, w["kw"], y, cu, src, dst, count=count, stream=stream)
        o = torch.zeros(h.shape[0], pool.nvh, D, device="cuda")
        rule(ctx, pool, l, y[:, :nk].unflatten(1, (-1, D)), y[:, nk:2 * nk].unflatten(1, (-1, D)), y[:, 2 * nk:].unflatten(1, (-1, D)),
             h @ w["a"], h @ w["b"], o, cu, src, dst, A=w["A"], dt=w["dt"], count=count, stream=stream)
        h = h + torch.tanh(o.flatten(1) @ w["out"])
    return h


def test_many_sequences(env):
    """As many as one call takes, of no, one or a few rows; more than a wave has lanes."""
    gpu, ctx = env
    for S in (65, 200, 4096):
        r = random.Random(S)
        lens = [r.choice([0, 1, 1, 2, 3]) if S == 4096 else r.choice([0, 1, 2, 31, 33, 70]) for _ in range(S)]
        for name in ("step", "prompt"):
            check_rule(env, name, lens, 1, 1, 64, BF16, F32, 800 + S, first=2)
        g, T = gen(S), sum(lens)
        pool = gpu.GdnPool.empty(1, S, 1, 1, 64)
        pool.hist.normal_(generator=g)
        before, slots = pool.hist[0].double().cpu(), r.sample(range(S), S)
        x, kw, y = randn(g, T, pool.channels), randn(g, pool.channels, 4), torch.empty(T, pool.channels, device="cuda")
        gpu.gdn_conv(ctx, pool, 0, x, kw, y, ints(borders(lens)), ints(slots), ints(slots))
        assert pool.take_status(ctx) == 0
        want, bound, hist, at = torch.empty(T, pool.channels, dtype=torch.float64), torch.empty(T, pool.channels, dtype=torch.float64), before.clone(), 0
        xc, kc = x.cpu(), kw.cpu()
        for j, n in enumerate(lens):
            want[at:at + n], hist[slots[j]], b = R.conv(xc[at:at + n], before[slots[j]], kc)
            bound[at:at + n] = R.rounded(want[at:at + n], b, F32)
            at += n
        close(y, want, bound, ("conv", S))
        assert torch.equal(pool.hist[0].double().cpu(), hist)


def test_far_rows_and_slots(env):
    """Rows and slots behind 2^31 elements: the bits of the same call on near ones."""
    gpu, ctx = env
    nkh, nvh, D, T, far = 16, 48, 128, 140, 2 ** 24 - 8
    g = gen(90)
    q, k, v, a, b, A, dt = rule_inputs(g, T, nkh, nvh, D, BF16)
    a, b = a.contiguous(), b.contiguous()
    big, out, gates = (torch.empty(T, far, device="cuda", dtype=t) for t in (BF16, BF16, F32))
    place = lambda to, at, x: to[:, at:at + x[0].numel()].copy_(x.flatten(1)).unflatten(1, x.shape[1:])
    Q, K, V = place(big, 0, q), place(big, 2048, k), place(big, 4096, v)
    far_a, far_b = place(gates, 0, a), place(gates, 64, b)
    O = out[:, :nvh * D].unflatten(1, (nvh, D))
    cu = ints([0, T - 3, T])
    near, wide = gpu.GdnPool.empty(1, 2, nkh, nvh, D), gpu.GdnPool.empty(2, 1400, nkh, nvh, D)
    assert (T - 1) * far > 2 ** 31 and 2799 * nvh * D * D > 2 ** 31
    for call in (gpu.gdn_prompt, gpu.gdn_step):
        near.state.normal_(generator=g)
        wide.state[1, [3, 1399]] = near.state[0]
        o = torch.empty(T, nvh, D, device="cuda", dtype=BF16)
        call(ctx, near, 0, q.contiguous(), k.contiguous(), v.contiguous(), a, b, o, cu, ints([0, 1]), ints([0, 1]), A, dt)
        call(ctx, wide, 1, Q, K, V, far_a, far_b, O, cu, ints([3, 1399]), ints([3, 1399]), A, dt)
        assert torch.equal(o, O) and torch.equal(near.state[0], wide.state[1, [3, 1399]])
    del gates
    x, kw = big[:, :near.channels], randn(g, near.channels, 4)
    y = torch.empty(T, near.channels, device="cuda", dtype=BF16)
    gpu.gdn_conv(ctx, near, 0, x.contiguous(), kw, y, cu, None, ints([0, 1]))
    gpu.gdn_conv(ctx, wide, 1, x, kw, out[:, :near.channels], cu, None, ints([3, 1399]))
    assert torch.equal(y, out[:, :near.channels]) and torch.equal(near.hist[0], wide.hist[1, [3, 1399]])
    V, tok = 100003, ints([7, 1, 100002] * 47)[:T]
    x = out[:, 64:64 + V]
    x.normal_(generator=g)
    res = []
    for z in (x, x.contiguous()):
        lp, H, ids = torch.empty(T, device="cuda"), torch.empty(T, device="cuda"), torch.empty(T, 5, device="cuda", dtype=torch.int32)
        gpu.logprobs(ctx, z, tok, lp, entropy=H, top_ids=ids)
        res.append((lp, H, ids))
    assert torch.equal(res[0][2], res[1][2])
    z = torch.log_softmax(x.double(), 1)
    for lp, H, _ in res:                                   # (sums split by the rows' alignment)
        close(lp, z[torch.arange(T, device="cuda"), tok.long()], R.logprobs_bound(V, V // 256 + 32, z[torch.arange(T, device="cuda"), tok.long()]).cpu(), "far")


def test_requests_from_prompt_to_answer(env):
    """Two layers and a head over packed requests: prompts, a fork, drafted chains scored and kept, log probabilities; the
    same tokens as one prompt give the same answers."""
    gpu, ctx = env
    g = gen(31)
    nkh, nvh, D, H, V = 2, 4, 64, 128, 1000
    ws = [layer_weights(g, gpu, nkh, nvh, D, H) for _ in range(2)]
    emb, head = randn(g, V, H), randn(g, H, V) / 4
    pool = gpu.GdnPool.empty(2, 6, nkh, nvh, D)
    prompts = [[int(t) for t in torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(n))] for n in (70, 5, 33)]
    flat = lambda seqs: emb[ints([t for s in seqs for t in s]).long()]
    h = model_step(gpu, ctx, pool, ws, flat(prompts), ints(borders([len(p) for p in prompts])), None, ints([0, 1, 2]), gpu.gdn_prompt)
    # request 0 goes on in two branches: slot 3 becomes a copy of slot 0
    none = emb[:0]
    model_step(gpu, ctx, pool, ws, none, ints([0, 0]), ints([0]), ints([3]), gpu.gdn_step)
    seqs, slots = [list(prompts[0]), list(prompts[1]), list(prompts[2]), list(prompts[0])], [0, 1, 2, 3]
    for cycle in range(3):
        drafts = [[(13 * cycle + 7 * i + j) % V for j in range(1 + (i + cycle) % 4)] for i in range(4)]
        keep = [1 + (i * cycle) % len(d) for i, d in enumerate(drafts)]
        cu = ints(borders([len(d) for d in drafts]))
        before = pool.state.clone(), pool.hist.clone()
        h = model_step(gpu, ctx, pool, ws, flat(drafts), cu, ints(slots), None, gpu.gdn_step)
        assert torch.equal(pool.state, before[0]) and torch.equal(pool.hist, before[1])
        model_step(gpu, ctx, pool, ws, flat(drafts), cu, ints(slots), ints(slots), gpu.gdn_step, count=ints(keep))
        for s, d, n in zip(seqs, drafts, keep):
            s += d[:n]
    assert pool.take_status(ctx) == 0
    last = torch.stack([h[0], h[1]])                       # any two rows of the last cycle: the head's answer
    logits = last @ head
    check_logprobs(env, logits, [5, 999], 8, "answer")
    other = gpu.GdnPool.empty(2, 6, nkh, nvh, D)
    h2 = model_step(gpu, ctx, other, ws, flat(seqs), ints(borders([len(s) for s in seqs])), None, ints([0, 1, 2, 3]), gpu.gdn_prompt)
    # the convolution's 16-bit outputs of later layers differ by a step where their inputs' sums differ in the last bits
    assert (pool.hist[0, :4] - other.hist[0, :4]).abs().max() < 1e-4
    rel = (pool.state[:, :4] - other.state[:, :4]).norm() / other.state[:, :4].norm()
    assert rel < 2.0 ** -7, rel
    assert bool(torch.isfinite(h2).all())


def test_captured_and_replayed(env):
    """A step and a prompt in one captured graph, replayed between eager work on the same pool: every replay equals the
    eager result."""
    gpu, ctx = env
    g = gen(33)
    nkh, nvh, D = 2, 4, 128
    pool = gpu.GdnPool.empty(1, 5, nkh, nvh, D)
    q, k, v, a, b, A, dt = rule_inputs(g, 90, nkh, nvh, D, BF16)
    o, o2 = (torch.zeros(90, nvh, D, device="cuda", dtype=BF16) for _ in range(2))
    x, kw, y = randn(g, 90, pool.channels), randn(g, pool.channels, 4), torch.zeros(90, pool.channels, device="cuda")
    lg, lp, ids = randn(g, 3, 20000), torch.zeros(3, device="cuda"), torch.zeros(3, 7, device="cuda", dtype=torch.int32)
    tok = ints([1, 2, 19999])
    cu, src, dst = ints([0, 50, 90]), ints([0, 1]), ints([0, 1])
    cu2, n2 = ints([0, 3, 5]), ints([2, 3])

    def work():
        gpu.gdn_conv(ctx, pool, 0, x, kw, y, cu, src, dst)
        gpu.gdn_prompt(ctx, pool, 0, q, k, v, a, b, o, cu, src, dst, A=A, dt=dt)
        gpu.gdn_step(ctx, pool, 0, q, k, v, a, b, o2, cu2, n2, n2, A=A, dt=dt)
        gpu.logprobs(ctx, lg, tok, lp, top_ids=ids)

    def reset(i):
        s = gen(100 + i)
        pool.state.normal_(generator=s).mul_(0.3)
        pool.hist.normal_(generator=s)
        lg.normal_(generator=s)
        q.normal_(generator=s)
        for t in (o, o2, y, lp, ids):
            t.zero_()

    reset(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for i in range(4):
        reset(i)
        work()
        want = [t.clone() for t in (pool.state, pool.hist, o, o2, y, lp, ids)]
        torch.cuda.synchronize()
        reset(i)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((pool.state, pool.hist, o, o2, y, lp, ids), want):
            assert torch.equal(got, w), i
    assert pool.take_status(ctx) == 0


def test_two_streams_with_one_context(env):
    """Calls on slots and scratch of their own may run side by side."""
    gpu, ctx = env
    g = gen(35)
    pools = [gpu.GdnPool.empty(1, 2, 4, 8, 128) for _ in range(2)]
    q, k, v, a, b, A, dt = rule_inputs(g, 300, 4, 8, 128, F16)
    lg = randn(g, 64, 30000)
    outs = [torch.zeros(300, 8, 128, device="cuda", dtype=F16) for _ in range(2)]
    ids = [torch.zeros(64, 9, device="cuda", dtype=torch.int32) for _ in range(2)]
    cu, dst = ints([0, 300]), ints([1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, pool, o, i in zip(streams, pools, outs, ids):
            gpu.gdn_prompt(ctx, pool, 0, q, k, v, a, b, o, cu, None, dst, A=A, dt=dt, stream=s)
            gpu.logprobs(ctx, lg, top_ids=i, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(pools[0].state, pools[1].state) and torch.equal(ids[0], ids[1])
    assert torch.equal(ids[0].long(), torch.sort(lg, dim=1, descending=True, stable=True).indices[:, :9])
