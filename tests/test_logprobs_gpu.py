"""Log probabilities on the GPU where rows are cut into parts."""
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


def run(env, x, tok, top):
    gpu, ctx = env
    rows = x.shape[0]
    f, i = (lambda *s: torch.empty(s, device="cuda")), (lambda *s: torch.empty(s, device="cuda", dtype=torch.int32))
    out = {"logprob": f(rows), "rank": i(rows), "entropy": f(rows), "lse": f(rows), "top_ids": i(rows, top), "top_logprobs": f(rows, top)}
    gpu.logprobs(ctx, x, tok, **out)
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_in_parts(env, dtype):
    """Vocabularies that are no whole number of turns, in one part and in several, aligned or not: every logit counts once (in
    the ranks).  Tokens stand at the ends of parts; logits are multiples of 1/8, so that there are ties."""
    for j, (rows, V) in enumerate(((1, 20000), (1, 50257), (3, 151936), (7, 16385), (300, 50257), (200, 32003), (385, 20001), (500, 50257))):
        for gap in (0, 3):
            g = gen(10 * j + gap)
            x = torch.randint(-40, 41, (rows, V + gap), device="cuda", generator=g).float().div(8).to(dtype)[:, gap:]
            tok = torch.randint(0, V, (rows,), device="cuda", generator=g)
            ends = torch.tensor([0, V - 1, V // 2, 4095, 4096, 8191, 8192, 12288], device="cuda")
            tok[::2] = ends[torch.arange(tok[::2].numel(), device="cuda") % 8]
            x[1::3, V - 1] = 6
            out = run(env, x, tok.int(), 20)
            z, r = torch.log_softmax(x.double(), 1), torch.arange(rows, device="cuda")
            xt, at = x[r, tok][:, None], torch.arange(V, device="cuda")[None]
            assert torch.equal(out["rank"].long(), ((x > xt) | ((x == xt) & (at < tok[:, None]))).sum(1)), (rows, V, gap)
            order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :20]
            assert torch.equal(out["top_ids"].long(), order), (rows, V, gap)
            # a thread adds up to V / 256 terms, each sum off by 2^-24; fewer than 100 roundings more; |x - m| <= 11 in the entropy's sum
            bound = 2.0 ** -24 * (V / 256 + 100)
            for name, want in (("logprob", z[r, tok]), ("lse", torch.logsumexp(x.double(), 1)), ("top_logprobs", torch.gather(z, 1, order))):
                assert (out[name].double() - want).abs().max() <= bound + 2.0 ** -23 * want.abs().max(), (rows, V, gap, name)
            H = -(torch.exp(z) * z).sum(1)
            assert (out["entropy"].double() - H).abs().max() <= 12 * bound, (rows, V, gap)


def test_one_scratch_for_every_call(env):
    """Batches of all sizes with one scratch give the bits of calls with their own."""
    gpu, ctx = env
    x = torch.randn(500, 40000, device="cuda", generator=gen(5))
    work = torch.empty(gpu.LOGPROBS_WORK_MAX, dtype=torch.uint8, device="cuda")
    for rows in (500, 1, 37, 384, 385, 2, 200):
        got = [[torch.empty(rows, device="cuda"), torch.empty(rows, 64, dtype=torch.int32, device="cuda")] for _ in range(2)]
        for (lse, ids), w in zip(got, (work, None)):
            gpu.logprobs(ctx, x[:rows], lse=lse, top_ids=ids, work=w)
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]), rows
        assert torch.equal(got[0][1].long(), torch.sort(x[:rows], dim=1, descending=True, stable=True).indices[:, :64]), rows


def test_many_small_terms_beside_a_large_one(env):
    """A thread's small terms, each below half a step of its sum, are not lost: 944 of e^-17 behind one of 1."""
    rows, V = 400, 248320                                       # one part a row, 61 turns
    x = torch.full((rows, V), -9.1, device="cuda")
    x[:, :4096] = 0
    x[:, 4096:8192:16] = 7.99
    tok = torch.full((rows,), 4096, device="cuda", dtype=torch.int32)
    out = run(env, x, tok, 1)
    z = torch.log_softmax(x[0].double(), 0)
    # 61 turns' sums, 6 roundings in a turn, 15 joins and 3 of exp, 2^-24 of the sum each; the entropy's second sum is 0.05 of
    # the first, with 16 more roundings of its factors
    bound = 85 * 2.0 ** -24
    for name, want, b in (("logprob", z[4096], bound), ("lse", torch.logsumexp(x[0].double(), 0), bound), ("entropy", -(torch.exp(z) * z).sum(), 1.1 * bound)):
        off = (out[name].double() - want).abs().max()
        assert off <= b + 2.0 ** -24 * want.abs(), (name, off / 2.0 ** -24)


def test_tokens_near_certainty(env):
    """Log probabilities around -3e-4 keep an f32 sum's roundings, not those of a logit's exponential."""
    rows, V = 2000, 8192
    g = gen(3)
    x, r = torch.randn(rows, V, device="cuda", generator=g), torch.arange(rows, device="cuda")
    tok = torch.randint(V, (rows,), device="cuda", generator=g)
    x[r, tok] = 17 + torch.rand(rows, device="cuda", generator=g)
    out = run(env, x, tok.int(), 1)
    want = torch.log_softmax(x.double(), 1)[r, tok]
    assert -1e-3 < want.min() and want.max() < -1e-4
    # the sum is 1 and a little: 2 turns, 6 roundings in one and 9 joins, half a step of 2^-23 each at most, 1 / sqrt(3) of that
    # in the mean: sqrt(17 / 3) 2^-24
    for got in (out["logprob"], out["top_logprobs"][:, 0]):
        off = (got.double() - want) * 2.0 ** 24
        assert off.abs().max() <= 17 and off.square().mean().sqrt() <= 3, (off.abs().max(), off.square().mean().sqrt())
