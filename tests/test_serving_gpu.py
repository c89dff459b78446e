"""The serving operators on the GPU against plain 64-bit references: rotary
positions, the paged cache's bookkeeping, attention of packed prompts and of
drafted trees, and a step of them together.  The bounds are those of
serving_ref.py, derived from the roundings that the kernels make."""
import math
import random

import pytest

import serving_ref as R

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


# ---------------------------------------------------------------- rotary positions
ROPES = [dict(head_dim=64, n_rot=64, theta=1e4), dict(head_dim=256, n_rot=64, theta=1e7, freq_dim=128),
         dict(head_dim=128, n_rot=96, theta=5e5, scaling="linear", factor=8.0),
         dict(head_dim=128, n_rot=128, theta=1e6, scaling="yarn", factor=4.0, orig_ctx=32768.0),
         dict(head_dim=96, n_rot=32, theta=1e4, scaling="yarn", factor=16.0, orig_ctx=4096.0, beta_fast=8.0, beta_slow=2.0, mscale=1.25)]


def turned(x, pos, cfg, layout, inverse=False):
    f, m = R.rope_freqs(cfg["n_rot"], **{k: v for k, v in cfg.items() if k not in ("head_dim", "n_rot")})
    return R.rope_turn(x, pos, cfg["n_rot"], layout, f, m, inverse), m


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("cfg", ROPES, ids=lambda c: f"{c['head_dim']}-{c['n_rot']}-{c.get('scaling', 'plain')}")
def test_rope_values(env, cfg, layout):
    gpu, ctx = env
    r, D = gpu.Rope(layout=layout, **cfg), cfg["head_dim"]
    for i, (T, H, tx, ty) in enumerate([(1, 1, F32, F32), (3, 5, F32, F16), (77, 24, BF16, BF16), (300, 3, F16, F32), (1, 40, F16, BF16),
                                        (33, 8, BF16, F16), (2, 8, F32, BF16), (19, 7, F16, F16), (5, 3, BF16, F32)]):
        g = gen(100 + i)
        x = randn(g, T, H, D, dtype=tx)
        pos = torch.randint(0, 131072, (T,), device="cuda", dtype=torch.int32, generator=g)
        pos[0], pos[-1] = 0, 2 ** 31 - 1 if T > 1 else 7
        y = torch.full((T, H, D), float("nan"), device="cuda").to(ty)
        gpu.rope(ctx, r, x, y, pos, inverse=bool(i & 1))
        want, m = turned(x, pos, cfg, layout, bool(i & 1))
        far = 2.0 ** -21 * 2 * math.pi * m * x.double().cpu().abs().max()   # the f64 product at 2^31 holds 2^-22 of a circle
        bound = R.rope_bound(x, cfg["n_rot"], layout, m, ty)
        bound[-1] += far
        close(y, want, bound, (layout, T, H, tx, ty))


def test_rope_strides_and_in_place(env):
    gpu, ctx = env
    cfg = dict(head_dim=128, n_rot=64, theta=1e4)
    r, g = gpu.Rope(**cfg), gen(7)
    big = randn(g, 50, 9, 144, dtype=F16)                      # rows with gaps, heads a token apart
    keep = big.clone()
    x = big[:, 2:7, 8:136]
    pos = torch.arange(50, device="cuda", dtype=torch.int32) * 31
    want, m = turned(x, pos, cfg, "pairs")
    out = torch.zeros(5, 50, 128, device="cuda", dtype=F32)    # head-major output
    gpu.rope(ctx, r, x, out.transpose(0, 1), pos)
    close(out.transpose(0, 1), want, R.rope_bound(x, 64, "pairs", m, F32), "strided")
    assert torch.equal(big, keep)
    gpu.rope(ctx, r, x, x, pos)
    close(x, want, R.rope_bound(keep[:, 2:7, 8:136], 64, "pairs", m, F16), "in place")
    big[:, 2:7, 8:136] = keep[:, 2:7, 8:136]
    assert torch.equal(big, keep)                              # nothing outside the heads
    gpu.rope(ctx, r, x[:0], x[:0], pos[:0])
    with pytest.raises(gpu.CwenError):
        gpu.rope(ctx, r, big[:, :, :128], big[:, :, 8:136], pos)   # overlapping, not the same


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_rope_inverse_is_the_gradient(env, layout):
    """<dy, turn(x)> = <turn'(dy), x> and the difference of turn along a direction."""
    gpu, ctx = env
    cfg = dict(head_dim=128, n_rot=64, theta=1e4, scaling="yarn", factor=4.0, orig_ctx=8192.0)
    r, g = gpu.Rope(layout=layout, **cfg), gen(3)
    x, dy, e = (randn(g, 40, 3, 128) for _ in range(3))
    pos = torch.arange(40, device="cuda", dtype=torch.int32) * 1003
    run = lambda t, inv=False: (lambda y: (gpu.rope(ctx, r, t, y, pos, inverse=inv), y)[1])(torch.empty_like(t))
    dx = run(dy, True)
    f, m = R.rope_freqs(64, **{k: v for k, v in cfg.items() if k not in ("head_dim", "n_rot")})
    assert abs(float((dy.double() * run(x).double()).sum() - (dx.double() * x.double()).sum())) <= 40 * 3 * 128 * 16 * 2.0 ** -22 * m
    leaf = x.double().cpu().requires_grad_()
    u, v = (leaf[..., 0:64:2], leaf[..., 1:64:2]) if layout == "pairs" else (leaf[..., :32], leaf[..., 32:64])
    a = pos.double().cpu()[:, None] * torch.tensor(f, dtype=torch.float64)[None]
    c, s = (m * torch.cos(a))[:, None], (m * torch.sin(a))[:, None]
    p, q = u * c - v * s, u * s + v * c
    y = torch.cat([torch.stack([p, q], -1).flatten(-2) if layout == "pairs" else torch.cat([p, q], -1), leaf[..., 64:]], -1)
    y.backward(dy.double().cpu())
    close(dx, leaf.grad, R.rope_bound(dy, 64, layout, m, F32), "formula")
    h = 2.0 ** -6
    diff = ((run(x + h * e).double() - run(x - h * e).double()) / (2 * h) * dy.double()).sum()
    assert abs(float(diff - (dx.double() * e.double()).sum())) <= 40 * 3 * 128 * 16 * 2.0 ** -23 * 8 / h * m


# ---------------------------------------------------------------- paged cache
class HostCache:
    """The cache's rules on host lists, one request after the other."""

    def __init__(self, S, M, P, page):
        self.S, self.M, self.P, self.page = S, M, P, page
        self.table, self.len, self.ref, self.status = [[] for _ in range(S)], [0] * S, [0] * P, 0
        self.rows = [[] for _ in range(S)]                    # what each position holds

    def up(self, n):
        return -(-n // self.page)

    def bad(self, seqs, i):
        return not 0 <= seqs[i] < self.S or seqs.count(seqs[i]) > 1

    def cut(self, s, pages):
        while len(self.table[s]) > pages:
            self.ref[self.table[s].pop()] -= 1

    def truncate(self, seqs, lens):
        for i, s in enumerate(seqs):
            if self.bad(seqs, i) or not 0 <= lens[i] <= self.len[s]:
                self.status |= 2
                continue
            self.len[s] = lens[i]
            self.rows[s] = self.rows[s][:lens[i]]
            self.cut(s, self.up(lens[i]))

    def fork(self, src, dst):
        fine = [0 <= a < self.S and 0 <= b < self.S and dst.count(b) == 1 and b not in src and a not in dst and not self.table[b]
                and self.len[b] == 0 for a, b in zip(src, dst)]
        for a, b, ok in zip(src, dst, fine):
            if not ok:
                self.status |= 2
                continue
            self.table[b] = self.table[a][:self.up(self.len[a])]
            for p in self.table[b]:
                self.ref[p] += 1
            self.len[b], self.rows[b] = self.len[a], list(self.rows[a])

    def reserve(self, seqs, n):
        if any(self.bad(seqs, i) or n[i] < 0 or self.len[s] + n[i] > self.M * self.page for i, s in enumerate(seqs)):
            self.status |= 2
            return
        ref, table = list(self.ref), [list(t) for t in self.table]
        free = [p for p in range(self.P) if ref[p] == 0]
        copies = []
        for s, g in zip(seqs, n):
            if g and self.len[s] % self.page and ref[table[s][self.len[s] // self.page]] > 1:
                if not free:
                    self.status |= 1
                    return
                old = table[s][self.len[s] // self.page]
                ref[old] -= 1
                table[s][self.len[s] // self.page] = free.pop(0)
                ref[table[s][self.len[s] // self.page]] = 1
                copies.append((old, table[s][self.len[s] // self.page], self.len[s] % self.page))
            while len(table[s]) < self.up(self.len[s] + g):
                if not free:
                    self.status |= 1
                    return
                table[s].append(free.pop(0))
                ref[table[s][-1]] = 1
        self.ref, self.table = ref, table

    def keep(self, seqs, count, path, ps):
        for i, s in enumerate(seqs):
            row = path[i][:count[i]] if path is not None else list(range(max(0, count[i])))
            if self.bad(seqs, i) or count[i] < 0 or count[i] > (ps if path is not None else 1 << 30) or \
                    self.len[s] + count[i] > len(self.table[s]) * self.page or \
                    any(r <= b for b, r in zip([-1] + row, row)) or any(self.len[s] + r >= len(self.table[s]) * self.page for r in row) or \
                    any(r != j and self.ref[self.table[s][(self.len[s] + j) // self.page]] != 1 for j, r in enumerate(row)):
                self.status |= 2
                yield i, None
                continue
            yield i, row
            self.len[s] += count[i]
            self.cut(s, self.up(self.len[s]))


def gather(kv, s, n):
    """Rows 0..n-1 of sequence s: [layers, n, heads, D] of k and v."""
    j = torch.arange(n, device="cuda")
    pg = kv.table[s, j // kv.page].long()
    return tuple(x[:, pg, :, j % kv.page].transpose(0, 1).contiguous() for x in (kv.k, kv.v))


@pytest.mark.parametrize("page,heads,D,seed", [(16, 2, 64, 1), (16, 4, 256, 2), (32, 1, 8, 3), (64, 3, 128, 4), (256, 1, 64, 5), (128, 5, 24, 6)])
def test_cache_follows_its_rules(env, page, heads, D, seed):
    """A random walk over every call, good and refused requests, against host lists; what each
    sequence's positions hold is checked too."""
    gpu, ctx = env
    rng, g = random.Random(seed), gen(seed)
    S, M, P, L = 7, 9, 30, 3
    kv = gpu.PagedKV.empty(L, heads, D, page, P, S, M, F16)
    kv.ref.fill_(9)
    kv.reset(ctx)
    host = HostCache(S, M, P, page)
    model = [(torch.zeros(L, 0, heads, D, dtype=F16, device="cuda"),) * 2 for _ in range(S)]

    def agree(what):
        for s in range(S):
            assert kv.table[s].tolist() == host.table[s] + [-1] * (M - len(host.table[s])), (what, s)
        assert kv.len.tolist() == host.len and kv.ref.tolist() == host.ref, what
        assert kv.held.tolist() == [len(t) for t in host.table], what
        assert kv.take_status(ctx) == host.status, what
        host.status = 0
        for s in range(S):
            k, v = gather(kv, s, host.len[s])
            assert torch.equal(k, model[s][0]) and torch.equal(v, model[s][1]), (what, s)

    for step in range(120):
        op = rng.choice(["reserve", "reserve", "fork", "keep", "keep", "truncate"])
        n = rng.randint(1, 4)
        seqs = rng.sample(range(S), n)
        if rng.random() < 0.1:
            seqs[rng.randrange(n)] = rng.choice([-1, S, seqs[0], 2 ** 31 - 1])
        if op == "reserve":
            m = [rng.choice([0, 1, rng.randint(1, 2 * page), rng.randint(1, 5 * page), -1 if rng.random() < 0.1 else 3]) for _ in seqs]
            kv.reserve(ctx, ints(seqs), ints(m))
            host.reserve(seqs, m)
        elif op == "fork":
            empty = [s for s in range(S) if not host.table[s]]
            dst = [rng.choice(empty) if empty and rng.random() < 0.9 else rng.randrange(S) for _ in seqs]
            kv.fork(ctx, ints(seqs), ints(dst))
            before = list(model)
            full = [len(t) for t in host.table]
            host.fork(seqs, dst)
            for a, b in zip(seqs, dst):
                if 0 <= a < S and b not in seqs and full[b] == 0 and len(host.table[b]):
                    model[b] = before[a]
        elif op == "truncate":
            to = [rng.randint(0, max(0, host.len[s])) if 0 <= s < S and rng.random() < 0.8 else rng.choice([0, 5 * page, -1]) for s in seqs]
            none = rng.random() < 0.4
            kv.truncate(ctx, ints(seqs), None if none else ints(to))
            host.truncate(seqs, [0] * n if none else to)
            model = [(k[:, :host.len[s]], v[:, :host.len[s]]) for s, (k, v) in enumerate(model)]
        else:
            ps = rng.randint(1, 40)
            room = [len(host.table[s]) * page - host.len[s] if 0 <= s < S else 0 for s in seqs]
            count, path = [], []
            for r in room:
                c = rng.randint(0, min(ps, r)) if rng.random() < 0.9 else rng.choice([ps + 1, -1, ps])
                row = sorted(rng.sample(range(max(r, c, 1)), max(0, min(c, ps, r))))
                if row and rng.random() < 0.1:
                    row[rng.randrange(len(row))] = rng.choice([row[0], r, -1, 2 ** 31 - 1])
                count.append(c)
                path.append(row + [-7] * (ps - len(row)))
            use = rng.random() < 0.8
            # fill the room of private pages with fresh values, as a step's projections do
            for s in {s for s in seqs if 0 <= s < S}:
                for i, p in enumerate(host.table[s]):
                    if host.ref[p] == 1:
                        a = max(0, host.len[s] - i * page)
                        if a < page:
                            kv.k[:, p, :, a:] = randn(g, L, heads, page - a, D, dtype=F16)
                            kv.v[:, p, :, a:] = randn(g, L, heads, page - a, D, dtype=F16)
            rows = [gather(kv, s, len(host.table[s]) * page) if 0 <= s < S else None for s in seqs]
            kv.keep(ctx, ints(seqs), ints(count), ints(path) if use else None)
            for i, row in host.keep(seqs, count, path if use else None, ps):
                if row is not None:
                    s = seqs[i]
                    at = torch.tensor(list(range(host.len[s])) + [host.len[s] + r for r in row], dtype=torch.long, device="cuda")
                    model[s] = (rows[i][0][:, at], rows[i][1][:, at])
        agree((step, op))


def test_reserve_takes_the_lowest_pages_over_a_large_pool(env):
    """More pages than one sweep of the search holds, in runs and holes; several requests, one
    of many pages; then one page more than there is."""
    gpu, ctx = env
    P, page = 20011, 16
    kv = gpu.PagedKV.empty(1, 1, 8, page, P, 40, 4000, BF16)
    used = torch.rand(P, device="cuda", generator=gen(5)) < 0.6
    used[4096:8192] = True
    kv.ref.copy_(used.int() * 2)
    free = (~used).nonzero().flatten().int()
    n = [0, 1, 16 * 3000, 17, 0, 16 * 2000 + 1]
    kv.reserve(ctx, ints([3, 39, 0, 7, 8, 1]), ints(n))
    at = 0
    for s, m in zip([3, 39, 0, 7, 8, 1], n):
        c = -(-m // page)
        assert torch.equal(kv.table[s, :c], free[at:at + c]) and bool((kv.table[s, c:] == -1).all())
        at += c
    assert kv.take_status(ctx) == 0 and bool((kv.ref[free[:at].long()] == 1).all()) and bool((kv.ref[free[at:].long()] == 0).all())
    left = free.numel() - at
    before = [t.clone() for t in (kv.table, kv.ref, kv.held)]
    kv.reserve(ctx, ints([20, 21, 22]), ints([page * min(left, 2000), page * max(0, min(left - 2000, 3000)), page * 3500]))
    fits = left >= min(left, 2000) + max(0, min(left - 2000, 3000)) + 3500
    assert kv.take_status(ctx) == (0 if fits else 1)
    if not fits:
        assert all(torch.equal(a, b) for a, b in zip(before, (kv.table, kv.ref, kv.held)))


def test_shared_last_page_is_copied_for_all_but_its_last_holder(env):
    gpu, ctx = env
    kv = gpu.PagedKV.empty(2, 2, 64, 16, 40, 12, 6, F16)
    kv.k.normal_(generator=gen(1)), kv.v.normal_(generator=gen(2))
    kv.reserve(ctx, ints([5]), ints([37]))
    kv.keep(ctx, ints([5]), ints([37]))
    kv.fork(ctx, ints([5] * 4), ints([1, 2, 3, 4]))
    kv.truncate(ctx, ints([5]))
    want = gather(kv, 1, 37)
    assert kv.ref.tolist()[:3] == [4, 4, 4]
    kv.reserve(ctx, ints([3, 1, 4, 2]), ints([1, 20, 3, 1]))
    assert kv.table[:5, :4].tolist() == [[-1] * 4, [0, 1, 4, 5], [0, 1, 2, -1], [0, 1, 3, -1], [0, 1, 6, -1]]
    assert kv.ref.tolist()[:8] == [4, 4, 1, 1, 1, 1, 1, 0] and kv.take_status(ctx) == 0
    for s in (1, 2, 3, 4):
        assert all(torch.equal(a, b) for a, b in zip(gather(kv, s, 37), want))


def test_keep_long_paths(env):
    """Paths of more rows than one sweep of the kernel holds, over many pages and layers, beside a
    short one and one that stays; an entry that is no page refuses its request."""
    gpu, ctx = env
    g = gen(33)
    kv = gpu.PagedKV.empty(3, 2, 72, 32, 150, 6, 60, BF16)
    kv.k.copy_(randn(g, *kv.k.shape)), kv.v.copy_(randn(g, *kv.v.shape))
    kv.reserve(ctx, ints([0, 1, 2]), ints([100, 40, 7]))
    kv.keep(ctx, ints([0, 1, 2]), ints([100, 40, 7]))
    kv.reserve(ctx, ints([0, 1, 2]), ints([1700, 1000, 90]))
    rng = random.Random(1)
    paths = [sorted(rng.sample(range(1700), 900)), list(range(300)) + sorted(rng.sample(range(300, 1000), 333)), list(range(64))]
    want = []
    for s, (n, row) in enumerate(zip((100, 40, 7), paths)):
        a = gather(kv, s, int(kv.held[s]) * 32)
        at = torch.tensor(list(range(n)) + [n + r for r in row], device="cuda")
        want.append([x[:, at] for x in a])
    table = [p + [-1] * (900 - len(p)) for p in paths]
    kv.keep(ctx, ints([0, 1, 2]), ints([len(p) for p in paths]), ints(table))
    assert kv.len.tolist()[:3] == [1000, 673, 71] and kv.take_status(ctx) == 0
    for s in range(3):
        assert all(torch.equal(a, b) for a, b in zip(gather(kv, s, int(kv.len[s])), want[s])), s
    assert int((kv.ref > 0).sum()) == sum(-(-n // 32) for n in (1000, 673, 71))
    kv.reserve(ctx, ints([2, 1]), ints([90, 5]))
    kv.table[2, 4] = 150
    before = [t.clone() for t in (kv.k, kv.v)]
    kv.keep(ctx, ints([2, 1]), ints([1, 2]), ints([[80, 0], [0, 1]]))
    assert kv.take_status(ctx) & gpu.KV_ARG and kv.len.tolist()[:3] == [1000, 675, 71]
    assert torch.equal(before[0], kv.k) and torch.equal(before[1], kv.v)


# ---------------------------------------------------------------- projections into the cache
@pytest.mark.parametrize("src,typ,page,layout", [(F32, F16, 16, "pairs"), (BF16, BF16, 64, "halves"), (F16, F16, 256, "halves"),
                                                 (F32, BF16, 32, "pairs")])
def test_rope_kv(env, src, typ, page, layout):
    gpu, ctx = env
    g, D, H, K, L = gen(11), 128, 6, 2, 3
    cfg = dict(head_dim=D, n_rot=64, theta=1e4)
    r = gpu.Rope(layout=layout, **cfg)
    kv = gpu.PagedKV.empty(L, K, D, page, 40, 5, 12, typ)
    kv.k.normal_(generator=g), kv.v.normal_(generator=g)
    kv.reserve(ctx, ints([0, 2]), ints([3 * page, 40]))
    kv.keep(ctx, ints([0, 2]), ints([2 * page, 7]))
    kv.reserve(ctx, ints([0, 4]), ints([page, 2 * page - 3]))
    kv.fork(ctx, ints([2]), ints([1]))                          # sequence 2's page 0 is shared now
    wide = randn(g, 37, (H + 2 * K) * D + 16, dtype=src)        # one projection's row
    q, k, v = (wide[:, a:b].unflatten(1, (-1, D)) for a, b in ((0, H * D), (H * D, (H + K) * D), ((H + K) * D, (H + 2 * K) * D)))
    seq = [0] * 12 + [4] * 12 + [0, 9, -1, 0, 3, 2, 0] + [4] * 6
    slot = [2 * page + i for i in range(12)] + [i for i in range(12)] + [-1, 0, 0, 99 * page, 0, 8, 2 ** 31 - 1] + \
        [12 + i for i in range(6)]
    pos = [s * 17 + 5 if s < 2 ** 20 else 3 for s in slot]
    ok = [0 <= s < 5 and sl >= 0 and sl < 3 * page and s in (0, 4) for s, sl in zip(seq, slot)]
    k0, v0 = kv.k.clone(), kv.v.clone()
    qo = torch.empty(37, H, D, device="cuda", dtype=typ)
    gpu.rope_kv(ctx, r, q, k, v, qo, kv, 1, ints(seq), ints(slot), ints(pos))
    assert kv.take_status(ctx) == gpu.KV_ARG                    # bad ids, slots and the shared page
    want, m = turned(q, ints(pos), cfg, layout)
    close(qo, want, R.rope_bound(q, 64, layout, m, typ), "q")
    want, _ = turned(k, ints(pos), cfg, layout)
    bound, table = R.rope_bound(k, 64, layout, m, typ), kv.table.cpu()
    for t in range(37):
        if ok[t]:
            pg, row = int(table[seq[t], slot[t] // page]), slot[t] % page
            close(kv.k[1, pg, :, row], want[t], bound[t], ("k", t))
            assert torch.equal(kv.v[1, pg, :, row], v[t].to(typ)), ("v", t)
            kv.k[1, pg, :, row], kv.v[1, pg, :, row] = k0[1, pg, :, row], v0[1, pg, :, row]
    assert torch.equal(kv.k, k0) and torch.equal(kv.v, v0)      # and nothing else


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("T", [1, 2, 7, 301])
def test_rope_small_rows_share_workgroups(env, layout, T):
    """Few heads: several tokens to a workgroup; many: one.  The same bits, the same refusals, padding
    and bad tokens among the others."""
    gpu, ctx = env
    g, D, K = gen(T), 64, 1
    r = gpu.Rope(head_dim=D, n_rot=48, theta=1e4, layout=layout)
    q, k, v = randn(g, T, 40, D, dtype=F16), randn(g, T, K, D, dtype=F16), randn(g, T, K, D, dtype=F16)
    pos = torch.randint(0, 1 << 30, (T,), device="cuda", dtype=torch.int32, generator=g)
    rng = random.Random(T)
    slot = [rng.choice([i, i, i, i, -1, 10 ** 6]) for i in range(T)]
    seq = [rng.choice([1, 1, 1, 1, 1, 7, -3]) for _ in range(T)]
    got = []
    for H in (40, 1, 2, 5):
        kv = gpu.PagedKV.empty(1, K, D, 16, 20, 2, 20, BF16)
        kv.reserve(ctx, ints([1]), ints([T]))
        qo = torch.empty(T, H, D, device="cuda", dtype=BF16)
        gpu.rope_kv(ctx, r, q[:, :H].contiguous(), k, v, qo, kv, 0, ints(seq), ints(slot), pos)
        y = torch.empty(T, H, D, device="cuda", dtype=F32)
        gpu.rope(ctx, r, q[:, :H], y, pos, inverse=True)
        got.append((qo, y, kv.k, kv.v, kv.take_status(ctx)))
    for H, one in zip((1, 2, 5), got[1:]):
        assert torch.equal(one[0], got[0][0][:, :H]) and torch.equal(one[1], got[0][1][:, :H])
        assert torch.equal(one[2], got[0][2]) and torch.equal(one[3], got[0][3]) and one[4] == got[0][4]
    assert (got[0][4] != 0) == any(s >= 0 and (s > 10 ** 5 or i != 1) for s, i in zip(slot, seq))


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_rope_kv_in_place(env, layout):
    """q turned where it lies, k and v beside it in the same rows: what two tensors give."""
    gpu, ctx = env
    g, D, H, K, T = gen(23), 64, 5, 2, 301
    r = gpu.Rope(head_dim=D, n_rot=48, theta=1e4, layout=layout)
    kv = gpu.PagedKV.empty(1, K, D, 16, 20, 1, 20, BF16)
    kv.reserve(ctx, ints([0]), ints([T]))
    wide = randn(g, T, (H + 2 * K) * D + 8, dtype=BF16)
    q, k, v = (wide[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    at, before, qo = ints(list(range(T))), wide.clone(), torch.empty(T, H, D, device="cuda", dtype=BF16)
    gpu.rope_kv(ctx, r, q, k, v, qo, kv, 0, at * 0, at, at)
    want = [kv.k.clone(), kv.v.clone()]
    kv.k.fill_(1), kv.v.fill_(1)
    gpu.rope_kv(ctx, r, q, k, v, q, kv, 0, at * 0, at, at)
    used = kv.table[0, :-(-T // 16)].long()
    for pool, w in zip((kv.k, kv.v), want):
        a, b = (x[0, used].transpose(1, 2).reshape(-1, K, D)[:T] for x in (pool, w))
        assert torch.equal(a, b)
    assert torch.equal(q, qo) and torch.equal(wide[:, H * D:], before[:, H * D:]) and kv.take_status(ctx) == 0


# ---------------------------------------------------------------- prompt attention
def prompt_case(gpu, ctx, g, typ, H, K, D, lq, lk=None, spread=1.0, gap=0, lse=True, scale=None, nan=None):
    lk = lk or lq
    Tq, Tk = sum(lq) + gap, sum(lk) + gap
    wide = spread * randn(g, max(Tq, Tk), (H + 2 * K) * D + 8, dtype=F32)
    wide = wide.to(typ)
    cut = lambda a, b, n: wide[:n, a * D:b * D].unflatten(1, (-1, D))
    q, k, v = cut(0, H, Tq), cut(H, H + K, Tk), cut(H + K, H + 2 * K, Tk)
    if nan:
        nan(k, v)
    o = torch.full((Tq, H, D), 7.0, device="cuda", dtype=typ)
    z = torch.full((Tq, H), 7.0, device="cuda") if lse else None
    border = lambda n: ints([sum(n[:i]) for i in range(len(n) + 1)])
    gpu.attn_prompt(ctx, q, k, v, o, border(lq), None if lk is lq else border(lk), lse=z, scale=scale)
    return q, k, v, o, z, lq, lk


def check_prompt(case, typ, scale=None, heads=None):
    q, k, v, o, z, lq, lk = case
    H, K, D = q.shape[1], k.shape[1], q.shape[2]
    a = b = 0
    for n, m in zip(lq, lk):
        sees = torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n)
        for h in heads or range(H):
            w = R.attention(q[a:a + n, h], k[b:b + m, h // (H // K)], v[b:b + m, h // (H // K)], sees, scale or D ** -0.5)
            eo, el = R.attention_bounds(*w, m, D, typ)
            close(o[a:a + n, h], w[0], eo, ("o", n, m, h))
            if z is not None:
                close(z[a:a + n, h], w[1], el, ("lse", n, m, h))
        a, b = a + n, b + m
    assert bool((o[a:] == 7).all()) and (z is None or bool((z[a:] == 7).all()))


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("H,K,D", [(4, 2, 64), (6, 1, 128), (3, 3, 256), (12, 2, 256), (5, 1, 64)])
def test_prompt_lengths(env, typ, H, K, D):
    gpu, ctx = env
    for i, lens in enumerate([[1], [2, 0, 1, 31], [32, 33, 63], [64, 65, 0, 0, 127, 128, 1], [129, 300], [0, 257, 0], [1] * 70, [513, 7]]):
        check_prompt(prompt_case(gpu, ctx, gen(i), typ, H, K, D, lens, gap=i % 3), typ)


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_keys_and_queries_differ(env, typ, D):
    """Contexts before the queries, and more queries than keys: the first rows see nothing."""
    gpu, ctx = env
    for i, (lq, lk) in enumerate([([1], [500]), ([5, 40, 3], [70, 10, 0]), ([200, 1, 64], [100, 1, 320]), ([130], [3]), ([33, 0, 9], [0, 50, 8])]):
        check_prompt(prompt_case(gpu, ctx, gen(40 + i), typ, 4, 2, D, lq, lk), typ)


def test_prompt_long_and_peaked(env):
    """Long rows, large scores (the maximum moves late), a scale of the caller's."""
    gpu, ctx = env
    check_prompt(prompt_case(gpu, ctx, gen(3), BF16, 2, 1, 128, [3001]), BF16)
    check_prompt(prompt_case(gpu, ctx, gen(4), F16, 2, 1, 64, [1500, 77], spread=6.0, lse=False), F16)
    check_prompt(prompt_case(gpu, ctx, gen(5), F16, 2, 2, 256, [700], scale=0.3), F16, scale=0.3)

    def rising(k, v):                                           # every later key scores higher than all before
        k.copy_((torch.arange(k.shape[0], device="cuda") * 0.05)[:, None, None].expand_as(k).to(k.dtype))
    q, k, v, o, z, lq, lk = prompt_case(gpu, ctx, gen(6), F16, 1, 1, 64, [900], nan=rising)
    check_prompt((q, k, v, o, z, lq, lk), F16)


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_hidden_values_have_no_influence(env, typ, D):
    """NaN and infinities in keys and values: rows before them stay finite, rows behind them follow
    the formula; other sequences' and uncovered tokens never leak in."""
    gpu, ctx = env
    odd = [float("nan"), float("inf"), -float("inf")]

    def spoil(k, v):
        for i, at in enumerate((37, 90, 170)):
            v[at, 0, 5 + i] = odd[i]
        k[150, 0, :] = float("nan")
        k[-3:], v[-3:] = float("nan"), float("inf")             # the gap behind the last sequence
        v[200, 1] = float("nan")
    check_prompt(prompt_case(gpu, ctx, gen(8), typ, 4, 2, D, [60, 140, 40, 1], gap=3, nan=spoil), typ)


def test_prompt_many_sequences(env):
    """The search for a workgroup's tile: 64 sequences, 65, 200; long ones between short and empty ones."""
    gpu, ctx = env
    rng = random.Random(9)
    for S, D in ((64, 64), (65, 128), (200, 64)):
        lens = [rng.choice([0, 1, rng.randint(1, 60), rng.randint(1, 200)]) for _ in range(S)]
        lens[3], lens[S - 2] = 700, 333
        check_prompt(prompt_case(gpu, ctx, gen(S), F16, 2, 1, D, lens, gap=2), F16, heads=[0])
    lk = [n + rng.randint(0, 90) for n in lens]
    check_prompt(prompt_case(gpu, ctx, gen(2), BF16, 2, 1, 64, lens, lk), BF16, heads=[1])


def test_prompt_wide_workgroups(env):
    """Sequences of 4096 tokens and more take workgroups of 8 waves."""
    gpu, ctx = env
    check_prompt(prompt_case(gpu, ctx, gen(1), BF16, 2, 1, 128, [4500]), BF16, heads=[1])
    check_prompt(prompt_case(gpu, ctx, gen(2), F16, 1, 1, 256, [4101], [4133]), F16)


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_many_workgroups(env, D, typ):
    """Heads enough that no tile's keys are halved between waves (they are where workgroups are few,
    as in most tests here): lengths around the tiles, keys and queries that differ, hidden NaN."""
    gpu, ctx = env
    H = 1500 if D == 64 else 800
    for i, (lq, lk) in enumerate([([1], None), ([31, 0, 33], [64, 5, 33]), ([64, 65], [65, 64]), ([70, 5], [131, 5]), ([129, 128], None),
                                  ([200], [199]), ([257], [321])]):
        check_prompt(prompt_case(gpu, ctx, gen(60 + i), typ, H, 2, D, lq, lk, gap=i % 2), typ, heads=[0, H // 2 - 1, H - 1])

    def spoil(k, v):
        v[37, 0, 5], v[90, 1, 6] = float("nan"), float("inf")
        k[120, 0, :] = float("nan")
        k[-3:], v[-3:] = float("nan"), float("inf")
    check_prompt(prompt_case(gpu, ctx, gen(8), typ, H, 2, D, [60, 100, 1], gap=3, nan=spoil), typ, heads=[0, 7, H - 1])


def test_prompt_few_workgroups_long(env):
    """Halved keys over many tiles, a late maximum in either half, and more queries than keys."""
    gpu, ctx = env
    for D, typ, n in ((64, BF16, 1111), (128, F16, 1030), (256, F16, 900)):
        for half in (0, 1):
            def late(k, v):                                     # the highest scores lie in one half of the tiles
                j = torch.arange(k.shape[0], device="cuda")
                k.mul_((1 + 3.0 * ((j // 32) % 2 == half) * j / n)[:, None, None].to(k.dtype))
            check_prompt(prompt_case(gpu, ctx, gen(n + half), typ, 2, 1, D, [n, 40], [n + 33, 9], nan=late), typ)


def test_prompt_offsets_past_32_bits(env):
    """Tokens 2^26 elements apart: the last keys lie past 4 GiB."""
    gpu, ctx = env
    g, n, D = gen(5), 70, 64
    big = torch.zeros(n, 1 << 25, dtype=F16, device="cuda")             # 4.4 GiB
    q = randn(g, n, 2, D, dtype=F16)
    big[:, :2 * D] = randn(g, n, 2 * D)
    k, v = big[:, :D].unflatten(1, (1, D)), big[:, D:2 * D].unflatten(1, (1, D))
    o, z = torch.empty_like(q), torch.empty(n, 2, device="cuda")
    gpu.attn_prompt(ctx, q, k, v, o, ints([0, 3, n]), lse=z)
    check_prompt((q, k, v, o, z, [3, n - 3], [3, n - 3]), F16)


def test_prompt_many_heads_sampled(env):
    gpu, ctx = env
    check_prompt(prompt_case(gpu, ctx, gen(9), F16, 24, 4, 256, [1000, 31]), F16, heads=[0, 5, 6, 23])
    check_prompt(prompt_case(gpu, ctx, gen(10), BF16, 32, 8, 128, [77, 1200]), BF16, heads=[0, 3, 4, 31])


# ---------------------------------------------------------------- tree attention
def tree_cache(gpu, ctx, g, typ, K, D, page, lens, nodes, L=2, extra=3):
    S = len(lens)
    M = max(-(-(a + b) // page) for a, b in zip(lens, nodes)) + 1
    P = sum(-(-(a + b) // page) for a, b in zip(lens, nodes)) + extra
    kv = gpu.PagedKV.empty(L, K, D, page, P, S + 2, M, typ)
    order = torch.randperm(P, generator=g, device="cuda").int()
    at = 0
    for s, (a, b) in enumerate(zip(lens, nodes)):
        c = -(-(a + b) // page)
        kv.table[s, :c] = order[at:at + c]
        kv.ref[order[at:at + c].long()] = 1
        kv.len[s], kv.held[s] = a, c
        at += c
    kv.k.copy_(randn(g, *kv.k.shape)), kv.v.copy_(randn(g, *kv.v.shape))
    return kv


def random_tree(rng, n, words):
    """Rows of ancestor bits; now and then a node that sees none of its group."""
    bits = []
    for i in range(n):
        p = rng.randint(-1, i - 1)
        bits.append((1 << i) | (bits[p] if p >= 0 else 0) if rng.random() < 0.9 else 0)
    return bits


def as_words(bits, words):
    out = []
    for b in bits:
        out.append([((b >> (64 * w)) & (2 ** 64 - 1)) - (2 ** 64 if (b >> (64 * w + 63)) & 1 else 0) for w in range(words)])
    return ints(out, torch.int64).view(len(bits), words)


def check_tree(kv, layer, q, o, z, lens, nodes, bits, typ, heads=None, scale=None):
    H, D, K, a = q.shape[1], q.shape[2], kv.heads, 0
    for s, (m, n) in enumerate(zip(lens, nodes)):
        j = torch.arange(m + n, device="cuda")
        pg = kv.table[s, j // kv.page].long()
        k, v = kv.k[layer][pg, :, j % kv.page], kv.v[layer][pg, :, j % kv.page]
        sees = torch.ones(n, m + n, dtype=torch.bool)
        for i in range(n):
            for u in range(n):
                sees[i, m + u] = (bits[a + i] >> u) & 1 if bits is not None else u <= i
        sees = sees.cuda()
        for h in heads or range(H):
            w = R.attention(q[a:a + n, h], k[:, h // (H // K)], v[:, h // (H // K)], sees, scale or D ** -0.5)
            eo, el = R.attention_bounds(*w, m + n, D, typ)
            close(o[a:a + n, h], w[0], eo, ("o", s, m, n, h))
            if z is not None:
                close(z[a:a + n, h], w[1], el, ("lse", s, m, n, h))
        a += n


def run_tree(gpu, ctx, kv, layer, q, lens, nodes, bits, words=1, max_len=None, max_nodes=None, lse=True):
    T = q.shape[0]
    cu = ints([sum(nodes[:i]) for i in range(len(nodes) + 1)])
    o = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype)
    z = torch.full((T, q.shape[1]), 7.0, device="cuda") if lse else None
    gpu.attn_tree(ctx, kv, layer, q, o, ints(list(range(len(lens)))), cu, max_nodes or max(nodes), max(lens) if max_len is None else max_len,
                  mask=None if bits is None else as_words(bits, words), lse=z)
    return o, z


TREES = [([0], [1]), ([1], [1]), ([15, 16, 17], [1, 2, 1]), ([0, 31, 32, 33], [3, 1, 0, 8]), ([500], [1]), ([700, 3], [40, 64]),
         ([130, 0, 64, 257, 1], [16, 5, 33, 1, 20]), ([90] * 20, [2] * 20)]


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("H,K,D,page", [(4, 2, 64, 16), (6, 1, 256, 16), (8, 8, 128, 32), (12, 2, 128, 64), (7, 1, 64, 128), (6, 2, 256, 256)])
def test_tree_shapes(env, typ, H, K, D, page):
    gpu, ctx = env
    for i, (lens, nodes) in enumerate(TREES):
        g, rng = gen(60 + i), random.Random(i)
        kv = tree_cache(gpu, ctx, g, typ, K, D, page, lens, nodes)
        q = randn(g, sum(nodes), H, D, dtype=typ)
        bits = None if i % 3 == 2 else [b for n in nodes for b in random_tree(rng, n, 1)]
        o, z = run_tree(gpu, ctx, kv, 1, q, lens, nodes, bits, lse=i != 4)
        check_tree(kv, 1, q, o, z, lens, nodes, bits, typ)
        assert kv.take_status(ctx) == 0


@pytest.mark.parametrize("H,K,D", [(4, 1, 128), (3, 1, 256)])
def test_tree_wide_masks_and_wrong_hints(env, H, K, D):
    """Groups of up to 256 nodes, masks of 4 words; hints of the longest context that are too small or
    far too large; the mask's bits past the group are ignored."""
    gpu, ctx = env
    lens, nodes, rng, g = [300, 40], [256, 130], random.Random(4), gen(4)
    kv = tree_cache(gpu, ctx, g, BF16, K, D, 16, lens, nodes)
    q = randn(g, sum(nodes), H, D, dtype=BF16)
    bits = [b for n in nodes for b in random_tree(rng, n, 4)]
    noisy = bits[:256] + [b | (((1 << 126) - 1) << 130) for b in bits[256:]]
    for hint in (300, 0, 30000):
        o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, noisy, words=4, max_len=hint)
        check_tree(kv, 0, q, o, z, lens, nodes, bits, BF16)
    o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, None)
    check_tree(kv, 0, q, o, z, lens, nodes, None, BF16)


def test_tree_long_context(env):
    gpu, ctx = env
    for seed, lens, nodes, H, K, D, typ, page in ((1, [20000], [1], 6, 1, 256, F16, 16), (2, [9000, 100], [10, 33], 8, 2, 128, BF16, 64),
                                                  (3, [6000], [64], 8, 2, 64, F16, 32)):
        g = gen(seed)
        kv = tree_cache(gpu, ctx, g, typ, K, D, page, lens, nodes)
        q = randn(g, sum(nodes), H, D, dtype=typ)
        bits = [b for n in nodes for b in random_tree(random.Random(seed), n, 1)]
        o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, bits)
        check_tree(kv, 0, q, o, z, lens, nodes, bits, typ)


@pytest.mark.parametrize("D,typ,per,nodes", [(64, F16, 2, 1), (128, BF16, 4, 3), (256, F16, 1, 2), (64, BF16, 8, 9), (128, F16, 5, 20)])
def test_tree_many_groups(env, D, typ, per, nodes):
    """More groups than a wave has lanes, contexts from 0 to 900, groups without nodes; joined in the
    launch and by one of its own."""
    gpu, ctx = env
    for S in (17, 40, 130):
        rng = random.Random(S + D)
        lens = [rng.choice([0, 1, rng.randint(1, 100), rng.randint(1, 900)]) for _ in range(S)]
        n = [rng.choice([0, 1, rng.randint(1, nodes), nodes]) for _ in range(S)]
        g = gen(S)
        kv = tree_cache(gpu, ctx, g, typ, 2, D, 16, lens, n, L=1)
        q = randn(g, sum(n), 2 * per, D, dtype=typ)
        bits = [b for m in n for b in random_tree(rng, m, 1)]
        for hint in (max(lens), 100000):
            o, z = run_tree(gpu, ctx, kv, 0, q, lens, n, bits, max_len=hint)
            check_tree(kv, 0, q, o, z, lens, n, bits, typ, heads=[0, 2 * per - 1])
        assert kv.take_status(ctx) == 0


def test_tree_row_tiles_side_by_side(env):
    """Every group with the same number of row tiles (2 and more), and groups that differ by one row."""
    gpu, ctx = env
    for D, H, K, lens, nodes in ((128, 16, 2, [700, 33, 1500], [40, 40, 33]), (256, 6, 1, [2100], [48]), (64, 8, 1, [900, 64], [64, 33]),
                                 (256, 12, 2, [300, 0, 77], [43, 22, 43]), (128, 8, 1, [640, 640], [17, 16])):
        g, rng = gen(D), random.Random(D)
        kv = tree_cache(gpu, ctx, g, F16, K, D, 64, lens, nodes, L=1)
        q = randn(g, sum(nodes), H, D, dtype=F16)
        bits = [b for m in nodes for b in random_tree(rng, m, 1)]
        o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, bits)
        check_tree(kv, 0, q, o, z, lens, nodes, bits, F16, heads=[0, H - 1])


def test_tree_offsets_past_32_bits(env):
    """A cache of more than 2^31 elements: the pages used lie at its two ends."""
    gpu, ctx = env
    g, P = gen(7), 34000
    kv = gpu.PagedKV(256, *(torch.zeros(1, P, 1, 256, 256, dtype=F16, device="cuda") for _ in range(2)),
                     torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), ints([0, 0]), ints([0, 0]), torch.zeros(P, dtype=torch.int32, device="cuda"))
    kv.ref[3:P - 3] = 1
    kv.reserve(ctx, ints([1]), ints([1300]))
    assert kv.table[1].tolist() == [0, 1, 2, P - 3, P - 2, P - 1, -1, -1]
    used = kv.table[1, :6].long()
    kv.k[:, used], kv.v[:, used] = randn(g, 1, 6, 1, 256, 256, dtype=F16), randn(g, 1, 6, 1, 256, 256, dtype=F16)
    kv.keep(ctx, ints([1]), ints([1290]))
    for H in (6, 40):
        q = randn(g, 3, H, 256, dtype=F16)
        o = torch.empty_like(q)
        gpu.attn_tree(ctx, kv, 0, q, o, ints([1]), ints([0, 3]), 3, 1290)
        view = gpu.PagedKV(256, kv.k, kv.v, kv.table[1:], kv.len[1:], kv.held[1:], kv.ref)
        check_tree(view, 0, q, o, None, [1290], [3], None, F16, heads=[0, H - 1])
    kv.fork(ctx, ints([1]), ints([0]))
    kv.ref[5] = 0
    kv.reserve(ctx, ints([0]), ints([4]))                      # copies the filled rows of the last page into page 5
    assert torch.equal(kv.k[:, 5, :, :10], kv.k[:, P - 1, :, :10]) and kv.take_status(ctx) == 0


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("H,K,D", [(4, 2, 64), (2, 2, 128), (20, 2, 128), (6, 1, 256)])
def test_tree_hidden_values_have_no_influence(env, typ, H, K, D):
    """Pages' stale rows are NaN, and so are nodes that others do not see."""
    gpu, ctx = env
    lens, nodes, g = [100, 37, 0], [6, 3, 4], gen(12)
    kv = tree_cache(gpu, ctx, g, typ, K, D, 32, lens, nodes)
    for s, (m, n) in enumerate(zip(lens, nodes)):
        for r in range(m + n, int(kv.held[s]) * 32):
            pg = int(kv.table[s, r // 32])
            kv.k[:, pg, :, r % 32] = float("nan")
            kv.v[:, pg, :, r % 32] = float("nan")
    free = (kv.ref == 0).nonzero().flatten()
    kv.k[:, free], kv.v[:, free] = float("nan"), float("inf")
    bits = [0b1, 0b11, 0b101, 0b1001, 0b11001, 0b100001, 0b1, 0b10, 0b100, 0b1, 0, 0b110, 0b1000]
    for s, node, val in ((0, 3, float("nan")), (0, 2, float("inf")), (1, 1, -float("inf")), (2, 2, float("nan"))):
        r = lens[s] + node
        pg = int(kv.table[s, r // 32])
        kv.v[:, pg, :, r % 32, 1::3] = val
        if s != 1:
            kv.k[:, pg, 0, r % 32, :] = val
    q = randn(g, sum(nodes), H, D, dtype=typ)
    o, z = run_tree(gpu, ctx, kv, 1, q, lens, nodes, bits)
    check_tree(kv, 1, q, o, z, lens, nodes, bits, typ)


@pytest.mark.parametrize("H,K,D,hint", [(6, 1, 256, 2500), (4, 1, 64, 200), (40, 2, 128, 2500)])
def test_tree_hidden_values_across_chunks(env, H, K, D, hint):
    """A hidden node's NaN and infinities where the keys are cut into chunks (joined in the launch and
    behind it): the other rows are those of the formula, the rows that see them are NaN or infinite."""
    gpu, ctx = env
    lens, nodes, g = [2500, 700], [4, 3], gen(17)
    kv = tree_cache(gpu, ctx, g, F16, K, D, 64, lens, nodes, L=1)
    bits = [0b1, 0b11, 0b101, 0b1101, 0b1, 0b10, 0b110]
    for s, node, val in ((0, 1, float("nan")), (0, 3, float("inf")), (1, 0, -float("inf"))):
        r = lens[s] + node
        kv.v[:, int(kv.table[s, r // 64]), :, r % 64, ::5] = val
    q = randn(g, 7, H, D, dtype=F16)
    o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, bits, max_len=hint)
    check_tree(kv, 0, q, o, z, lens, nodes, bits, F16, heads=[0, H - 1])


def test_tree_nodes_past_the_bound_and_bad_state(env):
    """Nodes past max_nodes stay untouched; an id out of range, a length past its pages and an entry
    that is no page raise the flag and touch nothing outside the cache."""
    gpu, ctx = env
    lens, nodes, g = [50, 20, 80], [6, 2, 3], gen(13)
    kv = tree_cache(gpu, ctx, g, F16, 2, 64, 16, lens, nodes)
    q = randn(g, sum(nodes), 4, 64, dtype=F16)
    o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, None, max_nodes=3)
    assert bool((o[3:6] == 7).all()) and bool((z[3:6] == 7).all()) and kv.take_status(ctx) == 0
    check_tree(kv, 0, torch.cat([q[:3], q[6:]]), torch.cat([o[:3], o[6:]]), torch.cat([z[:3], z[6:]]), lens, [3, 2, 3], None, F16)
    for spoil in ("entry", "low entry", "len", "held", "id"):
        c = gpu.PagedKV(16, kv.k, kv.v, kv.table.clone(), kv.len.clone(), kv.held.clone(), kv.ref.clone())
        seqs = ints([0, 1, 2])
        if spoil == "entry":
            c.table[2, 1] = c.c.n_pages
        elif spoil == "low entry":
            c.table[2, 1] = -2 ** 31
        elif spoil == "len":
            c.len[2] = 2 ** 31 - 1
        elif spoil == "held":
            c.held[2] = 1 << 20
        else:
            seqs = ints([0, 1, 900])
        o2 = torch.full(q.shape, 7.0, device="cuda", dtype=F16)
        gpu.attn_tree(ctx, c, 0, q, o2, seqs, ints([0, 6, 8, 11]), 6, 80)
        assert c.take_status(ctx) & gpu.KV_PAGE, spoil
        check_tree(kv, 0, q[:8], o2[:8], None, lens[:2], nodes[:2], None, F16)


# ---------------------------------------------------------------- streams, graphs, repeats
def test_repeats_are_bit_equal_and_graphs_replay(env):
    """A captured step (fork, reserve, rope_kv, tree attention, keep, truncate) replayed between eager
    work gives the eager bits; prompt attention too."""
    gpu, ctx = env
    g, D, H, K, S = gen(21), 128, 8, 2, 3
    lens, nodes = [200, 90, 333], [12, 12, 12]
    kv = tree_cache(gpu, ctx, g, BF16, K, D, 16, lens, [0, 0, 0], extra=40)
    kv2 = gpu.PagedKV.empty(2, K, D, 16, kv.c.n_pages, 6, kv.c.max_pages, BF16)
    for a, b in ((kv2.k, kv.k), (kv2.v, kv.v), (kv2.ref, kv.ref)):
        a.copy_(b)
    kv2.table[:5], kv2.len[:5], kv2.held[:5] = kv.table, kv.len, kv.held
    kv = kv2
    r = gpu.Rope(D, theta=1e5)
    q, k, v = randn(g, 36, H, D), randn(g, 36, K, D), randn(g, 36, K, D)
    qo, o = (torch.empty(36, H, D, device="cuda", dtype=BF16) for _ in range(2))
    src, dst, n12 = ints([0, 1, 2]), ints([3, 4, 5]), ints([12] * 3)
    seq = ints([3] * 12 + [4] * 12 + [5] * 12)
    slot = ints([m + i for m in lens for i in range(12)])
    bits = [b for i in range(3) for b in random_tree(random.Random(i), 12, 1)]
    mask, cu = as_words(bits, 1), ints([0, 12, 24, 36])
    path, count = ints([[0, 2, 5], [1, 3, -1], [11, -1, -1]]), ints([3, 2, 1])
    pq, pk, pv = randn(g, 500, H, D, dtype=BF16), randn(g, 500, K, D, dtype=BF16), randn(g, 500, K, D, dtype=BF16)
    po, pcu = torch.empty(500, H, D, device="cuda", dtype=BF16), ints([0, 130, 131, 500])

    def step(stream=None):
        kv.truncate(ctx, dst, stream=stream)
        kv.fork(ctx, src, dst, stream=stream)
        kv.reserve(ctx, dst, n12, stream=stream)
        gpu.rope_kv(ctx, r, q, k, v, qo, kv, 1, seq, slot, slot, stream=stream)
        gpu.attn_tree(ctx, kv, 1, qo, o, dst, cu, 12, 400, mask=mask, stream=stream)
        kv.keep(ctx, dst, count, path, stream=stream)
        gpu.attn_prompt(ctx, pq, pk, pv, po, pcu, stream=stream)

    out = lambda: [t.clone() for t in (o, qo, po, kv.table, kv.len, kv.held, kv.ref, kv.k[1], kv.v[1])]
    step()
    want = out()
    for _ in range(3):
        step()
        assert all(torch.equal(a, b) for a, b in zip(out(), want))
    check_tree_of = [kv.len[3:].tolist(), kv.take_status(ctx)]
    assert check_tree_of == [[203, 92, 334], 0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(4):
        o.fill_(i), qo.fill_(i), po.fill_(i)
        torch.cuda.synchronize()
        graph.replay()
        if i & 1:
            torch.cuda.synchronize()
            step()
        assert all(torch.equal(a, b) for a, b in zip(out(), want)), i
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out(), want))


@pytest.mark.parametrize("nodes,H", [(1, 4), (1, 12), (9, 8)])
def test_decode_step_in_a_graph(env, nodes, H):
    """A captured decode step (joined in its launch or not) replayed with eager steps of other shapes
    between: bit for bit the eager result, also as the context grows."""
    gpu, ctx = env
    g, lens = gen(5), [700, 90, 1100]
    kv = tree_cache(gpu, ctx, g, F16, 2, 128, 32, [x + 40 for x in lens], [nodes] * 3, L=1)
    q, big = randn(g, 3 * nodes, H, 128, dtype=F16), randn(g, 3 * 40, 16, 128, dtype=F16)
    o, ob = torch.empty_like(q), torch.empty_like(big)
    cu, cub, seqs = ints([i * nodes for i in range(4)]), ints([0, 40, 80, 120]), ints([0, 1, 2])
    run = lambda: gpu.attn_tree(ctx, kv, 0, q, o, seqs, cu, nodes, 1100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    run()
    with torch.cuda.graph(graph, stream=side):
        run()
    for i in range(5):
        kv.len[:3] = ints([x + 7 * i for x in lens])
        run()
        want = o.clone()
        gpu.attn_tree(ctx, kv, 0, big, ob, seqs, cub, 40, 1100)
        o.fill_(3)
        graph.replay()
        assert torch.equal(o, want), i
        check_tree(kv, 0, q, o, None, [x + 7 * i for x in lens], [nodes] * 3, None, F16, heads=[0, H - 1])


def test_counters_are_shared_with_the_gemvs(env):
    """Joins in the launch and GEMVs split over K count arrivals in the same words of a context: in
    turn, without a wait between, each gives the bits that it gives alone."""
    gpu, ctx = env
    from cwen_amd import synth
    qs, sc = synth.q4_rs(5, 48, 5120)
    W = gpu.Weight(ctx, 101, qs, sc, 5120, 48)                 # few rows: K is split
    g, lens = gen(31), [1900, 60, 1200]
    kv = tree_cache(gpu, ctx, g, F16, 4, 256, 16, lens, [1, 1, 1], L=1)
    q = randn(g, 3, 24, 256, dtype=F16)
    x, seqs, cu = randn(g, 8, 5120), ints([0, 1, 2]), ints([0, 1, 2, 3])
    o, y = torch.empty_like(q), torch.empty(8, 48, device="cuda")
    gpu.attn_tree(ctx, kv, 0, q, o, seqs, cu, 1, 1900)
    gpu.gemvb(ctx, W, x, y, 8)
    torch.cuda.synchronize()
    check_tree(kv, 0, q, o, None, lens, [1, 1, 1], None, F16, heads=[0, 23])
    o0, y0 = o.clone(), y.clone()
    for _ in range(20):
        o.fill_(0), y.fill_(0)
        gpu.attn_tree(ctx, kv, 0, q, o, seqs, cu, 1, 1900)
        gpu.gemvb(ctx, W, x, y, 8)
        gpu.attn_tree(ctx, kv, 0, q, o, seqs, cu, 1, 1900)
        assert torch.equal(o, o0) and torch.equal(y, y0)


def test_one_long_context_among_short_ones(env):
    """A batch whose one long context holds nearly all the pieces: more than the launch expects."""
    gpu, ctx = env
    for D, H, K in ((256, 6, 1), (64, 2, 1), (128, 24, 8)):
        lens, nodes = [3] * 20 + [9000] + [0] * 11, [1] * 32
        g = gen(D)
        kv = tree_cache(gpu, ctx, g, BF16, K, D, 64, lens, nodes, L=1)
        q = randn(g, 32, H, D, dtype=BF16)
        o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, [1] * 32)
        check_tree(kv, 0, q, o, z, lens, nodes, [1] * 32, BF16, heads=[0, H - 1])


def test_two_contexts_on_two_streams(env):
    """Calls on two contexts and caches at the same time give what they give alone."""
    gpu, _ = env
    jobs = []
    for i, (typ, D, H, lens, nodes) in enumerate(((F16, 256, 6, [3000], [1]), (BF16, 128, 16, [900, 2000], [20, 12]))):
        g, c = gen(i), gpu.Context(0)
        kv = tree_cache(gpu, c, g, typ, 2, D, 16, lens, nodes, L=1)
        q, pq, pk = randn(g, sum(nodes), H, D, dtype=typ), randn(g, 1500, 4, D, dtype=typ), randn(g, 1500, 2, D, dtype=typ)
        jobs.append(dict(c=c, kv=kv, q=q, o=torch.empty_like(q), pq=pq, pk=pk, po=torch.empty_like(pq), seqs=ints(list(range(len(lens)))),
                         cu=ints([sum(nodes[:k]) for k in range(len(nodes) + 1)]), n=max(nodes), m=max(lens), st=torch.cuda.Stream()))
    border = ints([0, 700, 1500])

    def run(j, stream=None):
        gpu.attn_tree(j["c"], j["kv"], 0, j["q"], j["o"], j["seqs"], j["cu"], j["n"], j["m"], stream=stream)
        gpu.attn_prompt(j["c"], j["pq"], j["pk"], j["pk"], j["po"], border, stream=stream)
    alone = []
    for j in jobs:
        run(j)
        torch.cuda.synchronize()
        alone.append((j["o"].clone(), j["po"].clone()))
        j["o"].fill_(0), j["po"].fill_(0)
    torch.cuda.synchronize()
    for _ in range(6):
        for j in jobs:
            run(j, j["st"])
    torch.cuda.synchronize()
    for j, (o, po) in zip(jobs, alone):
        assert torch.equal(j["o"], o) and torch.equal(j["po"], po)


# ---------------------------------------------------------------- a request, as it is served
@pytest.mark.parametrize("typ,H,K,D,page", [(F16, 6, 1, 256, 16), (BF16, 8, 2, 128, 64), (F16, 8, 4, 64, 32)])
def test_a_request_from_prompt_to_branch(env, typ, H, K, D, page):
    """Two prompts are written and attended, one is forked, both branches draft a tree, one path is kept,
    the next token decodes: every attention agrees with the formula over the tokens that are really there."""
    gpu, ctx = env
    g, rope = gen(31), dict(head_dim=D, n_rot=D // 2, theta=1e4, scaling="yarn", factor=2.0, orig_ctx=64.0)
    r = gpu.Rope(**rope)
    kv = gpu.PagedKV.empty(1, K, D, page, 60, 4, 20, typ)
    n = [75, 130]
    T = sum(n)
    cu, pos = ints([0, 75, 205]), ints(list(range(75)) + list(range(130)))
    seq = ints([0] * 75 + [1] * 130)
    kv.reserve(ctx, ints([0, 1]), ints(n))
    q, k, v = randn(g, T, H, D), randn(g, T, K, D), randn(g, T, K, D)
    qo, o = (torch.empty(T, H, D, device="cuda", dtype=typ) for _ in range(2))
    gpu.rope_kv(ctx, r, q, k, v, qo, kv, 0, seq, pos, pos)
    kr = torch.empty(T, K, D, device="cuda", dtype=typ)
    gpu.rope(ctx, r, k, kr, pos)
    vr = v.to(typ)
    gpu.attn_prompt(ctx, qo, kr, vr, o, cu)
    check_prompt((qo, kr, vr, o, None, n, n), typ)
    kv.keep(ctx, ints([0, 1]), ints(n))
    rows = [kr[:75], kr[75:]], [vr[:75], vr[75:]]
    for s in (0, 1):
        a, b = gather(kv, s, n[s])
        assert torch.equal(a[0], rows[0][s]) and torch.equal(b[0], rows[1][s])   # the fused write and the single turn agree
    # the prompt's last rows again, as a chain over the cache
    kv.truncate(ctx, ints([1]), ints([118]))
    kv.reserve(ctx, ints([1]), ints([12]))
    tail = torch.empty(12, H, D, device="cuda", dtype=typ)
    gpu.rope_kv(ctx, r, q[193:], k[193:], v[193:], qo[193:], kv, 0, seq[193:], pos[193:], pos[193:])
    gpu.attn_tree(ctx, kv, 0, qo[193:], tail, ints([1]), ints([0, 12]), 12, 118)
    w = [R.attention(qo[193:, h], rows[0][1][:, h // (H // K)], rows[1][1][:, h // (H // K)],
                     torch.arange(130, device="cuda")[None] <= 118 + torch.arange(12, device="cuda")[:, None], D ** -0.5) for h in range(H)]
    for h in range(H):
        close(tail[:, h], w[h][0], R.attention_bounds(*w[h], 130, D, typ)[0], ("tail", h))
    kv.keep(ctx, ints([1]), ints([12]))
    # two branches of sequence 1 with a tree each
    kv.fork(ctx, ints([1, 1]), ints([2, 3]))
    kv.reserve(ctx, ints([2, 3]), ints([9, 7]))
    parents = [[-1, 0, 0, 1, 1, 2, 3, 5, 7], [-1, 0, 1, 1, 3, 4, 0]]
    bits, depth = [], []
    for p in parents:
        b = []
        for i, x in enumerate(p):
            b.append((1 << i) | (b[x] if x >= 0 else 0))
        bits += b
        depth += [130 + bin(x).count("1") - 1 for x in b]
    tq, tk, tv = randn(g, 16, H, D), randn(g, 16, K, D), randn(g, 16, K, D)
    tseq, tslot = ints([2] * 9 + [3] * 7), ints([130 + i for i in range(9)] + [130 + i for i in range(7)])
    tqo, to = (torch.empty(16, H, D, device="cuda", dtype=typ) for _ in range(2))
    gpu.rope_kv(ctx, r, tq, tk, tv, tqo, kv, 0, tseq, tslot, ints(depth))
    gpu.attn_tree(ctx, kv, 0, tqo, to, ints([2, 3]), ints([0, 9, 16]), 9, 130, mask=as_words(bits, 1))
    view = gpu.PagedKV(page, kv.k, kv.v, kv.table[2:], kv.len[2:], kv.held[2:], kv.ref)
    check_tree(view, 0, tqo, to, None, [130, 130], [9, 7], bits, typ)
    kv.keep(ctx, ints([2, 3]), ints([4, 2]), ints([[0, 2, 5, 7], [0, 6, -1, -1]]))
    kv.truncate(ctx, ints([3]))
    assert kv.len.tolist() == [75, 130, 134, 0] and kv.take_status(ctx) == 0
    tkr = torch.empty(16, K, D, device="cuda", dtype=typ)
    gpu.rope(ctx, r, tk, tkr, ints(depth))
    a, b = gather(kv, 2, 134)
    assert torch.equal(a[0, 130:], tkr[[0, 2, 5, 7]]) and torch.equal(b[0, 130:], tv[[0, 2, 5, 7]].to(typ))
    assert torch.equal(a[0, :130], rows[0][1]) and torch.equal(b[0, :130], rows[1][1])


# ---------------------------------------------------------------- state that is no state
@pytest.mark.parametrize("H,K,D,n", [(4, 2, 64, 3), (12, 2, 128, 40), (6, 1, 256, 33)])
def test_tree_lengths_that_are_none(env, H, K, D, n):
    """A length below 0 or past the pages raises the flag in every form, with masks and without; the
    other groups are those of the formula and nothing outside the group is written."""
    gpu, ctx = env
    lens, nodes, g = [50, 80, 300], [n, n, n], gen(n)
    kv = tree_cache(gpu, ctx, g, F16, K, D, 16, lens, nodes, L=1)
    q = randn(g, 3 * n, H, D, dtype=F16)
    bits = [b for m in nodes for b in random_tree(random.Random(n), m, 1)]
    for bad in (-1, -100000, -2 ** 31, 2 ** 31 - 1):
        for mask in (bits, None):
            c = gpu.PagedKV(16, kv.k, kv.v, kv.table, kv.len.clone(), kv.held, kv.ref)
            c.len[1] = bad
            o = torch.full((3 * n + 1, H, D), 7.0, device="cuda", dtype=F16)
            gpu.attn_tree(ctx, c, 0, q, o[:-1], ints([0, 1, 2]), ints([0, n, 2 * n, 3 * n]), n, 300,
                          mask=None if mask is None else as_words(mask, 1))
            assert c.take_status(ctx) == gpu.KV_PAGE, bad
            assert bool((o[-1] == 7).all())
            for s in (0, 2):
                view = gpu.PagedKV(16, kv.k, kv.v, kv.table[s:], kv.len[s:], kv.held[s:], kv.ref)
                a, b = s * n, (s + 1) * n
                check_tree(view, 0, q[a:b], o[a:b], None, lens[s:s + 1], [n], None if mask is None else bits[a:b], F16, heads=[0, H - 1])


def test_truncate_of_a_length_past_its_pages(env):
    """A corrupt length: a cut that its pages do not hold is refused and changes nothing, in its own row
    of the table or a neighbour's; one that they hold makes the sequence whole again."""
    gpu, ctx = env
    kv = gpu.PagedKV.empty(1, 1, 64, 16, 40, 3, 10, F16)
    kv.reserve(ctx, ints([0, 1, 2]), ints([160, 40, 90]))
    kv.keep(ctx, ints([0, 1, 2]), ints([160, 40, 90]))
    kv.len[1] = 2 ** 31 - 1
    before = [t.clone() for t in (kv.table, kv.len, kv.held, kv.ref)]
    for to in (2 ** 31 - 1, 2 ** 31 - 16, 49, -2 ** 31):
        kv.truncate(ctx, ints([1]), ints([to]))
        assert kv.take_status(ctx) == gpu.KV_ARG
        assert all(torch.equal(a, b) for a, b in zip(before, (kv.table, kv.len, kv.held, kv.ref))), to
    kv.truncate(ctx, ints([1, 2]), ints([20, 90]))
    assert kv.take_status(ctx) == 0 and kv.len.tolist() == [160, 20, 90] and kv.held.tolist() == [10, 2, 6]
    assert int((kv.ref > 0).sum()) == 18 and int(kv.table[1, 2]) == -1 and torch.equal(kv.table[0], before[0][0])


@pytest.mark.parametrize("H,K,D,lens,nodes", [(384, 192, 128, [936, 808], [64, 192]), (384, 192, 128, [900, 900, 900], [64, 192, 128]),
                                              (512, 128, 128, [500, 500], [64, 192]), (800, 400, 64, [700, 600], [20, 200])])
def test_tree_row_tiles_that_average_the_pieces(env, H, K, D, lens, nodes):
    """Fewer pieces than a group has row tiles, and groups whose tiles add up to those of equal ones."""
    gpu, ctx = env
    g = gen(H)
    kv = tree_cache(gpu, ctx, g, F16, K, D, 64, lens, nodes, L=1)
    q = randn(g, sum(nodes), H, D, dtype=F16)
    o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, None)
    check_tree(kv, 0, q, o, z, lens, nodes, None, F16, heads=[0, H // 2 - 1, H - 1])


# ---------------------------------------------------------------- shares of a row that hold only scores of -inf
@pytest.mark.parametrize("lens,nodes,at", [([32], [1], {0: [32]}), ([700], [2], {0: range(128, 256)}), ([700, 33], [3, 1], {0: range(700), 1: range(33)}),
                                           ([700, 0], [2, 2], {0: range(702), 1: [0]}), ([2500], [3], {0: [2500, 2502]})],
                         ids=["a wave", "a unit", "all cached", "all", "nodes"])
@pytest.mark.parametrize("H,K,D,hint", [(6, 1, 256, 2500), (4, 1, 64, 200), (40, 2, 128, 2500), (24, 2, 128, 0)])
def test_tree_scores_of_minus_infinity(env, H, K, D, hint, lens, nodes, at):
    """Visible keys whose scores are -inf weigh nothing, wherever the keys are cut; a row that
    sees no others is NaN with lse -inf, and so is a dim where a value of weight 0 is NaN.  Also with
    a hidden NaN, which takes the rows one by one."""
    gpu, ctx = env
    for odd in (False, True):
        g = gen(91)
        kv = tree_cache(gpu, ctx, g, F16, K, D, 64, lens, nodes, L=1)
        row = lambda pool, s, r: pool[:, int(kv.table[s, r // 64]), :, r % 64]
        for s, rows in at.items():
            for r in rows:
                row(kv.k, s, r)[..., 0] = -math.inf
        if odd:                                                # the last node of each group is hidden from the others
            for s, (m, n) in enumerate(zip(lens, nodes)):
                if n > 1:
                    row(kv.v, s, m + n - 1)[..., 3] = float("nan")
        q = randn(g, sum(nodes), H, D, dtype=F16)
        q[..., 0] = 1
        o, z = run_tree(gpu, ctx, kv, 0, q, lens, nodes, None, max_len=hint)
        a = 0
        for s, (m, n) in enumerate(zip(lens, nodes)):
            j = torch.arange(m + n, device="cuda")
            pg = kv.table[s, j // 64].long()
            k, v = kv.k[0][pg, :, j % 64], kv.v[0][pg, :, j % 64]
            sees = j[None] <= m + torch.arange(n, device="cuda")[:, None]
            counts = torch.isfinite(k[:, 0, 0])[None] & sees
            for h in (0, H - 1):
                w = R.attention(q[a:a + n, h], k[:, h // (H // K)].nan_to_num(neginf=0), v[:, h // (H // K)], counts, D ** -0.5)
                eo, el = R.attention_bounds(*w, m + n, D, F16)
                some = counts.any(1)
                nan = ((sees & ~counts).float() @ torch.isnan(v[:, h // (H // K)]).float()) > 0       # 0 * NaN
                want = torch.where(some[:, None] & ~nan, w[0], torch.full_like(w[0], float("nan")))
                close(o[a:a + n, h], want, eo, ("o", odd, s, h))
                close(z[a:a + n, h], w[1], el, ("lse", odd, s, h))
            a += n
        assert kv.take_status(ctx) == 0


# ---------------------------------------------------------------- more KV heads than the partials' scratch has room for
@pytest.mark.parametrize("K,D,nodes", [(600, 256, 40), (2400, 256, 3), (2300, 64, 70)])
def test_tree_more_heads_than_the_scratch_holds(env, K, D, nodes):
    """One workgroup then takes all of a head's rows and leaves no partials."""
    gpu, ctx = env
    g, lens, n = gen(K), [150, 3], [nodes, 1]
    kv = tree_cache(gpu, ctx, g, BF16, K, D, 16, lens, n, L=1)
    q = randn(g, sum(n), K, D, dtype=BF16)
    o, z = run_tree(gpu, ctx, kv, 0, q, lens, n, None)
    check_tree(kv, 0, q, o, z, lens, n, None, BF16, heads=[0, 7, K - 1])


def test_rope_turns_as_the_model_does(env, oracle):
    """The configuration of the 27B shape's attention layers against the decoder's own rotation (run.c:1903-1948),
    whose frequencies and angles are f32: at most 6 roundings of the angle.  With freq_dim 0 it is another one."""
    gpu, ctx = env
    cfg = dict(head_dim=256, n_rot=64, theta=1e7, layout="pairs", freq_dim=128)
    g, pos = gen(77), [0, 1, 5, 97, 1000, 4095]
    x = randn(g, len(pos), 3, 256)
    y, other = torch.empty_like(x), torch.empty_like(x)
    gpu.rope(ctx, gpu.Rope(**cfg), x, y, ints(pos))
    gpu.rope(ctx, gpu.Rope(**{**cfg, "freq_dim": 0}), x, other, ints(pos))
    f, m = R.rope_freqs(64, 1e7, freq_dim=128)
    for t, p in enumerate(pos):
        want = torch.from_numpy(oracle.rope(x[t].cpu().numpy(), p)).double()
        mag = x[t].double().cpu().abs()
        pair = (mag[:, 0:64:2] + mag[:, 1:64:2]).repeat_interleave(2, 1)
        bound = torch.zeros_like(want)
        bound[:, :64] = pair * (6 * 2.0 ** -24 * p * torch.tensor(f, dtype=torch.float64).repeat_interleave(2) + (math.pi + 7 + 4) * 2.0 ** -24)
        close(y[t], want, bound, ("model", p))
        assert p == 0 or float((other[t].double().cpu() - want)[:, :64].abs().max()) > 0.01


# ---------------------------------------------------------------- every key in its place
@pytest.mark.parametrize("ctx_len,nodes,H,K,D,typ,page", [(20000, 1, 6, 1, 256, F16, 16), (19991, 1, 8, 2, 128, BF16, 64), (9000, 3, 4, 1, 64, F16, 16),
                                                          (9000, 20, 8, 2, 128, BF16, 16), (20000, 48, 6, 1, 256, F16, 64), (3001, 40, 4, 1, 64, BF16, 32),
                                                          (1100, 1, 24, 4, 256, F16, 16)])
def test_tree_long_context_key_by_key(env, ctx_len, nodes, H, K, D, typ, page):
    """Values that show which keys were taken with which weight: a block of 16 left out, taken twice or read from
    another page exceeds the bound."""
    gpu, ctx = env
    n, g = ctx_len + nodes, gen(ctx_len)
    kv = tree_cache(gpu, ctx, g, typ, K, D, page, [ctx_len], [nodes], L=1)
    level, dims = R.signature(n, D)
    j = torch.arange(n, device="cuda")
    pg = kv.table[0, j // page].long()
    kv.k.fill_(float("nan")), kv.v.fill_(float("nan"))                                 # whatever else is read shows too
    key, val = torch.zeros(n, D, dtype=typ, device="cuda"), torch.zeros(n, D, dtype=typ, device="cuda")
    key[:, 0] = -level.cuda().to(typ)
    val[j, dims.cuda()] = 1
    for h in range(K):                                                                 # a head's values lie a dim further
        kv.k[0, pg, h, j % page], kv.v[0, pg, h, j % page] = key, val.roll(h, 1)
    q = randn(g, nodes, H, D, dtype=typ)
    q[..., 0] = 1
    o, z = torch.empty_like(q), torch.empty(nodes, H, device="cuda")
    gpu.attn_tree(ctx, kv, 0, q, o, ints([0]), ints([0, nodes]), nodes, ctx_len, lse=z, scale=math.log(2))
    for i in {0, nodes // 2, nodes - 1}:
        m = ctx_len + i + 1
        want = R.signature_output(level[:m], dims[:m], D)
        total = float((2.0 ** -level[:m].double()).sum())
        for h in range(H):
            w = want.roll(h // (H // K))
            close(o[i, h], w, R.signature_bound(w, m, typ), ("o", i, h))
            assert abs(float(z[i, h]) - math.log(total)) <= m / 2 * 2.0 ** -24 + 2.0 ** -18, (i, h)
    assert kv.take_status(ctx) == 0


@pytest.mark.parametrize("n,ctx_len,H,K,D,typ", [(4500, 0, 4, 2, 128, BF16), (3001, 0, 2, 1, 256, F16), (2050, 7000, 2, 1, 64, F16), (300, 20000, 4, 1, 128, BF16),
                                                 (4200, 0, 24, 4, 256, F16), (1100, 0, 800, 2, 128, BF16)])
def test_prompt_long_rows_key_by_key(env, n, ctx_len, H, K, D, typ):
    gpu, ctx = env
    m, g = n + ctx_len, gen(n)
    level, dims = R.signature(m, D)
    k, v = (torch.zeros(m, K, D, dtype=typ, device="cuda") for _ in range(2))
    k[:, :, 0] = -level.cuda().to(typ)[:, None]
    for h in range(K):
        v[torch.arange(m, device="cuda"), h, (dims.cuda() + h) % D] = 1
    q = randn(g, n, H, D, dtype=typ)
    q[..., 0] = 1
    o = torch.empty_like(q)
    gpu.attn_prompt(ctx, q, k, v, o, ints([0, n]), ints([0, m]), scale=math.log(2))
    for i in {0, 31, 32, 127, 128, n // 2, n - 129, n - 2, n - 1}:
        w = R.signature_output(level[:ctx_len + i + 1], dims[:ctx_len + i + 1], D)
        for h in {0, H // K - 1, H // 2, H - 1}:
            x = w.roll(h // (H // K))
            close(o[i, h], x, R.signature_bound(x, ctx_len + i + 1, typ), ("o", i, h))


# ---------------------------------------------------------------- workgroups of 8 waves
@pytest.mark.parametrize("typ,H,K,D", [(BF16, 20, 2, 128), (F16, 20, 4, 128), (F16, 24, 4, 256), (BF16, 20, 1, 256)])
def test_prompt_wide_form(env, typ, H, K, D):
    """Long sequences and heads enough that the card is full take 256 queries to a workgroup (fewer heads have
    their tiles' keys halved instead): odd ends, keys and queries that differ, a short sequence beside."""
    gpu, ctx = env
    for i, (lq, lk) in enumerate([([4101], None), ([4096], [4133]), ([4353], [4200]), ([8100, 97], None)]):
        check_prompt(prompt_case(gpu, ctx, gen(70 + i), typ, H, K, D, lq, lk, gap=i & 1), typ, heads=[H - 1])


@pytest.mark.parametrize("typ,H,K,D", [(BF16, 20, 2, 128), (F16, 24, 4, 256)])
def test_prompt_wide_form_hidden_values(env, typ, H, K, D):
    """NaN and infinities that some rows of a workgroup see and others do not, at its first and last keys."""
    gpu, ctx = env

    def spoil(k, v):
        for at, val in ((0, 1e4), (3840, float("nan")), (3999, float("inf")), (4095, -float("inf")), (4300, float("nan"))):
            v[at, 0, at % 7] = val
        k[4200, 0, :] = float("nan")
        k[-3:], v[-3:] = float("nan"), float("inf")             # the gap behind the sequence
    q, k, v, o, z, lq, lk = prompt_case(gpu, ctx, gen(80), typ, H, K, D, [4400], gap=3, nan=spoil)
    for a, b in ((0, 40), (3800, 4400)):                         # the rows around
        sees = torch.arange(4400, device="cuda")[None] <= torch.arange(a, b, device="cuda")[:, None]
        w = R.attention(q[a:b, 0], k[:4400, 0], v[:4400, 0], sees, D ** -0.5)
        eo, el = R.attention_bounds(*w, 4400, D, typ)
        close(o[a:b, 0], w[0], eo, ("o", a))
        close(z[a:b, 0], w[1], el, ("lse", a))
    assert bool(torch.isfinite(o[:4200, H - 1].float()).all()) and bool((o[4400:] == 7).all())


@pytest.mark.parametrize("typ,H,K,D,n", [(F16, 2, 1, 64, 300), (BF16, 2, 1, 256, 300), (F16, 800, 2, 128, 200), (BF16, 20, 2, 128, 4200)])
def test_prompt_scores_of_minus_infinity(env, typ, H, K, D, n):
    """Keys with scores of -inf weigh nothing, whole tiles of them too; the first rows, which see no
    others, are NaN with lse -inf.  In every form, with keys before the queries."""
    gpu, ctx = env
    off, g = 40, gen(n)
    q, k, v = randn(g, n, H, D, dtype=typ), randn(g, n + off, K, D, dtype=typ), randn(g, n + off, K, D, dtype=typ)
    gone = torch.zeros(n + off, dtype=torch.bool, device="cuda")
    gone[:off + 5], gone[64:192], gone[n - 3:n] = True, True, True
    q[..., 0], k[gone, :, 0] = 1, -math.inf
    o, z = torch.empty_like(q), torch.empty(n, H, device="cuda")
    gpu.attn_prompt(ctx, q, k, v, o, ints([0, n]), ints([0, n + off]), lse=z)
    counts = (torch.arange(n + off, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + off) & ~gone[None]
    for h in (0, H - 1):
        w = R.attention(q[:, h], k[:, h // (H // K)].nan_to_num(neginf=0), v[:, h // (H // K)], counts, D ** -0.5)
        eo, el = R.attention_bounds(*w, n + off, D, typ)
        want = torch.where(counts.any(1)[:, None], w[0], torch.full_like(w[0], float("nan")))
        close(o[:, h], want, eo, ("o", h))
        close(z[:, h], w[1], el, ("lse", h))
