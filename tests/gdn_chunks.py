"""A model of the chunked delta rule with the operands that the matrix cores get, and the error bounds that it stands for.

An f32 value x enters a product as two f16 values, hi + lo: off by 2^-22 |x|, and by 2^-25 of its column's unit at least.
`chunks` forms the products of chunks of 32 rows from such operands (sums in 64 bits, results in 32); `single` names
operands that are left as their hi alone, 2^-11 off instead.  A chunk's values and T are scaled by a power of two that its
betas call for, so that what counts beside |S| is beta |v|."""
import math

import torch

import gdn_ref as R

N = 32
# State, right hand sides, T, the solved rows before the state and before the outputs, scores, keys, queries.
OPERANDS = ("S", "r", "T", "y", "x", "A", "K", "Q")


def scales(beta):
    """Per chunk and head: the power of two not below the chunk's largest beta, or 1 for betas above 1/4."""
    most = torch.stack([beta[c:c + N].float().amax(0) for c in range(0, beta.shape[0], N)])
    return torch.where(most > 0.25, 1.0, torch.exp2(torch.ceil(torch.log2(most.clamp(min=2.0 ** -60)))))


def chunks(q, k, v, g, beta, S, single=(), key_head="mod", scaled=True):
    """As gdn_ref.rule on f32 tensors, without M."""
    n, H, D = v.shape
    m = [h % k.shape[1] if key_head == "mod" else h // (H // k.shape[1]) for h in range(H)]
    per_head = lambda x: x[:, m].transpose(0, 1)                           # [H, n, D]
    length = lambda x: x.float() / torch.sqrt((x.float() ** 2).sum(-1, keepdim=True) + 1e-6)

    def halves(name, x):
        hi = x.float().half().double()
        return hi, torch.zeros_like(hi) if name in single else (x.double() - hi).half().double()

    def product(a, b):                                                     # without the product of the two low halves
        return (a[0] @ b[0] + a[1] @ b[0] + a[0] @ b[1]).float()

    scale = scales(beta) if scaled else torch.ones(-(-n // N), H)
    k, q, v = per_head(length(k)), per_head(length(q)), v.float().transpose(0, 1)
    g, beta = g.float().t(), beta.float().t()
    pad = -n % N
    grow = lambda x, to=0.0: torch.cat([x, torch.full((H, pad, *x.shape[2:]), to)], 1)
    k, q, v, g, beta = grow(k), grow(q), grow(v), grow(g), grow(beta)
    S = torch.zeros(H, D, D) if S is None else S.float().clone()
    o, unit = torch.zeros(H, n + pad, D), None
    low = torch.ones(N, N).tril().bool()
    for c in range((n + pad) // N):
        at, after = slice(c * N, c * N + N), slice(c * N + N, c * N + 2 * N)
        sc, here = scale[c][:, None], v[:, at].abs().amax(1) * scale[c][:, None]
        nxt = v[:, after].abs().amax(1) * scale[c + 1][:, None] if (c + 1) * N < n + pad else torch.zeros(H, D)
        if unit is None:
            unit = _unit(torch.maximum(S.abs().amax(1), here))
        s = S / unit[:, None]
        G = torch.cumsum(g[:, at].double(), 1)
        decay = (torch.exp(torch.where(low, G[:, :, None] - G[:, None], 0.0)) * low).float()
        K, Q, SS = halves("K", k[:, at]), halves("Q", q[:, at]), halves("S", s)
        turned = tuple(x.transpose(1, 2) for x in K)
        L = beta[:, at, None] * decay * product(K, turned) * low.tril(-1)
        T = torch.linalg.inv((torch.eye(N) + L).double()).float() * (beta[:, None, at] / sc[..., None])
        A = halves("A", 64 * decay * product(Q, turned))
        eG = torch.exp(G).float()[..., None]
        r = v[:, at] * sc[..., None] / unit[:, None] - eG * sc[..., None] * product(K, SS)
        d = product(halves("T", T), halves("r", r))
        o[:, at] = (eG * product(Q, SS) + product(A, halves("x", d)) / 64) * unit[:, None]
        y = d * torch.exp(G[:, -1:] - G).float()[..., None]
        S = (eG[:, -1:] * s + product(turned, halves("y", y))) * unit[:, None]
        fresh, in_units = _unit(torch.maximum(S.abs().amax(1), torch.maximum(here, nxt))), nxt / unit
        unit = torch.where((in_units < 0.125) | (in_units >= 16) | (c % 8 == 7), fresh, unit)
    return o[:, :n].transpose(0, 1) / math.sqrt(D), S


def _unit(x):
    return torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -120))))


def bounds(g, m, wider=1, linear=0):
    """Of each output [n, H, D] and of the state's columns' lengths [H, D], for keys, queries, values and gates that are
    independent of each other; g the log decays, m the largest of a column's |state| + s |v| in a row's chunk and the one before,
    s the chunk's scale.

    An operand's element is off by 2^-22 of itself at most, and by 2^-25 of its column's unit, which is no more than 8 m; below
    2^-22 m, with a sign of its own.  A row's d has the errors of S, k, s v, s r and T / s in it, each times a vector of length 1
    or less; it enters the state along k, with the errors of y and k there and 2^-22 m more for lengths, decays
    and sums in f32 (2^-24 times the root of their terms): sqrt(8) 2^-22 m a row.  Later rows do not enlarge what is there,
    they let it decay, and errors of independent signs add as their squares.  The largest of the columns may be twice that.
    An output has the state's error along q, and its own: S and q, and the 32 terms of the scores times x, from two operands
    each.  Queries have no direction in common with keys or errors: a product with one of length 1 is 1 / sqrt(D), 4 / sqrt(D)
    among all the outputs.

    `wider`: those errors that many times over; `linear`: besides, an error of that many 2^-22 m a row that is the same in
    every row, so that rows' errors add up."""
    n, D = m.shape[0], m.shape[2]
    e = 2.0 ** -22 * m
    fall = torch.exp(2 * g.double())[..., None]
    square, line, before = torch.zeros_like(e[0]), torch.zeros_like(e[0]), torch.empty_like(e)
    for t in range(n):
        square = square * fall[t] + 8 * (wider * e[t]) ** 2
        line = line * fall[t].sqrt() + linear * e[t]
        before[t] = square.sqrt() + line
    return 4 / math.sqrt(D) * (before + wider * math.sqrt(2 * N + 4) * e) / math.sqrt(D), 2 * square.sqrt() + line


def share(got, want, limits):
    """The largest error of outputs and state in units of their bounds."""
    part = lambda x, b: float((x / b).max())
    return part((got[0].double() - want[0]).abs(), limits[0]), part((got[1].double() - want[1]).norm(dim=1), limits[1])


def inputs(n, nkh, nvh, D, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    q, k, v = r(n, nkh, D).to(dtype), r(n, nkh, D).to(dtype), r(n, nvh, D).to(dtype)
    return q, k, v, -torch.exp(1.5 * r(n, nvh) - 3), torch.sigmoid(r(n, nvh)), 0.2 * r(nvh, D, D)


def reference(q, k, v, g, beta, S, key_head="mod", wider=1, linear=0):
    """(outputs, end state) in 64 bits, and the bounds of both."""
    n, H, D = v.shape
    scale = scales(beta)
    S = torch.zeros(H, D, D, dtype=torch.float64) if S is None else S.double()
    o, size = torch.empty(n, H, D, dtype=torch.float64), torch.empty(n, H, D, dtype=torch.float64)
    for t in range(n):
        r = slice(t, t + 1)
        before = S.norm(dim=1)
        o[t], S, _ = R.rule(q[r], k[r], v[r], g[r].double(), beta[r].double(), S, key_head)
        size[t] = torch.maximum(before, S.norm(dim=1)) + v[t].double().abs() * scale[t // N].double()[:, None]
    m = torch.stack([size[c:c + N].amax(0) for c in range(0, n, N)])
    m[1:] = torch.maximum(m[1:], m[:-1])
    return (o, S), bounds(g, m.repeat_interleave(N, 0)[:n], wider, linear)


def small_betas(n, H, D, seed, dtype=torch.float32):
    """A head each of betas around 2^-3, 2^-8, .. : the state is far below the values.  The last head's betas are small in its
    first chunks, then near 1 for a chunk, then small again."""
    q, k, v, g, beta, _ = inputs(n, H, H, D, seed, dtype)
    beta = beta * torch.exp2(-3.0 - 5 * torch.arange(H))
    beta[96:128, -1] = 0.9
    return q, k, v, g, beta, None


def long_betas(kind, n, H, D, seed, dtype=torch.float32):
    """Inputs with betas above 1, and how far the bounds of `bounds` widen (wider, linear).  With keys that are independent
    d's errors, and T's besides, grow by a beta each: 4 times.

    With one key for all rows T's entries are 4 in every row: a row's d has errors of 32 of them and of as many right hand sides,
    sqrt(2 * 32) * 4 2^-22 M, where the bounds count sqrt(8) 2^-22 M: 12 times.  And errors of sums that are alike in every row
    add up: the key's length is off by up to 4 * 2^-24 (a sum, a root, a quotient, a product), which enters d and y, times beta
    each: 4 2^-22 M; the sum T r has partial sums of 8 M (its terms of 4 M alternate), and a matrix instruction's adds of its 32
    terms, 8 of 4 at a time, may each cut 2^-23 of that off: 8 * 8 / 2 = 32 2^-22 M.  The value's sign alternates there, so that the
    state grows by two values a row, and the values grow to 16 units of their column right after the unit was chosen."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    q, k, v = r(n, H, D).to(dtype), r(n, H, D).to(dtype), r(n, H, D)
    gate, beta = torch.zeros(n, H), torch.full((n, H), 1.5 if kind == "1.5" else 2.0)
    if kind in ("2", "1.5"):
        gate = -torch.exp(1.5 * r(n, H) - 3)
        return (q, k, v.to(dtype), gate, beta, 0.2 * r(H, D, D)), dict(wider=4)
    k.zero_()
    k[:, :, 5] = 1.0078125                   # of length 1.98 in powers of two
    if kind == "spread":
        k.copy_(r(1, H, D).to(dtype).expand_as(k))
    t = torch.arange(n)[:, None, None]
    v = (1 + 0.2 * torch.rand(1, H, D, generator=g)) * torch.where(t < 9 * N, 1.0, 13 * (1 - 2.0 * (t % 2)))
    return (q, k, v.to(dtype), gate, beta, torch.zeros(H, D, D)), dict(wider=12, linear=36)
