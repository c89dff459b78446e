"""Plain 64-bit references of the serving operators of the GatedDeltaNet layers
and of the log probabilities, and the error bounds of the kernels."""
import math

import torch

EPS = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}  # half a step of the smallest


def conv(x, hist, kw):
    """x [n, C] behind hist [C, 3]: silu of the convolution, the history after it, and the bound of an f32 kernel
    (before the rounding to the output's type)."""
    row = torch.cat([hist.double().t(), x.double()])
    w, n = kw.double(), x.shape[0]
    z = sum(row[j:j + n] * w[:, j] for j in range(4)) if n else torch.zeros(0, x.shape[1], dtype=torch.float64)
    mag = sum((row[j:j + n] * w[:, j]).abs() for j in range(4)) if n else z
    y = z * torch.sigmoid(z)
    # four rounded steps of the sum; |silu'| <= 1.1; exp, sum, division and product 6 roundings of at most |z|
    return y, row[-3:].t(), (1.1 * 5 * mag + 8 * z.abs()) * EPS


def gates(a, b, A, dt):
    """Log decay and beta of [T, heads]."""
    if A is None:
        return a.double(), b.double()
    return A.double() * torch.nn.functional.softplus(a.double() + dt.double(), threshold=1e9), torch.sigmoid(b.double())


def unit(x):
    x = x.double()
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def rule(q, k, v, g, beta, S, key_head="mod"):
    """q, k [n, nkh, D], v [n, nvh, D], g (log decay), beta [n, nvh], S [nvh, D, D] or None: outputs, the end state, and
    M [nvh, D]: per column the largest of |state column| + |v| over the rows, which the bounds are in units of."""
    n, H, D = v.shape
    m = [h % k.shape[1] if key_head == "mod" else h // (H // k.shape[1]) for h in range(H)]
    q, k, v = unit(q)[:, m], unit(k)[:, m], v.double()
    S = torch.zeros(H, D, D, dtype=torch.float64) if S is None else S.double().clone()
    o, M = torch.zeros(n, H, D, dtype=torch.float64), S.norm(dim=1)
    for t in range(n):
        S = S * torch.exp(g[t])[:, None, None]
        d = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
        S = S + k[t][:, :, None] * d[:, None]
        o[t] = (S * q[t][:, :, None]).sum(1) / math.sqrt(D)
        M = torch.maximum(M, S.norm(dim=1) + v[t].abs())
    return o, S, M


def step_bounds(n, D, M, out):
    """Of outputs and state after n rows, row after row in f32.  A row's roundings, against a column's |S| + |v| = M:
    the sums S^T k over D / 8 terms a lane and 3 more adds, |k| = 1 (Cauchy-Schwarz); the length of k (the same sums
    halved, a root and a quotient); decay, beta and the two multiply-adds of an element: fewer than 2 (D / 8) + 40 in
    all.  The row's map S -> g (1 - beta k k^T) S does not enlarge what came before for 0 <= beta <= 2."""
    c = 2 * (D / 8) + 40
    state = n * c * EPS * M
    return (state + c * EPS * M) / math.sqrt(D), state


def prompt_bounds(n, D, M, out, full):
    """Of outputs and state after n rows in chunks of 32.  M as above.  Operands carry a relative error of 2^-21 at
    most (two f16 values, or what f32 products and sums leave); a chunk's right hand sides are off by 2^-21 (2 M) (the
    product S^T k, |k| = 1, and v), the solved rows, |T_ij| <= 1 with 32 terms, by 32 times that and again by the
    roundings of T and the right hand sides, and the state by the sum of 32 such rows: below 32 * 32 * 8 * 2^-21 M in
    the worst case, where every error has the same sign; errors of independent signs give the root of the number of
    terms instead: 32 * 8 * 2^-21.  Outputs of 16 bits: single f16 values of S, of the scores (|A| <= 1) and of the
    solved rows, half a step each: 2^-11 (|S| + 2 * 6 * max|d|) <= 2^-11 * 14 M, 6 > sqrt(32)."""
    chunks = (n + 31) // 32
    state = chunks * 256 * 2.0 ** -21 * M
    o = state + 256 * 2.0 ** -21 * M
    if not full:
        o = o + 14 * 2.0 ** -11 * M
    return o / math.sqrt(D), state


def rounded(o, bound, out):
    """The bound of a result `o` that is rounded to a type at the end."""
    return bound + UNIT[out] * (o.abs() + bound) + LEAST[out]


def logprobs(x, tokens, top):
    """logprob, rank, entropy, lse, top ids, top log probabilities of rows x [rows, V]."""
    x = x.double()
    rows, V = x.shape
    bad = x.isnan().any(1) | (x == math.inf).any(1)
    # relative to the largest: beside a logit of 1e38 the log of the sum is lost
    m = torch.where(bad, 0.0, x.nan_to_num(nan=0.0, posinf=0.0, neginf=-math.inf).amax(1))
    d = x - torch.where(torch.isinf(m), torch.zeros_like(m), m)[:, None]
    ls = torch.log(torch.exp(d).sum(1))
    lse = torch.where(bad, torch.nan, m + torch.where(torch.isinf(m), torch.zeros_like(ls), ls))
    z = torch.where((bad | torch.isinf(m))[:, None], torch.nan, d - ls[:, None])
    p = torch.exp(z)
    H = -torch.where(p > 0, p * z, torch.where(p.isnan(), p, 0.0)).sum(1)
    H = torch.where(torch.isinf(lse), torch.nan, H)
    lp, rank = torch.full((rows,), torch.nan, dtype=torch.float64), torch.full((rows,), -1, dtype=torch.int32)
    ids, best = torch.full((rows, top), -1, dtype=torch.int32), torch.full((rows, top), -math.inf, dtype=torch.float64)
    for r in range(rows):
        order = sorted((i for i in range(V) if not math.isnan(x[r, i])), key=lambda i: (-x[r, i].item(), i)) if V <= 5000 else \
            torch.argsort(-x[r], stable=True).tolist()
        for j, i in enumerate(order[:top]):
            ids[r, j], best[r, j] = i, z[r, i]
        t = -1 if tokens is None else int(tokens[r])
        if 0 <= t < V and not math.isnan(x[r, t]):
            lp[r], rank[r] = z[r, t], order.index(t)
    return lp, rank, H, lse, ids, best


def logprobs_bound(V, per_thread, value):
    """Of a log probability, a log of the sums or an entropy of size `value`.  A thread adds per_thread terms, the
    workgroup and the row another 8 + 6 sums; exp of a difference d is off by 3 |d| + 4 roundings, and the mean of |d|
    under the probabilities is at most ln V + 1; renewals of the reference, fewer than 10, 4 roundings each.  The
    entropy's second sum has the same roundings times that mean."""
    c = per_thread + 14 + 3 * (math.log(V) + 1) + 4 + 40
    return c * EPS * (2 + 2 * math.log(V)) + 4 * EPS * value.abs().nan_to_num(nan=0.0, posinf=0.0, neginf=0.0)
