"""Plain 64-bit references of the serving operators (rotary positions, paged
cache, prompt and tree attention) and the error bounds of the kernels."""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def rope_freqs(n_rot, theta, scaling="plain", factor=1.0, orig_ctx=0.0, beta_fast=32.0, beta_slow=1.0, freq_dim=0, mscale=0.0):
    d = freq_dim or n_rot
    f = [theta ** (-2.0 * i / d) for i in range(n_rot // 2)]
    m = mscale or 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        c = lambda b: d * math.log(orig_ctx / (2 * math.pi * b)) / (2 * math.log(theta))
        lo, hi = max(math.floor(c(beta_fast)), 0), min(math.ceil(c(beta_slow)), d - 1)
        hi = lo + 0.001 if hi == lo else hi
        r = [min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(n_rot // 2)]
        f = [x * (1 - a) + x / factor * a for x, a in zip(f, r)]
        m = mscale or 0.1 * math.log(factor) + 1
    return f, m


def rope_turn(x, pos, n_rot, layout, freqs, m, inverse=False):
    """x [T, H, D] in 64 bits, turned."""
    x = x.double().cpu().clone()
    a = pos.double().cpu()[:, None] * torch.tensor(freqs, dtype=torch.float64)[None]
    c, s = (m * torch.cos(a))[:, None], (m * torch.sin(a))[:, None] * (-1 if inverse else 1)
    if layout == "pairs":
        u, v = x[..., 0:n_rot:2].clone(), x[..., 1:n_rot:2].clone()
        x[..., 0:n_rot:2], x[..., 1:n_rot:2] = u * c - v * s, u * s + v * c
    else:
        h = n_rot // 2
        u, v = x[..., :h].clone(), x[..., h:n_rot].clone()
        x[..., :h], x[..., h:n_rot] = u * c - v * s, u * s + v * c
    return x


def rope_bound(x, n_rot, layout, m, out):
    """The largest error of a turned element: the sine and cosine (of an angle
    rounded to f32 after its reduction: 2^-24 of at most pi, and 2 ulp of the
    functions), their product with m, two products and a sum in f32, and the
    rounding to the output's type."""
    x = x.double().cpu().abs()
    mag = x.clone()
    if layout == "pairs":
        s = x[..., 0:n_rot:2] + x[..., 1:n_rot:2]
        mag[..., 0:n_rot:2] = mag[..., 1:n_rot:2] = s
    else:
        h = n_rot // 2
        s = x[..., :h] + x[..., h:n_rot]
        mag[..., :h] = mag[..., h:n_rot] = s
    calc = (math.pi + 4 + 3) * 2.0 ** -24 * m * mag
    least = 2.0 ** -25 if out == torch.float16 else 2.0 ** -133 if out == torch.bfloat16 else 0.0
    return calc + UNIT[out] * (m * mag + calc) + least


def attention(q, k, v, sees, scale):
    """q [n, D], k, v [m, D], sees [n, m]: outputs, lse, and the sums A = sum p |v| / l
    and S = scale * max over keys of sum |q||k| that the error bound takes.  Keys that
    a row does not see are left out, whatever they hold."""
    q, k, v = q.double(), k.double(), v.double()
    n, D = q.shape
    o = torch.zeros(n, v.shape[1], dtype=torch.float64, device=q.device)
    lse = torch.full((n,), -math.inf, dtype=torch.float64, device=q.device)
    A, S, V = torch.zeros_like(o), torch.zeros_like(lse), torch.zeros_like(lse)
    kz, vz = k.clone(), v.clone()
    anyone = sees.any(0)
    kz[~anyone], vz[~anyone] = 0, 0
    odd = ~(torch.isfinite(kz).all(1) & torch.isfinite(vz).all(1))
    for i in ([int(x) for x in torch.arange(n)] if bool(odd.any()) else [slice(None)]):
        rows = slice(i, i + 1) if isinstance(i, int) else i
        see = sees[rows]
        kk, vv = kz, vz
        if isinstance(i, int):
            kk, vv = kz.clone(), vz.clone()
            kk[~see[0]], vv[~see[0]] = 0, 0
        s = scale * (q[rows] @ kk.t().contiguous())
        s = torch.where(see, s, torch.full_like(s, -math.inf))
        some = see.any(1)
        z = torch.logsumexp(s, 1)
        p = torch.where(see, torch.exp(s - torch.where(some, z, torch.zeros_like(z))[:, None]), torch.zeros_like(s))
        o[rows], A[rows] = p @ vv, p @ vv.abs()
        lse[rows] = torch.where(some, z, torch.full_like(z, -math.inf))
        if m := k.shape[0]:
            S[rows] = scale * torch.where(see, q[rows].abs() @ kk.abs().t().contiguous(), torch.zeros_like(s)).max(1).values
            V[rows] = torch.where(torch.isfinite(vv), vv.abs(), torch.zeros_like(vv)).max()
    return o, lse, A, S, V


def attention_bounds(o, lse, A, S, V, n_keys, D, typ):
    """Errors of the outputs and of lse.  A score is a sum of D products in f32, scaled and
    shifted by the row's maximum: at most (D + 4) 2^-24 S off, plus 2^-22 for the exponential;
    a probability is then rounded to the operands' type (half a step, for f16 below its normal
    range 2^-25 against sums of at least 1); sums of n_keys terms in f32; the division and the
    rounding of the output."""
    d = (D + 4) * 2.0 ** -24 * S + 2.0 ** -22
    u = UNIT[typ]
    rel = (u + 2 * d + (n_keys + 4) * 2.0 ** -23)[:, None]
    eo = rel * A + (n_keys * 2.0 ** -25 * V if typ == torch.float16 else 0 * V)[:, None]
    eo = eo + u * (o.abs() + eo) + (2.0 ** -25 if typ == torch.float16 else 0)
    el = d + (n_keys + 4) * 2.0 ** -24 + 2.0 ** -22 * (1 + lse.abs().nan_to_num(posinf=0))
    return eo, el


def signature(n, D):
    """Keys whose place shows in the output: key j has the score -level[j] in powers of two (0 to 3, by units of
    128 keys) and the value 1 in dim dims[j] only, another one for every 16 keys.  All weights are powers of two and
    exact in 16 bits, so a row's output is 2^-level summed by dim over its whole sum."""
    j = torch.arange(n)
    return (j // 128 * 5 + j // 1024) % 4, (j // 16 * 7 + j // 4096) % D


def signature_output(level, dims, D):
    w = 2.0 ** -level.double()
    return torch.zeros(D, dtype=torch.float64).index_add_(0, dims, w) / w.sum()


def signature_bound(want, n, typ):
    """The output's rounding; the sum in f32, its n terms in lanes and waves of which one adds n / 2 at most; the exponents and factors."""
    return want * (UNIT[typ] + n / 2 * 2.0 ** -24 + 2.0 ** -20)
