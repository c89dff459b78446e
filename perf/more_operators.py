"""The linear layers' and the head's serving operators, as cases that can be timed.

Four operators, each through the package's public entry points:

  conv      the 4-tap causal convolution with SiLU over packed sequences, its
            history in the slots of a pool: `gdn_conv`
  prompt    the gated delta rule over packed prompts, states in slots: `gdn_prompt`
  step      the gated delta rule for one or a few tokens of each of many sequences: `gdn_step`
  logprobs  log probabilities of given tokens with their rank, the entropy and
            the top alternatives over given logits: `logprobs`

`listed` holds ordinary sizes, `draw` spreads them.  Shapes are those of the
27B-shape decoder's GatedDeltaNet layers (16 key and 48 value heads of 128) and
head (248320 rows), and generic ones.  The plain forms are elementary torch in
32 bits (the prompt's in chunks of 64, batched), `exact` the definitions in 64
bits, token after token.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
VOCAB = 248320


def listed():
    return [
        # a serial decode step of the 27B shape: one token's mixed row, as the projection leaves it
        {"name": "conv_token", "kind": "conv", "S": 1, "total": 1, "nkh": 16, "nvh": 48, "D": 128, "src": "f32", "type": "f32", "spread": 1},
        # packed prompts of a 16-bit program, some of them continued behind a cached prefix
        {"name": "conv_prompt", "kind": "conv", "S": 5, "total": 8192, "nkh": 16, "nvh": 48, "D": 128, "src": "bf16", "type": "bf16",
         "spread": 2},
        # many short prompts that arrive together
        {"name": "prompt_short", "kind": "prompt", "S": 40, "total": 2003, "nkh": 16, "nvh": 32, "D": 128, "type": "f16", "spread": 3},
        # one long prompt through one layer of the 27B shape: nothing but the heads runs side by side
        {"name": "prompt_layer", "kind": "prompt", "S": 1, "total": 8192, "nkh": 16, "nvh": 48, "D": 128, "type": "bf16", "spread": 4},
        # a full prefill batch
        {"name": "prompt_packed", "kind": "prompt", "S": 9, "total": 16301, "nkh": 16, "nvh": 48, "D": 128, "type": "bf16", "spread": 5},
        # this library's own f32 activations, short heads, grouped key heads
        {"name": "prompt_f32", "kind": "prompt", "S": 3, "total": 1029, "nkh": 8, "nvh": 24, "D": 64, "type": "f32", "spread": 6},
        # a serial decode step
        {"name": "step_token", "kind": "step", "S": 1, "draft": 1, "nkh": 16, "nvh": 48, "D": 128, "type": "bf16", "verify": False, "spread": 7},
        # a decode step of a full batch: the states in and out
        {"name": "step_batch", "kind": "step", "S": 128, "draft": 1, "nkh": 16, "nvh": 48, "D": 128, "type": "bf16", "verify": False,
         "spread": 8},
        # drafted chains of 9: scored with the states left alone, then the accepted prefixes alone move them
        {"name": "step_drafts", "kind": "step", "S": 24, "draft": 9, "nkh": 16, "nvh": 48, "D": 128, "type": "f32", "verify": True,
         "spread": 9},
        # what one request's new token is reported with
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "V": VOCAB, "type": "f32", "top": 5, "masked": False, "peak": 8},
        # a batch's new tokens under a grammar: masked logits, more alternatives
        {"name": "logprobs_batch", "kind": "logprobs", "rows": 96, "V": VOCAB, "type": "bf16", "top": 20, "masked": True, "peak": 6},
        # a prompt's tokens scored: every position, no alternatives but the best
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 1500, "V": VOCAB, "type": "f32", "top": 1, "masked": False, "peak": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["conv", "prompt", "prompt", "step", "step", "logprobs", "logprobs"])
    if kind == "logprobs":
        V, typ = _log(rng, 1000, VOCAB), rng.choice(["f32", "f16", "bf16"])
        return {"kind": kind, "rows": _log(rng, 1, 1500), "V": V, "type": typ, "top": rng.choice([0, 1, 2, 5, 10, 20, 33, 64]),
                "masked": rng.random() < 0.5, "peak": rng.randint(1, 12)}
    nkh, nvh, D = rng.choice([(16, 48, 128), (16, 32, 128), (4, 8, 128), (5, 5, 128), (8, 24, 64), (16, 16, 64), (1, 3, 64)])
    c = {"kind": kind, "nkh": nkh, "nvh": nvh, "D": D, "spread": rng.randint(10, 99999)}
    if kind == "step":
        c.update(S=_log(rng, 1, 128), draft=rng.choice([1, 1, 2, 4, 9, 16]), type=rng.choice(["f32", "f16", "bf16"]), verify=rng.random() < 0.4)
        c["S"] = min(c["S"], 1 + 256 // c["draft"])
        return c
    c["S"] = _log(rng, 1, 40)
    c["total"] = c["S"] + _log(rng, 1, 16000)
    if kind == "conv":
        c["total"] = min(c["total"], 8192)
        c.update(src=rng.choice(["f32", "f16", "bf16"]))
        c["type"] = rng.choice([c["src"], "f16", "bf16"])
    else:
        c["type"] = rng.choice(["f32", "f16", "bf16"])
    return c


# ---------------------------------------------------------------- shapes that follow from a case
def _lens(c):
    """The sequences' tokens: for prompts c["total"] over c["S"], none empty, unequal; for steps up to c["draft"]."""
    rng, S = random.Random(c["spread"]), c["S"]
    if c["kind"] == "step":
        return [c["draft"]] + [rng.randint(max(1, c["draft"] // 2), c["draft"]) for _ in range(S - 1)]
    w = [math.exp(2 * rng.random()) for _ in range(S)]
    n = [1 + int(x / sum(w) * (c["total"] - S)) for x in w]
    n[0] += c["total"] - sum(n)
    return n


def _slots(c):
    """(src, dst) of the sequences: prompts start anew but for every third, which continues its slot; steps continue."""
    S = c["S"]
    order = random.Random(c["spread"] + 1).sample(range(S + 1), S)
    if c["kind"] == "step":
        return order, order
    return [s if i % 3 == 2 else -1 for i, s in enumerate(order)], order


def _accepted(c):
    rng = random.Random(c["spread"] + 2)
    return [rng.randint(1, n) for n in _lens(c)]


def _channels(c):
    return (2 * c["nkh"] + c["nvh"]) * c["D"]


def work(c):
    w = {"f16": 2, "bf16": 2, "f32": 4}
    k = c["kind"]
    if k == "logprobs":
        n = c["rows"] * c["V"]
        return {"bytes": n * w[c["type"]] + c["rows"] * (4 + 16 + 8 * c["top"]), "flops": 5 * n}
    C, T = _channels(c), sum(_lens(c))
    src, dst = _slots(c)
    if k == "conv":
        hist = 12 * C * (sum(s >= 0 for s in src) + len(dst))
        return {"bytes": T * C * (w[c["src"]] + w[c["type"]]) + hist + 16 * C, "flops": 12 * T * C}
    state = 4 * c["nvh"] * c["D"] ** 2 * (sum(s >= 0 for s in src) + len(dst))
    rows = T * ((C + c["nvh"] * c["D"]) * w[c["type"]] + 8 * c["nvh"])
    return {"bytes": rows + state, "flops": 6 * T * c["nvh"] * c["D"] ** 2}


# ---------------------------------------------------------------- inputs
class _Source:
    """Seeded values on the GPU: the same for the same seed and order."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(9_973 * int(seed) + 29)

    def normal(self, typ, *shape):
        x = torch.empty(shape, dtype=TYPES[typ], device=DEV)
        return x.normal_(generator=self.g)

    def uniform(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=DEV).uniform_(generator=self.g)

    def ints(self, hi, *shape):
        return torch.randint(hi, shape, generator=self.g, device=DEV, dtype=torch.int32)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _inputs(c, seed):
    s, k = _Source(seed), c["kind"]
    if k == "logprobs":
        rows, V, top = c["rows"], c["V"], c["top"]
        x = s.normal(c["type"], rows, V).mul_(2.5)
        tok = s.ints(V, rows)
        # most rows have a few tokens well above the rest, as a trained head gives them; the given token is often one of them
        hot = s.ints(V, rows, 4).long()
        up = torch.arange(1, 5, device=DEV) * (c["peak"] * s.uniform(rows, 1))
        x.scatter_add_(1, hot, up.to(x.dtype))
        tok = torch.where(s.uniform(rows) < 0.7, hot[:, 3].int(), tok)
        if c["masked"]:
            for i in range(0, rows, 2):     # every other row is held to a random part of the vocabulary
                x[i].masked_fill_(s.uniform(V) < 0.6, float("-inf"))
        f = lambda: torch.empty(rows, dtype=torch.float32, device=DEV)
        return {"x": x, "tok": tok, "logprob": f(), "entropy": f(), "lse": f(), "rank": torch.empty(rows, dtype=torch.int32, device=DEV),
                "ids": torch.empty(rows, top, dtype=torch.int32, device=DEV),
                "top": torch.empty(rows, top, dtype=torch.float32, device=DEV)}
    lens, (src, dst), C = _lens(c), _slots(c), _channels(c)
    T, S, nvh, D = sum(lens), c["S"], c["nvh"], c["D"]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    st = {"lens": lens, "cu": _ints(cu), "src": _ints(src), "dst": _ints(dst)}
    if k == "conv":
        st.update(x=s.normal(c["src"], T, C), y=torch.empty(T, C, dtype=TYPES[c["type"]], device=DEV), kw=s.normal("f32", C, 4) * 0.3,
                  hist=s.normal("f32", 1, S + 1, C, 3))
        return st
    # the heads as the convolution leaves them, side by side in a token's row
    x = s.normal(c["type"], T, C)
    qk = c["nkh"] * D
    st.update(q=x[:, :qk].unflatten(1, (-1, D)), k=x[:, qk:2 * qk].unflatten(1, (-1, D)), v=x[:, 2 * qk:].unflatten(1, (-1, D)),
              a=s.normal("f32", T, nvh), b=s.normal("f32", T, nvh), A=-torch.exp(2 * s.uniform(nvh) - 1), dt=2 * s.normal("f32", nvh) - 3,
              o=torch.zeros(T, nvh, D, dtype=TYPES[c["type"]], device=DEV), state=0.1 * s.normal("f32", 1, S + 1, nvh, D, D),
              accepted=_ints(_accepted(c)))
    return st


_context = None


def _ctx():
    global _context
    if _context is None:
        from cwen_amd import gpu
        _context = gpu.Context(0)
    return _context


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = c = case
    if own:
        from cwen_amd import gpu
        st["gpu"], st["ctx"] = gpu, _ctx()
        if c["kind"] == "logprobs":
            st["work"] = gpu.logprobs_work(c["rows"], c["V"], c["top"])
        else:
            st["pool"] = gpu.GdnPool(c["nkh"], c["nvh"], c["D"], st.get("state"), st.get("hist"))
        if c["kind"] == "prompt":
            st["work"] = st["pool"].prompt_work(c["total"], c["S"], st["q"].dtype, st["o"].dtype)
    return st


# ---------------------------------------------------------------- the operators
def run(st):
    k = st["case"]["kind"]
    return (_own if own else _plain)[k](st)


def _own_conv(st):
    st["gpu"].gdn_conv(st["ctx"], st["pool"], 0, st["x"], st["kw"], st["y"], st["cu"], st["src"], st["dst"])
    return st["y"], st["hist"]


def _own_prompt(st):
    st["gpu"].gdn_prompt(st["ctx"], st["pool"], 0, st["q"], st["k"], st["v"], st["a"], st["b"], st["o"], st["cu"], st["src"], st["dst"],
                         A=st["A"], dt=st["dt"], work=st["work"])
    return st["o"], st["state"]


def _own_step(st):
    g, ctx, c = st["gpu"], st["ctx"], st["case"]
    rows = (st["q"], st["k"], st["v"], st["a"], st["b"])
    if not c["verify"]:
        g.gdn_step(ctx, st["pool"], 0, *rows, st["o"], st["cu"], st["src"], st["dst"], A=st["A"], dt=st["dt"])
    else:
        g.gdn_step(ctx, st["pool"], 0, *rows, st["o"], st["cu"], st["src"], None, A=st["A"], dt=st["dt"])
        g.gdn_step(ctx, st["pool"], 0, *rows, None, st["cu"], st["src"], st["dst"], A=st["A"], dt=st["dt"], count=st["accepted"])
    return st["o"], st["state"]


def _own_logprobs(st):
    st["gpu"].logprobs(st["ctx"], st["x"], st["tok"], st["logprob"], rank=st["rank"], entropy=st["entropy"], lse=st["lse"],
                       top_ids=st["ids"], top_logprobs=st["top"], work=st["work"])
    return st["logprob"], st["rank"], st["entropy"], st["lse"], st["ids"], st["top"]


def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_conv(st):
    x, cu, w = st["x"].float(), st["cu"].long(), st["kw"]
    T, (src, dst) = x.shape[0], (st["src"].long(), st["dst"].long())
    h = torch.where((src >= 0)[:, None, None], st["hist"][0][src.clamp(min=0)], 0.0)        # [S, C, 3]
    t = torch.arange(T, device=DEV)
    seq = (t[:, None] >= cu[None, 1:-1]).sum(1)
    at = t - cu[seq]
    y = x * w[:, 3]
    for back in (1, 2, 3):
        prev = torch.where((at >= back)[:, None], x[(t - back).clamp(min=0)], h[seq, :, (at - back + 3).clamp(max=2)])
        y += prev * w[:, 3 - back]
    st["y"].copy_(_silu(y))
    n = cu[1:] - cu[:-1]
    last = torch.stack([torch.where((n >= b)[:, None], x[(cu[1:] - b).clamp(min=0)],
                                    h[torch.arange(n.shape[0], device=DEV), :, (n - b + 3).clamp(max=2)]) for b in (3, 2, 1)], -1)
    st["hist"][0][dst] = last
    return st["y"], st["hist"]


def _gates(st):
    """Decay in powers of e and beta, [T, value heads]."""
    x = st["a"] + st["dt"]
    soft = torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))
    return st["A"] * soft, 1 / (1 + torch.exp(-st["b"]))


def _unit(x):
    """[T, key heads, D] with rows of length 1."""
    x = x.float()
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _per_value_head(st):
    """q, k, v [T, value heads, D] in 32 bits; value head h reads key head h % key heads."""
    m = torch.arange(st["case"]["nvh"], device=DEV) % st["case"]["nkh"]
    return _unit(st["q"])[:, m], _unit(st["k"])[:, m], st["v"].float()


def _plain_prompt(st):
    c, cu, src, dst = st["case"], st["cu"].long(), st["src"].long(), st["dst"].long()
    S, H, D, n, N = c["S"], c["nvh"], c["D"], cu[1:] - cu[:-1], 64
    M = -(-max(st["lens"]) // N)
    g, beta = _gates(st)
    i = torch.arange(M * N, device=DEV)
    there = i[None] < n[:, None]
    at = torch.where(there, cu[:-1, None] + i[None], 0)
    pick = lambda x: torch.where(there.view(S, M * N, *[1] * (x.dim() - 1)), x[at], 0.0)     # padded: no decay, beta 0
    heads = lambda x: pick(x).view(S, M, N, H, -1).permute(1, 0, 3, 2, 4).reshape(M, S * H, N, -1)
    q, k, v = (heads(x) for x in _per_value_head(st))
    g, beta = heads(g).squeeze(-1), heads(beta)
    j = torch.arange(N, device=DEV)
    # decay from j to i, summed over what lies between: exact also where much has decayed before j
    low, below = j[:, None] >= j[None], j[:, None] > j[None]
    cum = torch.cumsum(g.double(), -1)
    decay = torch.exp(torch.where(low, cum[..., :, None] - cum[..., None, :], 0.0).float()) * low
    L = beta * decay * torch.matmul(k, k.transpose(-1, -2).contiguous()) * below
    X = torch.eye(N, device=DEV).expand(M, S * H, N, N).clone()
    for r in range(1, N):       # (1 + L) X = 1, row after row
        X[:, :, r] -= torch.matmul(L[:, :, r:r + 1, :r].contiguous(), X[:, :, :r]).squeeze(2)
    A = torch.matmul(q, k.transpose(-1, -2).contiguous()) * decay
    first, rest = torch.exp(cum).float()[..., None], torch.exp(cum[..., -1:] - cum).float()[..., None]
    kq, krest, U = torch.cat([k, q], 2) * torch.cat([first, first], 2), (k * rest).transpose(-1, -2).contiguous(), beta * v
    s = torch.where((src >= 0)[:, None, None, None], st["state"][0][src.clamp(min=0)], 0.0).view(S * H, D, D)
    out = torch.empty(M, S * H, N, D, device=DEV)
    for m in range(M):
        seen = torch.bmm(kq[m], s)
        d = torch.bmm(X[m], U[m] - beta[m] * seen[:, :N])
        out[m] = seen[:, N:] + torch.bmm(A[m], d)
        s = first[m][:, -1:] * s + torch.bmm(krest[m], d)
    out = out.view(M, S, H, N, D).permute(1, 0, 3, 2, 4).reshape(S, M * N, H, D)
    st["o"].copy_((out[there] / math.sqrt(D)))
    st["state"][0][dst] = s.view(S, H, D, D)
    return st["o"], st["state"]


def _plain_chain(st, n, emit, keep):
    """n[i] tokens of each sequence, one after the other for all sequences together."""
    c, cu, src, dst = st["case"], st["cu"].long(), st["src"].long(), st["dst"].long()
    s = st["state"][0][src]
    g, beta = _gates(st)
    q, k, v = _per_value_head(st)
    for t in range(c["draft"]):
        here = t < n
        at = cu[:-1] + torch.where(here, t, 0)
        kt, one = k[at], here[:, None, None, None]
        d = s * torch.exp(g[at])[..., None, None]
        delta = beta[at][..., None] * (v[at] - (d * kt[..., None]).sum(2))
        d = d + kt[..., None] * delta[:, :, None]
        s = torch.where(one, d, s)
        if emit:
            o = (s * q[at][..., None]).sum(2) / math.sqrt(c["D"])
            st["o"][at[here]] = o[here].to(st["o"].dtype)
    if keep:
        st["state"][0][dst] = s


def _plain_step(st):
    n = st["cu"].long()[1:] - st["cu"].long()[:-1]
    if not st["case"]["verify"]:
        _plain_chain(st, n, True, True)
    else:
        _plain_chain(st, n, True, False)
        _plain_chain(st, st["accepted"].long(), False, True)
    return st["o"], st["state"]


def _plain_logprobs(st):
    top = st["case"]["top"]
    x, tok = st["x"].float(), st["tok"].long()[:, None]
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    ls = torch.log(s)
    st["lse"].copy_((m + ls)[:, 0])
    st["entropy"].copy_((ls - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / s)[:, 0])
    xt = x.gather(1, tok)
    st["logprob"].copy_((xt - m - ls)[:, 0])
    i = torch.arange(x.shape[1], device=DEV)[None]
    st["rank"].copy_(((x > xt) | ((x == xt) & (i < tok))).sum(1))
    if top:
        # distinct keys: the value's order first, then the lower index
        b = (x + 0.0).view(torch.int32)
        key = ((b ^ ((b >> 31) & 0x7FFFFFFF)).long() << 32) + (x.shape[1] - i)
        ids = torch.topk(key, min(top, x.shape[1]), 1).indices
        st["ids"].copy_(ids)
        st["top"].copy_(d.gather(1, ids) - ls)
    return st["logprob"], st["rank"], st["entropy"], st["lse"], st["ids"], st["top"]


_own = {"conv": _own_conv, "prompt": _own_prompt, "step": _own_step, "logprobs": _own_logprobs}
_plain = {"conv": _plain_conv, "prompt": _plain_prompt, "step": _plain_step, "logprobs": _plain_logprobs}


# ---------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    return _exact[case["kind"]](case, st)


def _exact_conv(c, st):
    """Each sequence behind its three past inputs, the taps as a correlation."""
    y, hist, w = torch.empty(st["y"].shape, dtype=torch.float64, device=DEV), st["hist"].double(), st["kw"].double()
    cu, src, dst = st["cu"].tolist(), st["src"].tolist(), st["dst"].tolist()
    ends = []
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        past = hist[0, src[i]].t() if src[i] >= 0 else torch.zeros(3, w.shape[0], dtype=torch.float64, device=DEV)
        row = torch.cat([past, st["x"][a:b].double()])
        z = sum(row[j:j + b - a] * w[:, j] for j in range(4))
        y[a:b] = z * torch.sigmoid(z)
        ends.append(row[-3:].t())
    for i, e in enumerate(ends):
        hist[0, dst[i]] = e
    return y, hist


def _exact_rule(c, st, lens, o, state):
    """The recurrence, token after token; sequences side by side (the longest first, so that those at work stay together)."""
    cu, src, dst = st["cu"].tolist(), st["src"].tolist(), st["dst"].tolist()
    order = sorted(range(c["S"]), key=lambda i: -lens[i])
    m = [h % c["nkh"] for h in range(c["nvh"])]
    unit = lambda x: x.double() * torch.rsqrt(x.double().pow(2).sum(-1, keepdim=True) + 1e-6)
    q, k, v = unit(st["q"])[:, m] * c["D"] ** -0.5, unit(st["k"])[:, m], st["v"].double()
    g = torch.exp(st["A"].double() * torch.nn.functional.softplus(st["a"].double() + st["dt"].double(), threshold=1e9))
    beta = torch.sigmoid(st["b"].double())
    zero = torch.zeros_like(state[0, 0])
    s = torch.stack([state[0, src[i]] if src[i] >= 0 else zero for i in order])
    first = torch.tensor([cu[i] for i in order], device=DEV)
    for t in range(lens[order[0]]):
        n = sum(lens[i] > t for i in order)
        at = first[:n] + t
        kt = k[at]
        s[:n] *= g[at][..., None, None]
        d = beta[at][..., None] * (v[at] - torch.matmul(kt[:, :, None], s[:n])[:, :, 0])
        s[:n].addcmul_(kt[..., None], d[:, :, None])
        if o is not None:
            o[at] = torch.matmul(q[at][:, :, None], s[:n])[:, :, 0]
    return {dst[i]: s[x] for x, i in enumerate(order)}


def _exact_prompt(c, st):
    state, o = st["state"].double(), torch.zeros(st["o"].shape, dtype=torch.float64, device=DEV)
    for slot, s in _exact_rule(c, st, st["lens"], o, state).items():
        state[0, slot] = s
    return o, state


def _exact_step(c, st):
    state, o = st["state"].double(), torch.zeros(st["o"].shape, dtype=torch.float64, device=DEV)
    ends = _exact_rule(c, st, st["lens"], o, state)
    if c["verify"]:
        ends = _exact_rule(c, st, _accepted(c), None, state)
    for slot, s in ends.items():
        state[0, slot] = s
    return o, state


def _exact_logprobs(c, st):
    n, top = c["rows"], c["top"]
    lp, H, Z = (torch.empty(n, dtype=torch.float64, device=DEV) for _ in range(3))
    best = torch.empty(n, top, dtype=torch.float64, device=DEV)
    for a in range(0, n, 64):
        x, tok = st["x"][a:a + 64].double(), st["tok"][a:a + 64].long()
        z = torch.log_softmax(x, 1)
        r = torch.arange(x.shape[0], device=DEV)
        lp[a:a + 64], Z[a:a + 64] = z[r, tok], torch.logsumexp(x, 1)
        H[a:a + 64] = torch.special.entr(torch.exp(z)).sum(1)
        if top:
            best[a:a + 64] = torch.topk(z, top, 1).values
    return lp, None, H, Z, None, best


_exact = {"conv": _exact_conv, "prompt": _exact_prompt, "step": _exact_step, "logprobs": _exact_logprobs}
