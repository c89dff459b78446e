"""Serving operators around a paged cache, as cases that can be timed.

Four operators, each through the package's public entry points:

  rope    rotary positions: `rope` turns one tensor's heads, `rope_kv` turns a
          step's queries and keys and writes keys and values into the pages
  pages   the paged cache between two steps: `PagedKV.truncate`, `fork`,
          `reserve` (with its copies of shared pages) and `keep`
  prompt  causal attention over packed prompts: `attn_prompt`
  tree    attention of drafted trees over the pages: `attn_tree`

`listed` holds ordinary sizes, `draw` spreads them.  Shapes are those of the
27B-shape decoder's full-attention layers (24/4 heads of 256, 64 rotated
dims), and generic ones of 64 and 128.  The plain forms are elementary torch
in 32 bits (angles in 64), `exact` the definitions in 64 bits.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a serial decode step of the 27B shape: one token's queries, keys and values as the projections leave them
        {"name": "rope_token", "kind": "rope_kv", "T": 1, "S": 1, "nh": 24, "nkv": 4, "D": 256, "rot": 64, "layout": "pairs",
         "scaling": "plain", "src": "f32", "type": "f16", "page": 16, "ctx": 4096},
        # a prompt chunk of a generic decoder with a context scaled past its training
        {"name": "rope_prompt", "kind": "rope_kv", "T": 8192, "S": 3, "nh": 32, "nkv": 8, "D": 128, "rot": 128, "layout": "halves",
         "scaling": "yarn", "src": "bf16", "type": "bf16", "page": 64, "ctx": 131072},
        # turning a tensor back (gradients, moved keys) in full precision, an odd number of tokens, part of the head
        {"name": "rope_back", "kind": "rope", "T": 2051, "nh": 16, "D": 128, "rot": 96, "layout": "pairs", "scaling": "linear",
         "src": "f32", "type": "f32", "inverse": True, "ctx": 32768},
        # one sequence forked, its last page copied, a drafted chain kept: the smallest step
        {"name": "pages_small", "kind": "pages", "layers": 4, "nkv": 4, "D": 256, "page": 16, "type": "f16", "parents": 1,
         "children": 1, "ctx": 100, "grow": 8},
        # beams of a batch: 64 children of 9 parents, trees of up to 32 nodes, all 16 full-attention layers of the 27B shape
        {"name": "pages_batch", "kind": "pages", "layers": 16, "nkv": 4, "D": 256, "page": 16, "type": "f16", "parents": 9,
         "children": 64, "ctx": 1000, "grow": 32},
        # many short ragged prompts in one pack
        {"name": "prompt_short", "kind": "prompt", "S": 40, "total": 5003, "nh": 16, "nkv": 4, "D": 64, "type": "f16", "spread": 5},
        # one prompt through a full-attention layer of the 27B shape
        {"name": "prompt_layer", "kind": "prompt", "S": 1, "total": 4096, "nh": 24, "nkv": 4, "D": 256, "type": "f16", "spread": 1},
        # a pack of unequal prompts
        {"name": "prompt_packed", "kind": "prompt", "S": 9, "total": 16301, "nh": 32, "nkv": 8, "D": 128, "type": "bf16", "spread": 3},
        # the longest context of the framework in one prompt
        {"name": "prompt_long", "kind": "prompt", "S": 1, "total": 32768, "nh": 32, "nkv": 8, "D": 128, "type": "bf16", "spread": 1},
        # serial decode behind a 4K context: one token of one sequence
        {"name": "tree_token", "kind": "tree", "S": 1, "ctx": 4096, "nodes": 1, "nh": 24, "nkv": 4, "D": 256, "type": "f16",
         "page": 16, "shape": 1},
        # a tree of 48 drafts of one sequence behind a long context
        {"name": "tree_long", "kind": "tree", "S": 1, "ctx": 32000, "nodes": 48, "nh": 24, "nkv": 4, "D": 256, "type": "f16",
         "page": 64, "shape": 2},
        # a serving batch: 48 sequences of ragged contexts, each with its own tree of up to 24 nodes
        {"name": "tree_batch", "kind": "tree", "S": 48, "ctx": 12000, "nodes": 24, "nh": 32, "nkv": 8, "D": 128, "type": "bf16",
         "page": 16, "shape": 3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope_kv", "rope", "pages", "prompt", "prompt", "tree", "tree"])
    nh, nkv, D = rng.choice([(24, 4, 256), (16, 4, 256), (32, 8, 128), (28, 4, 128), (8, 8, 128), (16, 4, 64), (32, 2, 64), (5, 1, 128)])
    typ = rng.choice(["f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if kind in ("rope_kv", "rope"):
        c = {"kind": kind, "T": _log(rng, 1, 8192), "nh": nh, "D": D, "rot": rng.choice([D // 4, D // 2, D]),
             "layout": rng.choice(["pairs", "halves"]), "scaling": rng.choice(["plain", "linear", "yarn"]),
             "src": rng.choice(["f32", "f16", "bf16"]), "ctx": _log(rng, 16384, 131072)}
        if kind == "rope":
            c.update(type=rng.choice(["f32", typ]), inverse=rng.random() < 0.5)
        else:
            c.update(type=typ, nkv=nkv, page=page, S=rng.randint(1, 8))
        return c
    if kind == "pages":
        return {"kind": kind, "layers": rng.randint(1, 16), "nkv": nkv, "D": D, "page": page, "type": typ, "parents": _log(rng, 1, 9),
                "children": _log(rng, 1, 64), "ctx": _log(rng, 16, 1000 * 16 // page), "grow": _log(rng, 1, 32)}
    if kind == "prompt":
        S = _log(rng, 1, 64)
        return {"kind": kind, "S": S, "total": S + _log(rng, 1, 16384), "nh": nh, "nkv": nkv, "D": D, "type": typ, "spread": rng.randint(1, 999)}
    S = _log(rng, 1, 48)
    return {"kind": kind, "S": S, "ctx": _log(rng, 16, 300000 // S if S > 9 else 32000), "nodes": _log(rng, 1, 64), "nh": nh, "nkv": nkv,
            "D": D, "type": typ, "page": page, "shape": rng.randint(1, 999)}


# ---------------------------------------------------------------- shapes that follow from a case
def _prompt_lens(c):
    """c["total"] tokens over c["S"] sequences, none empty, unequal."""
    rng, S = random.Random(c["spread"]), c["S"]
    w = [math.exp(2 * rng.random()) for _ in range(S)]
    n = [1 + int(x / sum(w) * (c["total"] - S)) for x in w]
    n[0] += c["total"] - sum(n)
    return n


def _tree_plan(c):
    """Contexts and parents (-1: a root) of each sequence's nodes."""
    rng, plan = random.Random(c["shape"]), []
    for s in range(c["S"]):
        ctx = c["ctx"] if s == 0 else _log(rng, max(1, c["ctx"] // 64), c["ctx"])
        n = c["nodes"] if s == 0 else rng.randint(1, c["nodes"])
        parents = [-1] + [rng.randint(max(0, i - 8), i - 1) for i in range(1, n)]
        plan.append((ctx, parents))
    return plan


def _ancestors(parents):
    """bits[i]: the nodes that node i attends, itself among them."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((1 << i) | (bits[p] if p >= 0 else 0))
    return bits


def _pages_plan(c):
    """Parents' lengths, each child's parent, and the rows each child keeps of its grow new ones."""
    rng = random.Random(17 * c["children"] + c["ctx"])
    lens = [c["ctx"]] + [_log(rng, max(1, c["ctx"] // 4), c["ctx"]) for _ in range(c["parents"] - 1)]
    src = [i % c["parents"] for i in range(c["children"])]
    keep = []
    for _ in src:  # a branch's first rows in place, the others from behind the rows kept: the step can be run again on what it leaves
        m = rng.randint(1, c["grow"])
        first = rng.randint(max(0, 2 * m - c["grow"]), m)
        keep.append(list(range(first)) + sorted(rng.sample(range(m, c["grow"]), m - first)))
    return lens, src, keep


def _up(a, b):
    return (a + b - 1) // b


def work(c):
    w = {"f16": 2, "bf16": 2, "f32": 4}
    k = c["kind"]
    if k in ("rope", "rope_kv"):
        rows = c["T"] * (c["nh"] + (2 * c["nkv"] if k == "rope_kv" else 0))
        turned = c["T"] * (c["nh"] + (c["nkv"] if k == "rope_kv" else 0)) * c["rot"]
        return {"bytes": rows * c["D"] * (w[c["src"]] + w[c["type"]]) + 4 * c["T"], "flops": 3 * turned}
    if k == "pages":
        lens, src, keep = _pages_plan(c)
        row = 2 * c["layers"] * c["nkv"] * c["D"] * 2
        moved = sum(lens[p] % c["page"] for p in src) + sum(sum(1 for i, r in enumerate(rows) if r != i) for rows in keep)
        return {"bytes": 2 * row * moved + 4 * sum(_up(lens[p], c["page"]) for p in src), "flops": 0}
    if k == "prompt":
        lens = _prompt_lens(c)
        pairs = sum(n * (n + 1) // 2 for n in lens)
        return {"bytes": 2 * c["D"] * c["total"] * (2 * c["nh"] + 2 * c["nkv"]) + 4 * c["total"] * c["nh"], "flops": 4 * c["D"] * c["nh"] * pairs}
    plan = _tree_plan(c)
    total = sum(len(p) for _, p in plan)
    pairs = sum(ctx * len(p) + sum(bin(b).count("1") for b in _ancestors(p)) for ctx, p in plan)
    keys = sum(ctx + len(p) for ctx, p in plan)
    return {"bytes": 4 * c["D"] * c["nkv"] * keys + (4 * c["D"] + 4) * c["nh"] * total, "flops": 4 * c["D"] * c["nh"] * pairs}


# ---------------------------------------------------------------- inputs
class _Source:
    """Seeded values on the GPU: the same for the same seed and order."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(7_919 * int(seed) + 11)

    def normal(self, typ, *shape):
        x = torch.empty(shape, dtype=TYPES[typ], device=DEV)
        return x.normal_(generator=self.g)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV).int()


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _cache(s, c, layers, lens, room, spare, seqs):
    """A cache whose sequences 0.. hold `lens` positions (and room[i] more reserved) on shuffled pages."""
    page, need = c["page"], [_up(n + r, c["page"]) for n, r in zip(lens, room)]
    n_pages = sum(need) + spare
    order = s.perm(n_pages)
    t = {"k": s.normal(c["type"], layers, n_pages, c["nkv"], page, c["D"]),
         "v": s.normal(c["type"], layers, n_pages, c["nkv"], page, c["D"])}
    table = torch.full((seqs, max(need) + _up(c.get("grow", 0), page) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    ref = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    ref[order[:at].long()] = 1
    pad = [0] * (seqs - len(lens))
    t.update(table=table, ref=ref, len=_ints(lens + pad), held=_ints(need + pad))
    return t


def _rope_cfg(c):
    scale = max(1.0, c["ctx"] / 32768)
    return {"head_dim": c["D"], "n_rot": c["rot"], "theta": 1e7, "layout": c["layout"], "scaling": c["scaling"], "factor": 2 * scale,
            "orig_ctx": 16384.0}


def _positions(c):
    """The sequences' tokens follow each other; each sequence ends at c["ctx"] or before."""
    rng, T, S = random.Random(c["T"]), c["T"], min(c.get("S", 1), c["T"])
    seq, pos = [], []
    for i in range(S):
        n = T // S + (1 if i < T % S else 0)
        first = c["ctx"] - n - (rng.randint(0, c["ctx"] // 8) if i else 0)
        seq += [i] * n
        pos += range(max(0, first), max(0, first) + n)
    return seq, pos


def _inputs(c, seed):
    s, k = _Source(seed), c["kind"]
    if k == "rope":
        _, pos = _positions(c)
        return {"x": s.normal(c["src"], c["T"], c["nh"], c["D"]), "pos": _ints(pos), "cfg": _rope_cfg(c),
                "y": torch.empty(c["T"], c["nh"], c["D"], dtype=TYPES[c["type"]], device=DEV), "inverse": c["inverse"]}
    if k == "rope_kv":
        seq, pos = _positions(c)
        S = max(seq) + 1
        n = [seq.count(i) for i in range(S)]
        first = [pos[seq.index(i)] for i in range(S)]
        # the cache holds a window: slots count from a few positions before the step's first token
        lens = [p % 97 for p in first]
        slot = [p - first[i] + lens[i] for i, p in zip(seq, pos)]
        t = _cache(s, c, 2, lens, n, 5, S)
        return {"q": s.normal(c["src"], c["T"], c["nh"], c["D"]), "kx": s.normal(c["src"], c["T"], c["nkv"], c["D"]),
                "vx": s.normal(c["src"], c["T"], c["nkv"], c["D"]), "seq": _ints(seq), "slot": _ints(slot), "pos": _ints(pos),
                "qo": torch.empty(c["T"], c["nh"], c["D"], dtype=TYPES[c["type"]], device=DEV), "cache": t, "layer": 1, "cfg": _rope_cfg(c)}
    if k == "pages":
        lens, src, keep = _pages_plan(c)
        P, n = c["parents"], c["children"]
        spare = sum(_up(lens[p] + c["grow"], c["page"]) - lens[p] // c["page"] for p in src) + 3
        t = _cache(s, c, c["layers"], lens, [0] * P, spare, P + n)
        path = [r + [-1] * (c["grow"] - len(r)) for r in keep]
        return {"cache": t, "src": _ints(src), "dst": _ints(list(range(P, P + n))), "zero": _ints([0] * n), "grow": _ints([c["grow"]] * n),
                "path": _ints(path), "count": _ints([len(r) for r in keep])}
    if k == "prompt":
        lens = _prompt_lens(c)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        T = c["total"]
        return {"q": s.normal(c["type"], T, c["nh"], c["D"]), "k": s.normal(c["type"], T, c["nkv"], c["D"]),
                "v": s.normal(c["type"], T, c["nkv"], c["D"]), "cu": _ints(cu), "lens": lens,
                "o": torch.empty(T, c["nh"], c["D"], dtype=TYPES[c["type"]], device=DEV),
                "lse": torch.empty(T, c["nh"], dtype=torch.float32, device=DEV)}
    plan = _tree_plan(c)
    nodes = [len(p) for _, p in plan]
    cu, bits = [0], []
    for _, p in plan:
        cu.append(cu[-1] + len(p))
        bits += [b - (1 << 64) if b >> 63 else b for b in _ancestors(p)]
    t = _cache(s, c, 1, [x for x, _ in plan], nodes, 7, c["S"])
    return {"q": s.normal(c["type"], cu[-1], c["nh"], c["D"]), "cache": t, "seqs": _ints(list(range(c["S"]))), "cu": _ints(cu),
            "mask": _ints(bits, torch.int64).view(-1, 1), "plan": plan, "max_nodes": max(nodes), "max_len": max(x for x, _ in plan),
            "o": torch.empty(cu[-1], c["nh"], c["D"], dtype=TYPES[c["type"]], device=DEV),
            "lse": torch.empty(cu[-1], c["nh"], dtype=torch.float32, device=DEV)}


_context = None


def _ctx():
    global _context
    if _context is None:
        from cwen_amd import gpu
        _context = gpu.Context(0)
    return _context


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        from cwen_amd import gpu
        st["gpu"], st["ctx"] = gpu, _ctx()
        if "cfg" in st:
            st["rope"] = gpu.Rope(**st["cfg"])
        if "cache" in st:
            st["kv"] = gpu.PagedKV(case["page"], **st["cache"])
    elif "cfg" in st:
        st["freq"], st["mscale"] = _freqs(st["cfg"])
    return st


# ---------------------------------------------------------------- the operators
def run(st):
    k = st["case"]["kind"]
    return (_own if own else _plain)[k](st)


def _own_rope(st):
    st["gpu"].rope(st["ctx"], st["rope"], st["x"], st["y"], st["pos"], inverse=st["inverse"])
    return st["y"]


def _own_rope_kv(st):
    st["gpu"].rope_kv(st["ctx"], st["rope"], st["q"], st["kx"], st["vx"], st["qo"], st["kv"], st["layer"], st["seq"], st["slot"], st["pos"])
    return st["qo"], st["cache"]["k"], st["cache"]["v"]


def _own_pages(st):
    """Drop the last step's candidates, fork the parents anew, make room, keep the accepted rows."""
    kv, ctx = st["kv"], st["ctx"]
    kv.truncate(ctx, st["dst"], st["zero"])
    kv.fork(ctx, st["src"], st["dst"])
    kv.reserve(ctx, st["dst"], st["grow"])
    kv.keep(ctx, st["dst"], st["count"], st["path"])
    t = st["cache"]
    return t["k"], t["v"], t["table"], t["len"], t["held"], t["ref"]


def _own_prompt(st):
    st["gpu"].attn_prompt(st["ctx"], st["q"], st["k"], st["v"], st["o"], st["cu"], lse=st["lse"])
    return st["o"], st["lse"]


def _own_tree(st):
    st["gpu"].attn_tree(st["ctx"], st["kv"], 0, st["q"], st["o"], st["seqs"], st["cu"], st["max_nodes"], st["max_len"], mask=st["mask"],
                        lse=st["lse"])
    return st["o"], st["lse"]


def _freqs(cfg):
    """Angular frequencies of the pairs in 64 bits, and the factor on cos and sin."""
    d, theta, s = cfg["n_rot"], cfg["theta"], cfg["factor"]
    i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
    f = torch.exp(-2 * i / d * math.log(theta))
    if cfg["scaling"] == "plain":
        return f, 1.0
    if cfg["scaling"] == "linear":
        return f / s, 1.0
    at = lambda beta: d * math.log(cfg["orig_ctx"] / (2 * math.pi * beta)) / (2 * math.log(theta))
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / s * ramp, 0.1 * math.log(s) + 1


def _turn(st, x, pos, inverse=False):
    """x [T, heads, D] turned, in 32 bits."""
    cfg, x = st["cfg"], x.float()
    n = cfg["n_rot"]
    a = pos.double()[:, None] * st["freq"][None]
    a = a - torch.floor(a / (2 * math.pi)) * (2 * math.pi)
    cos = (torch.cos(a) * st["mscale"]).float()[:, None]
    sin = (torch.sin(a) * (-st["mscale"] if inverse else st["mscale"])).float()[:, None]
    y = x.clone()
    if cfg["layout"] == "pairs":
        u, v = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2], y[..., 1:n:2] = u * cos - v * sin, u * sin + v * cos
    else:
        u, v = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2], y[..., n // 2:n] = u * cos - v * sin, u * sin + v * cos
    return y


def _plain_rope(st):
    st["y"].copy_(_turn(st, st["x"], st["pos"], st["inverse"]))
    return st["y"]


def _plain_rope_kv(st):
    t, l = st["cache"], st["layer"]
    typ, page = t["k"].dtype, t["k"].shape[3]
    st["qo"].copy_(_turn(st, st["q"], st["pos"]))
    seq, slot = st["seq"].long(), st["slot"].long()
    at = t["table"][seq, slot // page].long()
    t["k"][l][at, :, slot % page] = _turn(st, st["kx"], st["pos"]).to(typ)
    t["v"][l][at, :, slot % page] = st["vx"].to(typ)
    return st["qo"], t["k"], t["v"]


def _plain_release(t, seqs, first):
    """Give back the sequences' pages from index `first` [n] on."""
    seqs, first = seqs.long(), first.long()
    col = torch.arange(t["table"].shape[1], device=DEV)[None]
    rows = t["table"][seqs]
    gone = (col >= first[:, None]) & (col < t["held"][seqs][:, None])
    n = t["ref"].shape[0]
    at = torch.where(gone, rows, n).long().flatten()
    t["ref"] -= torch.zeros(n + 1, dtype=torch.int32, device=DEV).index_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:n]
    t["table"][seqs] = torch.where(gone, -1, rows)
    t["held"][seqs] = torch.minimum(t["held"][seqs], first.int())


def _plain_pages(st):
    t = st["cache"]
    page, n_pages, width = t["k"].shape[3], t["ref"].shape[0], t["table"].shape[1]
    src, dst, grow, count = st["src"].long(), st["dst"].long(), st["grow"].long(), st["count"].long()
    n, col = dst.shape[0], torch.arange(width, device=DEV)[None]
    # truncate
    _plain_release(t, dst, (st["zero"] + page - 1) // page)
    t["len"][dst] = st["zero"]
    # fork: whole pages are shared
    ln = t["len"][src].long()
    pages = (ln + page - 1) // page
    rows = torch.where(col < pages[:, None], t["table"][src], -1)
    t["table"][dst], t["len"][dst], t["held"][dst] = rows, ln.int(), pages.int()
    at = torch.where(rows >= 0, rows, n_pages).long().flatten()
    t["ref"] += torch.zeros(n_pages + 1, dtype=torch.int32, device=DEV).index_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:n_pages]
    # reserve: a copy of the last page where others hold it too, then fresh pages, lowest ids first
    last = t["table"][dst, (ln // page).clamp(max=width - 1)].long()
    open_ = (ln % page != 0) & (grow > 0)
    earlier = torch.tril((last[:, None] == last[None, :]) & open_[None, :], -1).sum(1)
    copy = open_ & (t["ref"][last.clamp(min=0)] - earlier > 1)
    want = torch.maximum((ln + grow + page - 1) // page, pages)
    need = want - pages + copy
    first = torch.cumsum(need, 0) - need
    free = torch.argsort((t["ref"] != 0).int(), stable=True)
    for i in range(_up(st["case"]["grow"], page) + 2):
        use = i < need
        page_id = free[(first + i).clamp(max=n_pages - 1)]
        where = torch.where(copy, torch.where(torch.full_like(pages, i) == 0, ln // page, pages + i - 1), pages + i)[use]
        t["table"][dst[use], where] = page_id[use].int()
        t["ref"][page_id[use]] = 1
    old = torch.where(copy, last, n_pages)
    t["ref"] -= torch.zeros(n_pages + 1, dtype=torch.int32, device=DEV).index_add_(0, old, torch.ones_like(old, dtype=torch.int32))[:n_pages]
    t["held"][dst] = want.int()
    fresh = free[first.clamp(max=n_pages - 1)]
    row = torch.arange(page, device=DEV)[None].expand(n, page)
    pick = copy[:, None] & (row < (ln % page)[:, None])
    a, b, r = last[:, None].expand(n, page)[pick], fresh[:, None].expand(n, page)[pick], row[pick]
    # keep: accepted rows move down behind the context
    i = torch.arange(st["path"].shape[1], device=DEV)[None].expand(n, -1)
    used = i < count[:, None]
    frm = (ln[:, None] + st["path"].long())[used]
    to = (ln[:, None] + i)[used]
    who = dst[:, None].expand(n, i.shape[1])[used]
    p0, p1 = t["table"][who, frm // page].long(), t["table"][who, to // page].long()
    for pool in (t["k"], t["v"]):
        for l in range(pool.shape[0]):
            pool[l][b, :, r] = pool[l][a, :, r]
            pool[l][p1, :, to % page] = pool[l][p0, :, frm % page]
    t["len"][dst] += count.int()
    _plain_release(t, dst, (t["len"][dst] + page - 1) // page)
    return t["k"], t["v"], t["table"], t["len"], t["held"], t["ref"]


def _softmax_rows(s, v):
    """Rows of scores [.., q, k] (hidden ones -inf) over v [.., k, D]: outputs and log of the sums."""
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(l == 0, torch.ones_like(l), l)
    return o, (m + torch.log(l)).squeeze(-1)


def _plain_prompt(st):
    q, k, v, D = st["q"], st["k"], st["v"], st["q"].shape[2]
    g, at = q.shape[1] // k.shape[1], 0
    for n in st["lens"]:
        for h in range(k.shape[1]):
            kt = k[at:at + n, h].float().t().contiguous()
            vf = v[at:at + n, h].float().contiguous()
            for a in range(0, n, 2048):
                b = min(n, a + 2048)
                x = q[at + a:at + b, h * g:(h + 1) * g].float().transpose(0, 1).reshape(-1, D)
                s = torch.matmul(x, kt[:, :b].contiguous()).view(g, b - a, b) / math.sqrt(D)
                i = torch.arange(a, b, device=DEV)
                s = s.masked_fill(torch.arange(b, device=DEV)[None] > i[:, None], float("-inf"))
                o, lse = _softmax_rows(s.view(-1, b), vf[:b])
                st["o"][at + a:at + b, h * g:(h + 1) * g] = o.view(g, b - a, D).transpose(0, 1).to(q.dtype)
                st["lse"][at + a:at + b, h * g:(h + 1) * g] = lse.view(g, b - a).t()
        at += n
    return st["o"], st["lse"]


def _plain_tree(st):
    t, q, at = st["cache"], st["q"], 0
    nkv, page, D = t["k"].shape[2:]
    g = q.shape[1] // nkv
    for s, (ctx, parents) in enumerate(st["plan"]):
        n = len(parents)
        j = torch.arange(ctx + n, device=DEV)
        pages = t["table"][s, j // page].long()
        k, v = t["k"][0][pages, :, j % page].float(), t["v"][0][pages, :, j % page].float()      # [keys, nkv, D]
        bit = (st["mask"][at:at + n] >> torch.arange(n, device=DEV)[None]) & 1
        hidden = torch.cat([torch.zeros(n, ctx, dtype=torch.bool, device=DEV), bit == 0], 1)
        x = q[at:at + n].float().view(n, nkv, g, D).permute(1, 2, 0, 3).reshape(nkv, g * n, D).contiguous()
        sc = torch.matmul(x, k.permute(1, 2, 0).contiguous()).view(nkv, g, n, -1) / math.sqrt(D)
        o, lse = _softmax_rows(sc.masked_fill(hidden, float("-inf")).view(nkv, g * n, -1), v.transpose(0, 1).contiguous())
        st["o"][at:at + n] = o.view(nkv, g, n, D).permute(2, 0, 1, 3).reshape(n, -1, D).to(q.dtype)
        st["lse"][at:at + n] = lse.view(nkv, g, n).permute(2, 0, 1).reshape(n, -1)
        at += n
    return st["o"], st["lse"]


_own = {"rope": _own_rope, "rope_kv": _own_rope_kv, "pages": _own_pages, "prompt": _own_prompt, "tree": _own_tree}
_plain = {"rope": _plain_rope, "rope_kv": _plain_rope_kv, "pages": _plain_pages, "prompt": _plain_prompt, "tree": _plain_tree}


# ---------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    return _exact[case["kind"]](case, st)


def _exact_turn(cfg, x, pos, sign=1.0):
    """One complex product per pair: (x + i y) m exp(i pos f)."""
    n, L, s = cfg["n_rot"], cfg["orig_ctx"], cfg["factor"]
    f, m = [cfg["theta"] ** (-2.0 * i / n) for i in range(n // 2)], 1.0
    if cfg["scaling"] == "linear":
        f = [w / s for w in f]
    if cfg["scaling"] == "yarn":
        edge = [n * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(cfg["theta"])) for turns in (32.0, 1.0)]
        lo, hi = float(max(math.floor(edge[0]), 0)), float(min(math.ceil(edge[1]), n - 1))
        if lo == hi:
            hi += 0.001
        r = [min(1.0, max(0.0, (i - lo) / (hi - lo))) for i in range(n // 2)]
        f, m = [w * ((1 - a) + a / s) for w, a in zip(f, r)], 0.1 * math.log(s) + 1.0
    turn = torch.polar(torch.tensor(m, dtype=torch.float64, device=DEV).expand(pos.shape[0], n // 2).contiguous(),
                       sign * torch.outer(pos.double(), torch.tensor(f, dtype=torch.float64, device=DEV)))[:, None]
    x = x.double()
    head, tail = x[..., :n], x[..., n:]
    if cfg["layout"] == "pairs":
        z = torch.view_as_complex(head.unflatten(-1, (n // 2, 2)).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(head[..., :n // 2].contiguous(), head[..., n // 2:].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, tail], -1)


def _exact_rope(c, st):
    return _exact_turn(st["cfg"], st["x"], st["pos"], -1.0 if c["inverse"] else 1.0)


def _exact_rope_kv(c, st):
    t, page = st["cache"], c["page"]
    k, v = t["k"].double(), t["v"].double()
    kt, table = _exact_turn(st["cfg"], st["kx"], st["pos"]), t["table"].tolist()
    slots = st["slot"].tolist()
    ids = _ints([table[s][x // page] for s, x in zip(st["seq"].tolist(), slots)], torch.int64)
    rows = _ints([x % page for x in slots], torch.int64)
    for h in range(c["nkv"]):
        k[st["layer"], :, h].index_put_((ids, rows), kt[:, h])
        v[st["layer"], :, h].index_put_((ids, rows), st["vx"][:, h].double())
    return _exact_turn(st["cfg"], st["q"], st["pos"]), k, v


def _exact_pages(c, st):
    """The step on host lists, one sequence after the other; rows copied one page at a time."""
    t, page = st["cache"], c["page"]
    table, ln, held, ref = (t[n].tolist() for n in ("table", "len", "held", "ref"))
    k, v = t["k"].clone(), t["v"].clone()
    src, dst, keep = st["src"].tolist(), st["dst"].tolist(), _pages_plan(c)[2]
    for a, b in zip(src, dst):
        ln[b], held[b] = ln[a], _up(ln[a], page)
        for i in range(held[b]):
            table[b][i] = table[a][i]
            ref[table[a][i]] += 1
    free = [p for p in range(len(ref)) if ref[p] == 0]
    for b in dst:
        if ln[b] % page and ref[table[b][ln[b] // page]] > 1:
            old, new = table[b][ln[b] // page], free.pop(0)
            ref[old] -= 1
            ref[new] = 1
            table[b][ln[b] // page] = new
            for pool in (k, v):
                pool[:, new, :, :ln[b] % page] = pool[:, old, :, :ln[b] % page]
        while held[b] < _up(ln[b] + c["grow"], page):
            table[b][held[b]] = free.pop(0)
            ref[table[b][held[b]]] = 1
            held[b] += 1
    for b, rows in zip(dst, keep):
        at = lambda x: (table[b][x // page], x % page)
        for pool in (k, v):
            got = [pool[:, at(ln[b] + r)[0], :, at(ln[b] + r)[1]].clone() for r in rows]
            for i, g in enumerate(got):
                p, r = at(ln[b] + i)
                pool[:, p, :, r] = g
        ln[b] += len(rows)
        while held[b] > _up(ln[b], page):
            held[b] -= 1
            ref[table[b][held[b]]] -= 1
            table[b][held[b]] = -1
    return k, v, _ints(table), _ints(ln), _ints(held), _ints(ref)


def _exact_prompt(c, st):
    g, o, lse = c["nh"] // c["nkv"], torch.empty(st["q"].shape, dtype=torch.float64, device=DEV), \
        torch.empty(st["lse"].shape, dtype=torch.float64, device=DEV)
    cu = st["cu"].tolist()
    for a, b in zip(cu, cu[1:]):
        for h in range(c["nh"]):
            kk, vv = st["k"][a:b, h // g].double(), st["v"][a:b, h // g].double().contiguous()
            for i in range(a, b, 4096):
                e = min(b, i + 4096)
                w = (st["q"][i:e, h].double() * c["D"] ** -0.5) @ kk[:e - a].t().contiguous()
                w[torch.arange(e - a, device=DEV)[None] + a > torch.arange(i, e, device=DEV)[:, None]] = -math.inf
                z = torch.logsumexp(w, 1)
                o[i:e, h] = torch.exp(w - z[:, None]) @ vv[:e - a]
                lse[i:e, h] = z
    return o, lse


def _exact_tree(c, st):
    g, t = c["nh"] // c["nkv"], st["cache"]
    o = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.empty(st["lse"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for s, (ctx, parents) in enumerate(st["plan"]):
        ids = t["table"][s, :_up(ctx + len(parents), c["page"])].long()
        n = len(parents)
        sees = torch.zeros(n, ctx + n, dtype=torch.bool, device=DEV)
        sees[:, :ctx] = True
        up = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            j = i
            while j >= 0:
                up[i, j] = True
                j = parents[j]
        sees[:, ctx:] = up.to(DEV)
        for h in range(c["nkv"]):
            kk, vv = (t[x][0, ids, h].flatten(0, 1)[:ctx + n].double() for x in ("k", "v"))
            for u in range(h * g, (h + 1) * g):
                w = st["q"][row:row + n, u].double() @ kk.t().contiguous() * c["D"] ** -0.5
                w[~sees] = -math.inf
                z = torch.logsumexp(w, 1)
                o[row:row + n, u] = torch.exp(w - z[:, None]) @ vv
                lse[row:row + n, u] = z
        row += n
    return o, lse


_exact = {"rope": _exact_rope, "rope_kv": _exact_rope_kv, "pages": _exact_pages, "prompt": _exact_prompt, "tree": _exact_tree}
