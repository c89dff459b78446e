"""The serving operators without a GPU: refusals of every entry point, rotary
configurations, and the cache's page arithmetic on bad state."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from cwen_amd import gpu

ROOT = Path(__file__).resolve().parent.parent
EINVAL, ETYPE, OK = -1, -4, 0


class FakeCtx(C.Structure):
    """Never dereferenced by a call that refuses its arguments."""
    _fields_ = [("pad", C.c_char * 256)]


CTX = C.addressof(FakeCtx())
_keep = C.create_string_buffer(1 << 16)
P = (C.addressof(_keep) + 4095) & ~4095      # an aligned address; no call below reaches the GPU


def kv(**change):
    c = gpu.KvCache(gpu.T_F16, 2, 4, 128, 16, 64, 8, 32, P, P, P, P, P, P, P, P)
    for n, v in change.items():
        setattr(c, n, v)
    return C.byref(c)


BAD_KV = [dict(type=gpu.T_F32), dict(n_layers=0), dict(n_kv_head=0), dict(head_dim=12), dict(head_dim=520), dict(page=24), dict(page=8),
          dict(page=512), dict(n_pages=0), dict(n_pages=(1 << 24) + 1), dict(max_seqs=0), dict(max_seqs=65537), dict(max_pages=0),
          dict(max_pages=1 << 26), dict(k=None), dict(v=P + 8), dict(table=None), dict(len=None), dict(held=None), dict(ref=P + 4),
          dict(work=None), dict(status=None), dict(table=P + 2)]


@pytest.mark.parametrize("bad", BAD_KV, ids=lambda d: "-".join(map(str, d.items())))
def test_cache_refusals(bad):
    L, c = gpu.lib(), kv(**bad)
    want = ETYPE if "type" in bad else EINVAL
    assert L.cwen_kv_reset(CTX, c, None) == want
    assert L.cwen_kv_reserve(CTX, c, P, P, 1, None) == want
    assert L.cwen_kv_fork(CTX, c, P, P, 1, None) == want
    assert L.cwen_kv_keep(CTX, c, P, P, None, 0, 1, None) == want
    assert L.cwen_kv_truncate(CTX, c, P, None, 1, None) == want
    assert L.cwen_kv_status(CTX, c, C.byref(C.c_int()), None) == want
    assert L.cwen_attn_tree(CTX, c, 0, P, 512, P + 2048, 512, None, P, P, None, 0, 1, 1, 1, 1, 4, 1.0, None) == want


def test_request_refusals():
    L = gpu.lib()
    for f in (lambda a, b, n: L.cwen_kv_reserve(CTX, kv(), a, b, n, None), lambda a, b, n: L.cwen_kv_fork(CTX, kv(), a, b, n, None),
              lambda a, b, n: L.cwen_kv_keep(CTX, kv(), a, b, None, 0, n, None)):
        assert f(P, P, -1) == EINVAL and f(None, P, 1) == EINVAL and f(P, None, 1) == EINVAL and f(P + 2, P, 1) == EINVAL
        assert f(P, P, 9) == EINVAL                       # more requests than sequences
        assert f(None, None, 0) == OK
    big = kv(max_seqs=65536)
    assert L.cwen_kv_reserve(CTX, big, P, P, gpu.KV_REQ_MAX + 1, None) == EINVAL
    assert L.cwen_kv_truncate(CTX, kv(), None, None, 1, None) == EINVAL
    assert L.cwen_kv_truncate(CTX, kv(), None, None, 0, None) == OK
    assert L.cwen_kv_keep(CTX, kv(), P, P, P, 0, 1, None) == EINVAL
    assert L.cwen_kv_reserve(None, kv(), P, P, 1, None) == EINVAL
    assert L.cwen_kv_reserve(CTX, None, P, P, 1, None) == EINVAL
    assert L.cwen_kv_status(CTX, kv(), None, None) == EINVAL


GOOD = dict(head_dim=128, n_rot=64, theta=1e4)


@pytest.mark.parametrize("bad", [dict(head_dim=0), dict(head_dim=12), dict(head_dim=520), dict(n_rot=0), dict(n_rot=136), dict(n_rot=4),
                                 dict(n_rot=8, layout="halves"), dict(theta=1.0), dict(theta=float("inf")), dict(theta=float("nan")),
                                 dict(mscale=-1.0), dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0),
                                 dict(scaling="yarn", factor=2.0, orig_ctx=4096, beta_fast=1.0, beta_slow=2.0),
                                 dict(scaling="yarn", factor=2.0, orig_ctx=4096, beta_slow=0.0), dict(freq_dim=-1)],
                         ids=lambda d: "-".join(map(str, d.items())))
def test_rope_config_refusals(bad):
    with pytest.raises(gpu.CwenError) as e:
        gpu.Rope(**{**GOOD, **bad})
    assert e.value.rc == EINVAL


def test_rope_call_refusals():
    L, r = gpu.lib(), gpu.Rope(128, 64)
    f32, f16 = gpu.T_F32, gpu.T_F16

    def call(x=P, xts=512, xhs=128, xt=f32, y=P + 16384, yts=512, yhs=128, yt=f16, pos=P, T=2, nh=4, ctx=CTX, h=r.h):
        return L.cwen_rope_apply(ctx, h, xt, x, xts, xhs, yt, y, yts, yhs, pos, T, nh, 0, None)
    assert call(T=0) == OK and call(x=None, T=0) == OK
    assert call(xt=3) == ETYPE and call(yt=8) == ETYPE
    for bad in (dict(ctx=None), dict(h=None), dict(T=-1), dict(nh=0), dict(x=None), dict(y=None), dict(pos=None), dict(x=P + 8),
                dict(y=P + 4), dict(xts=508), dict(xhs=-128), dict(yts=12), dict(yts=0), dict(yhs=64), dict(yts=256, yhs=128),
                dict(y=P + 1024), dict(y=P), dict(y=P, yt=f32, yts=1024), dict(pos=P + 1)):
        assert call(**bad) == EINVAL, bad

    def fused(q=P, qs=512, k=P + 8192, ks=512, v=P + 16384, vs=512, o=P + 24576, os=512, c=None, layer=1, T=2, nh=4, xt=f32, idx=P):
        return L.cwen_rope_kv(CTX, r.h, xt, q, qs, k, ks, v, vs, o, os, c or kv(), layer, idx, idx, idx, T, nh, None)
    assert fused(T=0) == OK and fused(xt=2) == ETYPE
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(q=P + 8), dict(qs=504), dict(qs=256), dict(ks=256), dict(vs=12),
                dict(os=128), dict(layer=2), dict(layer=-1), dict(c=kv(head_dim=64)), dict(T=-1), dict(nh=0), dict(idx=None), dict(o=P + 64),
                dict(o=P + 8192)):
        assert fused(**bad) == EINVAL, bad


def test_rope_kv_in_place_refusals():
    """q in place: k and v beside it in the rows of one product, never under its heads."""
    L, r = gpu.lib(), gpu.Rope(128, 64)

    def call(k, v, qs=512 + 1152, T=2, xt=gpu.T_F16, ks=None):
        return L.cwen_rope_kv(CTX, r.h, xt, P, qs, k, ks or qs, v, qs, P, qs, kv(), 0, P, P, P, T, 4, None)
    for k, v in ((P + 1024 - 16, P + 2048), (P + 1024, P + 2304 + 16), (P + 512, P + 2048), (P + 1024, P), (P + 1024, P + 3328 - 16),
                 (P + 3328 + 512, P + 2048), (P - 16, P + 2048)):
        assert call(k, v) == EINVAL, (k - P, v - P)
    assert call(P + 1024, P + 2048, ks=1024) == EINVAL
    assert call(P + 1024 - 16, P + 2048, T=1) == EINVAL
    assert call(P + 1024, P + 2048, T=1 << 24) == EINVAL
    assert L.cwen_rope_apply(CTX, r.h, gpu.T_F16, P, 512, 128, gpu.T_F16, P, 512, 128, P, 1 << 24, 4, 0, None) == EINVAL
    assert L.cwen_kv_reset(CTX, kv(max_seqs=65536, max_pages=32768), None) == EINVAL      # 2^31 table entries


def test_attention_refusals():
    L = gpu.lib()

    def prompt(t=gpu.T_BF16, q=P, qs=512, k=P + 8192, ks=256, v=P + 16384, vs=256, o=P + 24576, os=512, cu=P, n=1, tq=2, tk=2, nh=4,
               nkv=2, D=128, scale=1.0, cuk=P, ctx=CTX, lse=None):
        return L.cwen_attn_prompt(ctx, t, q, qs, k, ks, v, vs, o, os, lse, cu, cuk, n, tq, tk, nh, nkv, D, scale, None)
    assert prompt(n=0) == OK and prompt(tq=0) == OK and prompt(t=gpu.T_F32) == ETYPE
    for bad in (dict(ctx=None), dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(cu=None), dict(q=P + 2), dict(qs=504),
                dict(ks=128), dict(vs=260), dict(os=256), dict(nh=3), dict(nkv=0), dict(D=96), dict(D=512), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(n=-1), dict(tq=-1), dict(tk=1 << 30),
                dict(cuk=None, tk=3), dict(o=P), dict(o=P + 8192), dict(o=P + 16384), dict(cu=P + 2), dict(lse=P + 1), dict(n=65537),
                dict(ks=1 << 27), dict(vs=1 << 27)):
        assert prompt(**bad) == EINVAL, bad

    def tree(c=None, layer=0, q=P, qs=512, o=P + 8192, os=512, seqs=P, cu=P, mask=P, mw=1, n=1, total=2, mn=2, ml=5, nh=4, scale=1.0):
        return L.cwen_attn_tree(CTX, c or kv(), layer, q, qs, o, os, None, seqs, cu, mask, mw, n, total, mn, ml, nh, scale, None)
    assert tree(n=0) == OK and tree(total=0) == OK and tree(mn=0) == OK
    for bad in (dict(c=kv(head_dim=96)), dict(layer=2), dict(layer=-1), dict(q=None), dict(o=None), dict(seqs=None), dict(cu=None),
                dict(mask=P + 4), dict(mw=0), dict(mw=5), dict(mn=65), dict(mn=257, mask=None), dict(mn=-1), dict(n=9), dict(n=-1),
                dict(total=-1), dict(ml=-1), dict(nh=6), dict(scale=0.0), dict(o=P), dict(qs=256), dict(os=516)):
        assert tree(**bad) == EINVAL, bad


def test_wrapper_checks():
    torch = pytest.importorskip("torch")
    mk = lambda *n, dtype=torch.float16: torch.zeros(n, dtype=dtype)
    with pytest.raises(ValueError):                       # one device for everything, and no GPU here
        gpu.PagedKV(16, mk(1, 4, 2, 16, 64), mk(1, 4, 2, 8, 64), *(torch.zeros(2, dtype=torch.int32),) * 4)
    ints = lambda *n: torch.zeros(n, dtype=torch.int32)
    with pytest.raises(ValueError):
        gpu.PagedKV(16, mk(1, 4, 2, 16, 64), mk(1, 4, 2, 16, 64), ints(2, 3), ints(3), ints(2), ints(4))
    c = gpu.PagedKV(16, mk(1, 4, 2, 16, 64), mk(1, 4, 2, 16, 64), ints(2, 3), ints(2), ints(2), ints(4))
    assert (c.c.n_pages, c.c.max_seqs, c.c.max_pages, c.c.page, c.c.head_dim) == (4, 2, 3, 16, 64)

    class Ctx:
        device, h = 0, None
    with pytest.raises(ValueError):
        c.reserve(Ctx, ints(1), ints(1))                  # host tensors
    for f, a in ((gpu._heads, ("x", mk(3, 4))), (gpu._heads, ("x", mk(4, 3, 64).transpose(0, 1))), (gpu._type, (ints(2),)),
                 (gpu._vec, ("x", ints(3), 2)), (gpu._vec, ("x", ints(4)[::2], 2)), (gpu._vec, ("x", mk(2), 2))):
        with pytest.raises(ValueError):
            f(*a)


def test_wrapper_refuses_paths_without_rows():
    """A path of no rows names nothing; it is not "the first rows stay"."""
    torch = pytest.importorskip("torch")
    pool, ints = torch.zeros(1, 4, 2, 16, 64, dtype=torch.float16), lambda *n: torch.zeros(n, dtype=torch.int32)
    c = gpu.PagedKV(16, pool, pool.clone(), ints(2, 3), ints(2), ints(2), ints(4))

    class Ctx:
        device, h = -1, None                              # where host tensors are
    for path in (ints(1, 0), ints(2, 3), ints(3)):
        with pytest.raises(ValueError):
            c.keep(Ctx, ints(1), ints(1), path, stream=0)


# ---------------------------------------------------------------- page arithmetic on bad state
HARNESS = r"""
#include "kv_table.h"
extern "C" {
int cover(int n, int page) { return kv_cover(n, page); }
int fits(int len, int n, int page, int max_pages) { return kv_fits(len, n, page, max_pages); }
int page_ok(int e, int n, int *bad) { bool b = false; int r = kv_page_ok(e, n, &b); *bad = b; return r; }
int readable(int len, int extra, int held, int page, int max_pages, int *bad) {
  bool b = false; int r = kv_readable(len, extra, held, page, max_pages, &b); *bad = b; return r; }
long long at(int l, int p, int h, int r, int np, int nh, int page, int d) { return kv_at(l, p, h, r, np, nh, page, d); }
}
"""


@pytest.fixture(scope="module")
def pages(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", f"-I{ROOT / 'cwen_amd' / 'csrc'}", str(d / "h.cpp"), "-o", str(d / "h.so")], check=True)
    L = C.CDLL(str(d / "h.so"))
    L.at.restype = C.c_longlong
    return L


def test_page_arithmetic(pages):
    L, bad = pages, C.c_int()
    assert [L.cover(n, 16) for n in (0, 1, 16, 17)] == [0, 1, 1, 2]
    big = 2 ** 31 - 1
    assert L.fits(0, 64, 16, 4) and not L.fits(0, 65, 16, 4) and not L.fits(-1, 1, 16, 4) and not L.fits(1, -1, 16, 4)
    assert not L.fits(big, big, 256, 100)                 # no overflow
    for e in (-1, 7, 100, big, -2 ** 31):
        assert L.page_ok(e, 7, C.byref(bad)) == 0 and bad.value
    assert L.page_ok(6, 7, C.byref(bad)) == 6 and not bad.value
    # a reader never goes past the pages held, whatever the state claims
    for len_, extra, held, want in ((20, 4, 2, 24), (20, 30, 2, 32), (big, 5, 2, 32), (-5, 6, 2, 0), (20, 4, 99, 0), (20, 4, -3, 0), (0, 0, 0, 0)):
        n = L.readable(len_, extra, held, 16, 8, C.byref(bad))
        assert n == want and bool(bad.value) == (n != len_ + extra), (len_, extra, held)
    # offsets past 32 bits
    assert L.at(15, (1 << 24) - 1, 7, 255, 1 << 24, 8, 256, 256) == (((15 * 2 ** 24 + 2 ** 24 - 1) * 8 + 7) * 256 + 255) * 256


BAD_STATE = r"""
#include "kv_table.h"
extern "C" int drafted(int len, int extra, int held, int page, int max_pages) {
  bool b = false;
  const int keys = kv_readable(len, extra, held, page, max_pages, &b);
  return keys - kv_cached(len, keys); }
"""


def harness(tmp_path, source):
    (tmp_path / "h.cpp").write_text(source)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", f"-I{ROOT / 'cwen_amd' / 'csrc'}", str(tmp_path / "h.cpp"), "-o", str(tmp_path / "h.so")],
                   check=True)
    return C.CDLL(str(tmp_path / "h.so"))


def test_drafted_keys_of_bad_lengths(tmp_path):
    """The keys that a tree's masks are read for: as many as the group has nodes at most, and none of a
    sequence whose length is no length."""
    L, big = harness(tmp_path, BAD_STATE), 2 ** 31 - 1
    for extra in (0, 1, 64, 256):
        for held in (-1, 0, 1, 8, 9):
            for len_ in (-2 ** 31, -100000, -1, 0, 1, 15, 16, 127, 128, 129, 100000, big - 256, big):
                n, fits = L.drafted(len_, extra, held, 16, 8), 0 <= held <= 8 and 0 <= len_ and len_ + extra <= 16 * held
                assert 0 <= n <= extra and (n == extra or not fits) and (n == 0 or len_ >= 0), (len_, extra, held, n)


def test_cuts_of_bad_lengths(tmp_path):
    """What a cut leaves is never more than the pages held, nor an index before the first."""
    L = harness(tmp_path, '#include "kv_table.h"\nextern "C" int cut(int to, int cur, int held, int page) { return kv_cut(to, cur, held, page); }')
    some = (-2 ** 31, -1, 0, 1, 16, 17, 64, 65, 2 ** 30, 2 ** 31 - 16, 2 ** 31 - 1)
    for page in (16, 256):
        for held in (0, 1, 4, 2 ** 20):
            for cur in some:
                for to in some:
                    want = -(-to // page) if 0 <= to <= min(cur, held * page) else -1
                    assert L.cut(to, cur, held, page) == want, (to, cur, held, page)


def test_levels_are_taken_for_equal_groups_only(tmp_path):
    """The tree attention gives each row tile a line of its own when the groups' tiles, weighed by their keys,
    add up to as many as equal groups have: no mixture of up to `tiles` may reach that."""
    L = harness(tmp_path, '#include "kv_table.h"\nextern "C" int levels(long long tiles, int pieces) { return tree_levels(tiles, pieces); }')
    L.levels.argtypes = [C.c_longlong, C.c_int]
    for tiles in range(1, 40):
        for pieces in range(1, 40):
            n = L.levels(tiles, pieces)
            assert n == tiles <= pieces or n == 1, (tiles, pieces)
            for a in range(1, tiles + 1):
                for b in range(1, tiles + 1):
                    equal = n > 1 and 3 * a + 5 * b == (3 + 5) * n     # groups of 3 and of 5 units
                    assert not equal or a == b == n
    assert L.levels(2 ** 33, 1024) == 1


@pytest.mark.parametrize("scale,rc", [(3e38, EINVAL), (2.4e38, EINVAL), (1e38, None)])
def test_scales_past_the_powers_of_two(scale, rc):
    """scale * log2(e) has to be a float: with infinity there a score of 0 would be NaN.  (Taken scales
    go on to the device, which is not here; no launch is made without one.)"""
    L = gpu.lib()
    if rc is None and __import__("torch").cuda.is_available():
        pytest.skip("made-up addresses: never where a device would take them")
    got = (L.cwen_attn_prompt(CTX, gpu.T_F16, P, 512, P + 8192, 256, P + 16384, 256, P + 24576, 512, None, P, P, 1, 2, 2, 4, 2, 128, scale, None),
           L.cwen_attn_tree(CTX, kv(), 0, P, 512, P + 8192, 512, None, P, P, None, 0, 1, 2, 2, 5, 4, scale, None))
    assert got == (rc, rc) if rc else EINVAL not in got


@pytest.mark.parametrize("n", [1100, 3001, 9000, 20000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_signatures_show_a_lost_or_wrong_block(n, D):
    """The long-context tests' values: 16 keys left out, taken twice, or read where other 16 lie exceed the bound
    twice (once for the roundings that a right row may have, once to be seen beside them), in bf16 too."""
    torch = pytest.importorskip("torch")
    import serving_ref as R
    level, dims = R.signature(n, D)
    want = R.signature_output(level, dims, D)
    bound = R.signature_bound(want, n, torch.bfloat16)
    seen = lambda other: bool(((other - want).abs() > 2 * bound).any())
    j = torch.arange(n)
    for b in range(0, n - 32, 16 * 7):
        one = (j // 16) == b // 16
        assert seen(R.signature_output(level[~one], dims[~one], D)), ("lost", b)
        assert seen(R.signature_output(torch.cat([level, level[one]]), torch.cat([dims, dims[one]]), D)), ("twice", b)
        for away in (16, 32, 128, 512):                    # values of a block that lies elsewhere
            if b + away + 16 <= n:
                moved = dims.clone()
                moved[one] = dims[b + away:b + away + 16]
                assert seen(R.signature_output(level, moved, D)), ("wrong", b, away)


def test_calls_past_a_launch_are_refused():
    """A launch has less than 2^32 threads: more sequences x heads than that in one call are refused before the device is asked."""
    L = gpu.lib()
    prompt = lambda n, t, nh: L.cwen_attn_prompt(CTX, gpu.T_F16, P, nh * 64, P + (1 << 44), 64, P + (1 << 45), 64, P + (1 << 46), nh * 64, None, P, P, n, t, t,
                                                 nh, 1, 64, 1.0, None)
    big = kv(max_seqs=65536, max_pages=16, n_kv_head=1, head_dim=64)
    tree = lambda t, nh: L.cwen_attn_tree(CTX, big, 0, P, nh * 64, P + (1 << 46), nh * 64, None, P, P, None, 0, 65536, t, 1, 5, nh, 1.0, None)
    for f, n in ((prompt, (65536, 65536, 256)), (prompt, (1, (1 << 30) - 1, 2)), (tree, (1 << 23, 64)), (tree, (1 << 23, 33))):
        assert f(*n) == EINVAL, n
    if not __import__("torch").cuda.is_available():            # taken, and then there is no device
        for f, n in ((prompt, (65536, 128, 255)), (tree, ((1 << 24) - 1, 32))):
            assert f(*n) not in (EINVAL, OK), n
