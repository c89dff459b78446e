"""The serving operators of the GatedDeltaNet layers and the log probabilities
without a GPU: refusals of every entry point, and the arithmetic of packed
sequences and slots on bad state."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from cwen_amd import gpu

ROOT = Path(__file__).resolve().parent.parent
EINVAL, ETYPE, ESCRATCH, OK = -1, -4, -5, 0
F32, F16, BF16 = gpu.T_F32, gpu.T_F16, gpu.T_BF16


class FakeCtx(C.Structure):
    """Never dereferenced by a call that refuses its arguments."""
    _fields_ = [("pad", C.c_char * 256)]


CTX = C.addressof(FakeCtx())
_keep = C.create_string_buffer(1 << 17)
P = (C.addressof(_keep) + 4095) & ~4095      # an aligned address; no call below reaches the GPU


def pool(**change):
    c = gpu.GdnPoolC(2, 8, 2, 4, 64, 0, P, P, P)
    for n, v in change.items():
        setattr(c, n, v)
    return C.byref(c)


CH = (2 * 2 + 4) * 64                         # channels of that pool


def conv(c=None, ctx=CTX, layer=0, xt=BF16, x=P, xs=CH, kw=P, yt=BF16, y=P + 32768, ys=CH, cu=P, count=None, src=P, dst=P, n=1, total=2):
    return gpu.lib().cwen_gdn_conv(ctx, c or pool(), layer, xt, x, xs, kw, yt, y, ys, cu, count, src, dst, n, total, None)


def rule(name, c=None, ctx=CTX, layer=0, xt=BF16, q=P, qs=CH, k=P + 256, ks=CH, v=P + 512, vs=CH, a=P, b=P, gs=4, A=P, dt=P, ot=BF16,
         o=P + 32768, os=256, cu=P, count=None, src=P, dst=P, n=1, total=2, work=P, wb=1 << 60):
    args = [ctx, c or pool(), layer, xt, q, qs, k, ks, v, vs, a, b, gs, A, dt, ot, o, os, cu, count, src, dst, n, total]
    if name == "step":
        return gpu.lib().cwen_gdn_step(*args, None)
    return gpu.lib().cwen_gdn_prompt(*args, work, wb, None)


BAD_POOL = [dict(n_layers=0), dict(n_layers=32768), dict(n_slots=0), dict(n_slots=65537), dict(nkh=0), dict(nvh=0), dict(nvh=5), dict(nvh=4098),
            dict(dk=32), dict(dk=96), dict(dk=256), dict(key_head=2), dict(key_head=-1), dict(state=P + 8), dict(hist=P + 4), dict(status=None),
            dict(status=P + 2)]


@pytest.mark.parametrize("bad", BAD_POOL, ids=lambda d: "-".join(map(str, d.items())))
def test_pool_refusals(bad):
    assert conv(pool(**bad)) == EINVAL
    assert rule("step", pool(**bad)) == EINVAL and rule("prompt", pool(**bad)) == EINVAL
    n = C.c_size_t(7)
    assert gpu.lib().cwen_gdn_prompt_work(pool(**bad), F16, F16, 1, 5, C.byref(n)) == EINVAL and n.value == 0
    assert gpu.lib().cwen_gdn_status(CTX, pool(**bad), C.byref(C.c_int()), None) == EINVAL


SEQS = [dict(ctx=None), dict(layer=-1), dict(layer=2), dict(n=-1), dict(n=gpu.GDN_SEQ_MAX + 1), dict(total=-1), dict(total=1 << 30),
        dict(cu=None), dict(cu=P + 2), dict(count=P + 1), dict(src=P + 2), dict(dst=P + 3)]


def test_conv_refusals():
    assert conv(n=0) == OK and conv(n=0, cu=None, total=0, x=None, y=None) == OK
    assert conv(xt=3) == ETYPE and conv(yt=101) == ETYPE
    for bad in SEQS + [dict(x=None), dict(x=P + 8), dict(xs=CH - 8), dict(xs=CH + 4), dict(kw=None), dict(kw=P + 4), dict(y=P + 32768 + 4),
                       dict(ys=CH - 8), dict(ys=CH + 2), dict(y=P), dict(y=P + 2 * CH), dict(c=pool(hist=None)), dict(y=P + CH, ys=2 * CH, xs=2 * CH),
                       dict(y=P, yt=F32)]:
        assert conv(**bad) == EINVAL, bad


def test_rule_refusals():
    for name in ("step", "prompt"):
        f = lambda **kw: rule(name, **kw)
        assert f(n=0) == OK and f(n=0, total=0, q=None, k=None, v=None, a=None, b=None, o=None, cu=None) == OK
        assert f(xt=2) == ETYPE and f(ot=14) == ETYPE
        for bad in SEQS + [dict(q=None), dict(k=None), dict(v=None), dict(a=None), dict(b=None), dict(a=P + 2), dict(b=P + 1), dict(gs=3),
                           dict(A=None), dict(dt=None), dict(A=P + 2), dict(dt=P + 1), dict(q=P + 8), dict(k=P + 4), dict(v=P + 2), dict(qs=120),
                           dict(qs=CH + 4), dict(ks=124), dict(vs=248), dict(o=P + 32768 + 8), dict(os=248), dict(os=260), dict(o=P),
                           dict(o=P + 256), dict(o=P + 512), dict(o=P + 768, os=CH), dict(c=pool(state=None))]:
            assert f(**bad) == EINVAL, (name, bad)
        # what one call of either could do, refused for its scratch only
    n = C.c_size_t()
    assert gpu.lib().cwen_gdn_prompt_work(pool(), BF16, BF16, 1, 40, C.byref(n)) == OK
    if n.value:
        assert rule("prompt", o=None, total=40, wb=n.value - 1) == ESCRATCH
        assert rule("prompt", o=None, total=40, work=None) == EINVAL and rule("prompt", o=None, total=40, work=P + 64) == EINVAL
    assert rule("prompt", c=pool(nvh=4096, nkh=1), vs=4096 * 64, os=4096 * 64, gs=4096, qs=4096 * 64, ks=4096 * 64, total=1 << 20,
                q=P, k=P, v=P, o=None) == EINVAL          # chunks times heads past a launch
    L = gpu.lib()
    assert rule("prompt", c=pool(nvh=1024, nkh=1), vs=1024 * 64, os=1024 * 64, gs=1024, o=None, n=4096) == EINVAL       # sequences times heads past one
    assert L.cwen_gdn_prompt_work(pool(), BF16, BF16, 1, 40, None) == EINVAL
    assert L.cwen_gdn_prompt_work(pool(), 3, BF16, 1, 40, C.byref(n)) == ETYPE
    assert L.cwen_gdn_prompt_work(pool(), BF16, BF16, -1, 40, C.byref(n)) == EINVAL
    assert L.cwen_gdn_prompt_work(pool(), BF16, BF16, 1, -1, C.byref(n)) == EINVAL
    assert L.cwen_gdn_prompt_work(pool(), BF16, BF16, 0, 0, C.byref(n)) == OK and n.value == 0
    assert L.cwen_gdn_status(CTX, pool(), None, None) == EINVAL and L.cwen_gdn_status(None, pool(), C.byref(C.c_int()), None) == EINVAL


def test_logprobs_refusals():
    L = gpu.lib()

    def f(ctx=CTX, t=F32, x=P, ls=100, V=100, rows=2, tok=P, lp=P, rank=P, H=P, lse=P, top=5, ids=P, tlp=P, work=P, wb=1 << 40):
        return L.cwen_logprobs(ctx, t, x, ls, V, rows, tok, lp, rank, H, lse, top, ids, tlp, work, wb, None)
    assert f(rows=0) == OK and f(t=2) == ETYPE
    for bad in (dict(ctx=None), dict(x=None), dict(x=P + 2), dict(ls=99), dict(V=0), dict(V=(1 << 30) + 1), dict(rows=-1), dict(rows=1 << 18),
                dict(tok=None), dict(tok=None, lp=None), dict(tok=P + 2), dict(lp=P + 1), dict(rank=P + 2), dict(H=P + 2), dict(lse=P + 3),
                dict(top=-1), dict(top=65), dict(ids=P + 2), dict(tlp=P + 2), dict(x=P + 1, t=BF16)):
        assert f(**bad) == EINVAL, bad
    n = C.c_size_t()
    assert L.cwen_logprobs_work(1, 248320, 20, C.byref(n)) == OK and n.value > 0
    big = dict(rows=1, V=248320, ls=248320, top=20)
    assert f(**big, wb=n.value - 1) == ESCRATCH
    assert f(**big, work=None) == EINVAL and f(**big, work=P + 8) == EINVAL
    assert L.cwen_logprobs_work(0, 10, 0, C.byref(n)) == OK and n.value == 0
    for a in ((-1, 10, 0), (1, 0, 0), (1, 10, 65), (1, 10, -1)):
        assert L.cwen_logprobs_work(*a, C.byref(n)) == EINVAL
    assert L.cwen_logprobs_work(1, 10, 0, None) == EINVAL
    for V in list(range(1, 70)) + [4095, 4096, 4097, 8191, 8192, 248320, 1 << 30]:      # every size has a division
        for rows in (1, 2, 96, 1500, (1 << 18) - 1):
            assert L.cwen_logprobs_work(rows, V, 64, C.byref(n)) == OK
            assert n.value <= rows * 64 * (4 + 128) * 4 and (n.value > 0) == (rows <= 96 and V > 12000), (rows, V, n.value)


PROG = r"""
#include <stdio.h>
#include <limits.h>
#include "gdn_table.h"
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main(void) {
  static const int odd[] = {INT_MIN, INT_MIN + 1, -7, -1, 0, 1, 2, 31, 32, 33, 99, 100, 101, INT_MAX - 1, INT_MAX};
  const int n = sizeof odd / sizeof odd[0];
  for (int i = 0; i < n; ++i) {
    const int b = gdn_border(odd[i], 100);
    CHECK(b >= 0 && b <= 100);
    for (int j = 0; j < n; ++j) {
      const int e = gdn_border(odd[j], 100), r = gdn_rows(b, e);
      CHECK(r >= 0 && b + r <= 100 && (e < b || b + r == e));
      CHECK(gdn_count_ok(odd[i], r) == (odd[i] >= 0 && odd[i] <= r));
    }
    CHECK(gdn_slot_ok(odd[i], 33) == (odd[i] >= -1 && odd[i] < 33));
    CHECK(!gdn_clash(-1, odd[i], odd[i]));
    CHECK(gdn_clash(5, odd[i], 5) && gdn_clash(5, 5, odd[i]) && !gdn_clash(5, 4, -1));
  }
  // the pieces of all sequences are apart and below gdn_pieces, whatever their lengths
  for (int N = 1; N <= 32; N += 31)
    for (unsigned seed = 1; seed < 400; ++seed) {
      unsigned x = seed;
      int first = 0, next = 0, S = 1 + seed % 9;
      for (int s = 0; s < S; ++s) {
        x = x * 1664525u + 1013904223u;
        const int rows = (x >> 8) % (seed % 3 ? 70 : 2), p0 = gdn_piece0(first, s, N);
        CHECK(p0 >= next);
        next = p0 + (rows + N - 1) / N;
        first += rows;
        CHECK(next <= gdn_piece0(first, s + 1, N));
      }
      CHECK(next <= gdn_pieces(first, S, N));
    }
  CHECK(gdn_pieces(INT_MAX, 65536, 1) == (long long)INT_MAX + 65536);
  return 0;
}
"""


def test_sequence_arithmetic(tmp_path):
    src = tmp_path / "t.c"
    src.write_text(PROG)
    for cc in (["gcc", "-std=c11", "-fsanitize=undefined", "-fno-sanitize-recover"], ["g++", "-std=c++17", "-x", "c++"]):
        subprocess.run([*cc, "-Wall", "-Wextra", "-Wno-unused-function", f"-I{ROOT / 'cwen_amd' / 'csrc'}", "-o", str(tmp_path / "t"), str(src)],
                       check=True)
        r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout + r.stderr
