"""How the log probabilities' rows are cut into parts, without a GPU."""
import ctypes as C
import subprocess
from pathlib import Path

from cwen_amd import gpu

ROOT = Path(__file__).resolve().parent.parent


def run_c(tmp_path, text):
    src = tmp_path / "t.c"
    src.write_text('#include <limits.h>\n#include <stdio.h>\n#include "logprobs_table.h"\n'
                   '#define CHECK(x) do { if (!(x)) { printf("line %d: %s\\n", __LINE__, #x); return 1; } } while (0)\n' + text)
    for cc in (["gcc", "-std=c11", "-fsanitize=undefined", "-fno-sanitize-recover"], ["g++", "-std=c++17", "-x", "c++"]):
        subprocess.run([*cc, "-O1", "-Wall", "-Wextra", "-Wno-unused-function", f"-I{ROOT / 'cwen_amd' / 'csrc'}", "-o", str(tmp_path / "t"), str(src), "-lm"],
                       check=True)
        r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout + r.stderr


DIVISION = r"""
static int one(int rows, int V, int E) {
  const lp_split s = lp_divide(rows, V, E);
  const int turn = LP_THREADS * LP_LOGITS / E, pieces = V / E, rest = pieces - (s.n - 1) * s.vecs;
  CHECK(s.n >= 1 && s.n <= LP_SPLITS && s.vecs >= 1);
  CHECK(s.n == 1 || (long long)s.n * rows <= LP_WORKGROUPS);      // no second round of workgroups, no join for many rows
  CHECK(s.n == 1 || V >= 2 * 8192);
  if (s.n > 1) {
    CHECK(s.vecs % turn == 0);
    CHECK(rest >= turn / 2);                                     // no part that holds next to nothing,
    CHECK(rest < s.vecs + turn / 2);                             // nor one that holds far more than the others
  }
  return 0;
}
int main(void) {
  static const int some[] = {1, 2, 3, 4, 7, 8, 12, 24, 48, 95, 96, 97, 128, 200, 256, 300, 383, 384, 385, 767, 768, 769, 1500, 4096, (1 << 18) - 1};
  for (int i = 0; i < (int)(sizeof some / sizeof *some); ++i)
    for (int E = 4; E <= 8; E += 4) {
      for (int V = 1; V < 300000; V += 1 + V / 97)
        if (one(some[i], V, E)) { printf("rows %d V %d E %d\n", some[i], V, E); return 1; }
      static const int names[] = {32000, 50257, 128256, 151936, 201088, 248320, 262144, 1 << 20, (1 << 30) - 1, 1 << 30};
      for (int j = 0; j < (int)(sizeof names / sizeof *names); ++j)
        if (one(some[i], names[j], E)) { printf("rows %d V %d E %d\n", some[i], names[j], E); return 1; }
    }
  for (int rows = 1; rows < 1600; ++rows)
    for (int E = 4; E <= 8; E += 4)
      if (one(rows, 151936, E) || one(rows, 248320, E)) { printf("rows %d E %d\n", rows, E); return 1; }
  return 0;
}
"""


def test_division_of_rows(tmp_path):
    run_c(tmp_path, DIVISION)


def test_many_rows_need_no_scratch():
    """Whatever the vocabulary: rows that fill the card have one part each."""
    n = C.c_size_t()
    for V in (6000, 13000, 50257, 128256, 151936, 201088, 248320, 262144):
        for rows in (385, 768, 1500, (1 << 18) - 1):
            assert gpu.lib().cwen_logprobs_work(rows, V, 20, C.byref(n)) == 0 and n.value == 0, (rows, V, n.value)
        assert gpu.lib().cwen_logprobs_work(1, V, 20, C.byref(n)) == 0 and (n.value > 0) == (V > 16384), (V, n.value)


def test_scratch_that_serves_every_call():
    """The scratch of a call is not less for fewer rows; the stated maximum covers all of them."""
    n, most = C.c_size_t(), 0
    for rows in [*range(1, 400), 500, 768, 769, 1500]:
        for V in (1, 8192, 16384, 20000, 50257, 128256, 151936, 201088, 248320, 262144, 1 << 24, 1 << 30):
            for top in (0, 1, 2, 5, 20, 63, 64):
                assert gpu.lib().cwen_logprobs_work(rows, V, top, C.byref(n)) == 0
                assert n.value <= 768 * (16 + 8 * (top + 1)) and n.value <= gpu.LOGPROBS_WORK_MAX, (rows, V, top, n.value)
                most = max(most, n.value)
    assert most == gpu.LOGPROBS_WORK_MAX
    header = (ROOT / "include" / "cwen_gpu.h").read_text()
    assert "#define CWEN_LOGPROBS_WORK_MAX (768 * (16 + 8 * CWEN_LOGPROBS_TOP))" in header


PLACES = r"""
#include <math.h>
#include <string.h>
static float f(unsigned b) { float x; memcpy(&x, &b, 4); return x; }
int main(void) {
  static const int toks[] = {INT_MIN, INT_MIN + 1, -9, -1, 0, 1, 2, 3, 4, 7, 8, 9, 4095, 4096, (1 << 30) - 1, 1 << 30, INT_MAX - 1, INT_MAX};
  for (int i = 0; i < (int)(sizeof toks / sizeof *toks); ++i)
    for (int E = 4; E <= 8; E += 4)
      for (int head = 0; head < E; ++head) {
        const int p = lp_piece(toks[i], head, E);
        CHECK((p >= 0) == (toks[i] >= head));
        CHECK(p < 0 || ((long long)p * E + head <= toks[i] && toks[i] < ((long long)p + 1) * E + head));
      }
  static const unsigned bits[] = {0, 0x80000000u, 1, 0x80000001u, 0x80000002u, 0x007fffff, 0x00800000, 0x3f800000, 0xbf800000u, 0x7f7fffff, 0xff7fffffu, 0xff800000u};
  for (int i = 0; i < (int)(sizeof bits / sizeof *bits); ++i) CHECK(f(lp_above(bits[i])) == nextafterf(f(bits[i]), INFINITY));
  static const unsigned none[] = {0x7f800000, 0x7fc00000, 0x7fffffff, 0xffc00000u, 0xffffffffu};      /* +inf and NaN: any bits, no overflow */
  for (int i = 0; i < (int)(sizeof none / sizeof *none); ++i) CHECK(lp_above(none[i]) != none[i]);
  return 0;
}
"""


def test_places_of_tokens(tmp_path):
    """Any int as a token, any bits as its logit, without an overflow."""
    run_c(tmp_path, PLACES)
