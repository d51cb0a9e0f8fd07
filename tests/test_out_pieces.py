"""Results that leave through a warp's two pieces of shared memory: no piece is written while a copy may read it,
whatever products follow one another.  The bookkeeping is the kernel's own header, compiled for the host; the
copies are those of a model that lets each finish as late as the waits allow."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# every sequence of eight results; p: a part of a sum (both pieces), k: a result and what it was before the activation
# (both), a, b: the first and second half of a tile with an addend, r: any other result, s: a sum kept without a copy
MODEL = r"""
#include "treebeard_b200/csrc/out_pieces.h"
#include <cstdio>
#include <cstring>
int main() {
  const char kinds[] = "pkabrs";
  long waits = 0, all = 0;
  for (long code = 0; code < 1679616; ++code) {   // 6^8
    tb::OutPieces out{0};
    unsigned under_way[2] = {0, 0};                   // read by the newest copy and the one before it
    long c = code;
    for (int i = 0; i < 8; ++i, c /= 6) {
      const char k = kinds[c % 6];
      const unsigned pieces = k == 'p' || k == 'k' || k == 's' ? 3 : k == 'a' ? 1 : k == 'b' ? 2 : out.other();
      const unsigned may = out.claim(pieces);
      if (k == 's') out.read = 0;
      if (may > 1) return 1;
      under_way[1] = 0;                               // all but the newest `may` copies have ended
      if (!may) under_way[0] = 0, ++waits;
      ++all;
      if (pieces & (under_way[0] | under_way[1])) return printf("written while read: code %ld at %d\n", code, i), 1;
      if (k != 's') under_way[1] = under_way[0], under_way[0] = pieces;
      else if (under_way[0]) return printf("kept sums over a copy: code %ld at %d\n", code, i), 1;
    }
  }
  // a product of plain results never waits for the copy before
  tb::OutPieces out{0};
  for (int i = 0; i < 100; ++i)
    if (!out.claim(out.other())) return 2;
  return 0;
}
"""


def test_no_piece_is_written_while_it_is_copied_out(tmp_path):
    (tmp_path / "model.cpp").write_text(MODEL)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", ROOT, "-o", str(tmp_path / "model"), str(tmp_path / "model.cpp")], check=True)
    done = subprocess.run([str(tmp_path / "model")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_the_kernels_ask_before_they_write():
    """Every wait for copies out of a warp's pieces goes through that bookkeeping."""
    text = open(os.path.join(ROOT, "treebeard_b200", "csrc", "dense.cuh")).read()
    body = text.split("void out_claim(", 1)
    assert "out_free<" not in body[0].split("void out_free()")[0]
    inside, after = body[1].split("\n}\n", 1)
    assert inside.count("out_free<") == 2 and "out_free<" not in after


def test_only_the_leaf_map_is_read_as_constant():
    """Kernels that are resident while their predecessor runs read its results by plain loads."""
    csrc = os.path.join(ROOT, "treebeard_b200", "csrc")
    for name in ("leaf_sum.cuh", "dense.cuh", "element.cuh"):
        code = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        assert "ld.global.nc" not in code and "__restrict__" not in code
        assert not [a for a in re.findall(r"__ldg\(([^;]*)", code) if not re.match(r"(m\.(trees|rows)|words) \+", a)]


def test_addresses_between_elements_are_refused():
    """On the host, before any launch: such a read would end the program."""
    torch = pytest.importorskip("torch")    # (the binding's)
    from treebeard_b200 import leaf_model as lm
    L, p = lm.lib(), 1 << 20
    names = "x w bias res out pre".split()

    def linear(**odd):
        a = {n: p + odd.get(n, 0) for n in names}
        return L.tbk_linear(a["x"], 8, a["w"], 8, a["bias"], 0, a["res"], 4, a["out"], 4, a["pre"], 4, 4, 8, 4, 2, None, 0, 0, None)
    for name in names:
        assert linear(**{name: 1}) == 1 and b"multiple" in L.tbk_last_error(), name

    def back(g=0, x=0, w=0, pre=0, skip=0, gx=0, gw=0, gb=0):
        return L.tbk_linear_backward(p + g, 4, p + x, 8, p + w, 8, p + pre, 4, 2, p + skip, 8, p + gx, 8, p + gw, 8, p + gb, 4, 8, 4, 1, p, 1 << 40, 0, None)
    for name in "g x w pre skip gx gw gb".split():
        assert back(**{name: 1}) == 1 and b"multiple" in L.tbk_last_error(), name

    def loss(x=0, w=0, bias=0, labels=0, loss=0, lse=0):
        return L.tbk_class_loss(p + x, 8, p + w, 8, p + bias, p + labels, 8, p + loss, p + lse, 4, 8, 100, 1, p, 1 << 40, 0, None)
    for name, by in (("x", 1), ("w", 1), ("bias", 1), ("labels", 4), ("loss", 2), ("lse", 2)):
        assert loss(**{name: by}) == 1 and b"multiple" in L.tbk_last_error(), name

    def loss_back(g=0, x=0, w=0, bias=0, labels=0, lse=0, gx=0, gw=0, gb=0):
        return L.tbk_class_loss_backward(p + g, p + x, 8, p + w, 8, p + bias, p + labels, 4, p + lse, p + gx, 8, p + gw, 8, p + gb, 4, 8, 100, 1, p, 1 << 40, 0, None)
    for name, by in (("g", 2), ("x", 1), ("w", 1), ("bias", 1), ("labels", 2), ("lse", 2), ("gx", 1), ("gw", 1), ("gb", 1)):
        assert loss_back(**{name: by}) == 1 and b"multiple" in L.tbk_last_error(), name
