"""Refusals of the windowed operator, and which key tiles its rows visit; neither needs a GPU."""
import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash_attn_with_score_b200", "csrc")


@pytest.fixture(scope="module")
def lib():
    from flash_attn_with_score_b200 import build, _lib
    build.build()
    return _lib.load()


def _problem(**over):
    from flash_attn_with_score_b200 import _lib
    t = lambda: _lib.Tensor(4096, 4 * 128 * 64, 128 * 64, 64)
    f = dict(B=1, Hq=4, Hk=4, M=128, N=128, D=64, causal=1, sm_scale=1.0, m_end=128, q=t(), k=t(), v=t(), out=t())
    f.update(over)
    return _lib.Problem(**f)


def test_refusals(lib):
    from flash_attn_with_score_b200 import _lib
    none = _lib.Tensor(None, 1, 1, 1)
    call = lambda p, window=5, sinks=0, splits=1, ws=None, n=0: lib.faws_attention_with_window(C.byref(p), window, sinks, splits, ws, n, None)
    for p, kw, status in [(_problem(), dict(window=0), -1), (_problem(), dict(sinks=-1), -1), (_problem(causal=0), {}, -1),
                          (_problem(m_begin=1), {}, -1), (_problem(m_end=64), {}, -1), (_problem(dropout_p=0.5), {}, -2),
                          (_problem(D=48), {}, -2), (_problem(Hq=3), {}, -1), (_problem(out=none), {}, -1), (_problem(v=none), {}, -1),
                          (_problem(), dict(splits=0), -1), (_problem(), dict(splits=2), -1),
                          (_problem(N=1024), dict(splits=2), -3), (_problem(N=1024), dict(splits=2, ws=4100, n=1 << 30), -3),
                          (_problem(N=1024), dict(splits=2, ws=4096, n=100), -3)]:
        assert call(p, **kw) == status, (kw, status)
    assert lib.faws_attention_with_window(None, 5, 0, 1, None, 0, None) == -1
    g = _lib.Grads(_lib.Tensor(4096, 1, 1, 1), _lib.Tensor(4096, 1, 1, 1), _lib.Tensor(4096, 1, 1, 1), _lib.Tensor(4096, 1, 1, 1))
    back = lambda p, g=g, window=5, sinks=0: lib.faws_attention_with_window_backward(C.byref(p), C.byref(g), window, sinks, 4096, 1 << 30, None)
    assert back(_problem(), window=0) == -1 and back(_problem(), sinks=-1) == -1 and back(_problem(causal=0)) == -1
    assert back(_problem()) == -1  # no log-normaliser
    assert lib.faws_window_split_plan(C.byref(_problem(M=0)), 5, 0) == 1


PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include "faws_launch_plan.h"
using namespace faws;
int main() {
  long checked = 0;
  for (int M : {1, 5, 128, 129, 300, 700})
    for (int N : {1, 4, 127, 128, 300, 700, 1000})
      for (int window : {1, 2, 64, 127, 128, 129, 500, 1 << 30})
        for (int sinks : {0, 1, 4, 128, 129, 400, 1 << 30})
          for (int rows : {128, 256})
            for (int r = 0; r < M; r += rows) {
              const int end = std::min(M, r + rows), p_seq = N - M;
              std::set<int> want;
              for (int i = r; i < end; ++i)
                for (int j = 0; j < N && j <= i + p_seq; ++j)
                  if (j > i + p_seq - window || j < sinks) want.insert(j / 128);
              const KeyTiles t = key_tiles(r, end, p_seq, N, window, sinks);
              std::set<int> got;
              int last = -1;
              for (int it = 0; it < t.count(); ++it) {
                if (t.tile(it) <= last) return printf("not ascending\n"), 1;
                last = t.tile(it);
                got.insert(last);
              }
              for (int x : want)
                if (!got.count(x)) return printf("M %d N %d w %d s %d r %d: tile %d missing\n", M, N, window, sinks, r, x), 1;
              // beyond what is seen: at most what lies between windows of a row block's rows
              if (!got.empty() && (want.empty() || *got.rbegin() > *want.rbegin())) return printf("a tile too many\n"), 1;
              if (got.size() > want.size() + 1) return printf("M %d N %d w %d s %d r %d: %zu tiles, %zu wanted\n", M, N, window, sinks, r, got.size(), want.size()), 1;
              ++checked;
            }
  printf("%ld\n", checked);
  return 0;
}
"""


def test_visited_key_tiles(tmp_path):
    src, exe = str(tmp_path / "tiles.cpp"), str(tmp_path / "tiles")
    with open(src, "w") as f:
        f.write(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, "-o", exe, src], check=True)
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout
    assert int(got.stdout) > 5000
