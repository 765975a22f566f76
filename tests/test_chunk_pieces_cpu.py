"""How the attention of chunks counts the pieces of a row block's keys, compiled for the host."""
from __future__ import annotations

import ctypes
import shutil
import subprocess

import pytest

from tests.conftest import ROOT

PROGRAM = r"""
#include <cmath>
#include "chunk_pieces.hpp"
extern "C" int unit_shift(int max_tokens) { return lb::unit_shift(max_tokens); }
extern "C" int units_of(int keys, int shift) { return lb::units_of(keys, shift); }
extern "C" int pieces(int units, int most, int places) {
  float inverse = 1.0f / (float)most;   // the hardware's reciprocal may be one place off
  if (places) inverse = std::nextafterf(inverse, places > 0 ? 2.0f : 0.0f);
  return lb::pieces_in(units, most, inverse);
}
// the first of `count` lengths from `units` on, `step` apart, that is counted wrongly; -1: none.  most <= 0: so many less than the length
extern "C" int wrong(int units, int step, int count, int most, int places) {
  for (int i = 0; i < count; ++i) {
    const int t = units + i * step, m = most > 0 ? most : t + most;
    if (m >= 1 && pieces(t, m, places) != (t + m - 1) / m) return t;
  }
  return -1;
}
"""


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    compiler = shutil.which("g++") or shutil.which("clang++") or shutil.which("amdclang++")
    if compiler is None:
        pytest.skip("no host compiler")
    at = tmp_path_factory.mktemp("pieces")
    (at / "p.cpp").write_text(PROGRAM)
    subprocess.run([compiler, "-O1", "-std=c++17", "-ffp-contract=on", "-shared", "-fPIC", f"-I{ROOT / 'neurova_amd' / 'csrc'}", str(at / "p.cpp"),
                    "-o", str(at / "p.so")], check=True)
    return ctypes.CDLL(str(at / "p.so"))


MOST = 1 << 20


def test_units_of_every_table(pieces):
    """A tile, and more only where the table would have more than 2^20 of them; tables have 2^28 tokens at most."""
    for tokens in (0, 1, 64, 65, 131072, MOST * 64 - 1, MOST * 64):
        assert pieces.unit_shift(tokens) == 6
    for tokens in (MOST * 64 + 1, 1 << 27, (1 << 27) + 1, (1 << 28) - 16, 1 << 28):
        shift = pieces.unit_shift(tokens)
        assert shift > 6 and pieces.units_of(tokens, shift) <= MOST < pieces.units_of(tokens, shift - 1)
    for keys, shift in ((0, 6), (1, 6), (64, 6), (65, 6), (1 << 28, 8), ((1 << 28) - 255, 8)):
        assert pieces.units_of(keys, shift) == -(-keys >> shift) == -(-keys // (1 << shift))


@pytest.mark.parametrize("places", [-1, 0, 1])
def test_pieces_are_counted_exactly(pieces, places):
    """Whole row blocks, multiples, and one unit more or less, up to the longest that are counted."""
    for less in (0, -1, -2):
        assert pieces.wrong(3, 1, 5000, less, places) == -1
        assert pieces.wrong(MOST // 2, 13, MOST // 26, less, places) == -1
        assert pieces.wrong(MOST - 5000, 1, 5001, less, places) == -1
    for most in (1, 2, 3, 7, 24, 63, 1000, 4097, 65535, 349525, 699051, MOST // 2, MOST - 1, MOST):
        for k in range(1, 40):
            for units in (k * most - 1, k * most, k * most + 1):
                if 1 <= units <= MOST:
                    assert pieces.wrong(units, 0, 1, most, places) == -1, (units, most)
        assert pieces.wrong(MOST - 500 * 2000, 500, 2001, most, places) == -1, most
