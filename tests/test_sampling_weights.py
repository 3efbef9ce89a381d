"""The weights of `sample` as whole numbers (csrc/sample_weights.h, compiled for the host) against 2^-y in 80 bits.

A weight is off by half a unit of 2^-f and 2^-38 of itself: the series of 2^-r leaves r^4 / 24 <= 2^-38.7, y in units of 2^-40 another 2^-41.5, the
table, y itself and the products 2^-45 together."""
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_amd", "csrc")
PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "sample_weights.h"
int main(int, char **v) {   // V; y as float64 on the standard input, whole numbers on the standard output
  const int V = std::atoi(v[1]);
  double powers[256];
  for (int j = 0; j < 256; ++j) powers[j] = std::exp2(tamd::fraction_bits(V) - j * 0.00390625);
  std::fprintf(stderr, "%d", tamd::fraction_bits(V));
  std::vector<double> y(1 << 16);
  while (const size_t n = std::fread(y.data(), 8, y.size(), stdin))
    for (size_t i = 0; i < n; ++i) {
      const uint64_t u = tamd::weight_units(y[i], powers);
      std::fwrite(&u, 8, 1, stdout);
    }
  return 0;
}
"""


@pytest.fixture(scope="module")
def units(tmp_path_factory):
    at = tmp_path_factory.mktemp("weights")
    (at / "w.cpp").write_text(PROGRAM)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-ffp-contract=off", "-I", CSRC, str(at / "w.cpp"), "-o", str(at / "w")])

    def run(V, y):
        done = subprocess.run([str(at / "w"), str(V)], input=np.ascontiguousarray(y, np.float64).tobytes(), capture_output=True, check=True)
        return np.frombuffer(done.stdout, np.uint64), int(done.stderr)
    return run


def of_kind(kind, V):
    """log2(1 / w) of V logits, the largest first."""
    rng = np.random.default_rng(V)
    if kind == "normal":
        z = np.sort((2.5 * rng.standard_normal(V)).astype(np.float32).astype(np.float64))[::-1]
        return (z[0] - z) / np.log(2.0)
    y = np.full(V, 39.7 if kind == "dominant" else 0.0)   # one holds nearly everything; all alike
    y[0] = 0.0
    return y


@pytest.mark.parametrize("V", [1, 100, 2047, 2048, 50001, 1 << 17, 1 << 20])
def test_every_weight(units, V):
    y = np.random.default_rng(1).uniform(0, 53, 200000)
    y[:4] = 0.0, 1.0, 2.0**-45, 0.5
    got, f = units(V, y)
    assert f == min(51, 62 - V.bit_length()) and got[0] == 2**f and got[1] == 2**(f - 1)
    exact = np.exp2(f - y.astype(np.longdouble))
    counts = y < f + 1
    off = np.abs(got.astype(np.longdouble) - exact)[counts]
    assert (off <= 0.5 + 2.0**-38 * exact[counts]).all()


@pytest.mark.parametrize("kind", ["normal", "dominant", "equal"])
@pytest.mark.parametrize("V", [1 << 17, 1 << 20])
def test_sums(units, V, kind):
    """Running sums over whole rows: within n / 2 units and 2^-38, and, where the roundings are not all alike, within eight standard
    deviations of that many roundings, a twelfth of a unit squared each."""
    y = of_kind(kind, V)
    got, f = units(V, y)
    got = np.where(y < f + 1, got, 0)
    exact = np.exp2(f - y.astype(np.longdouble))
    assert int(got.sum()) < 2**62
    off = np.abs(np.cumsum(got.astype(np.longdouble)) - np.cumsum(exact))
    n = np.arange(1, V + 1)
    assert (off <= n / 2 + 2.0**-38 * np.cumsum(exact)).all()
    if kind == "normal":
        assert (off <= 8 * np.sqrt(n / 12) + 1 + 2.0**-38 * np.cumsum(exact)).all()
