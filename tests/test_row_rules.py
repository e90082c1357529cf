"""The top logits' host rule, compiled from the library's own header with g++ (no GPU): a last wave of few lanes does not
spoil the bound of a row of any length, so that only ties, short rows of many and their like go to the search for ties."""

import pathlib
import shutil
import subprocess

import numpy as np
import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
CSRC = ROOT / "alpha-fly_amd" / "csrc"
HIP_INCLUDE = pathlib.Path("/opt/rocm/include")

PROGRAM = r"""
#include "row_rules.hpp"
#include <cstdio>
int main() {
  long long rows, cols;
  int elem, k;
  while (scanf("%lld %lld %d %d", &rows, &cols, &elem, &k) == 4) {
    const auto s = fly::top_shape(rows, cols, elem, k);
    printf("%d %d %d %d\n", s.row.threads, s.row.kept, s.holders, s.spread);
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None or not (HIP_INCLUDE / "hip" / "hip_runtime.h").exists():
        pytest.skip("g++ or the HIP headers are not installed")
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-D__HIP_PLATFORM_AMD__", f"-I{HIP_INCLUDE}", f"-I{CSRC}", f"-I{ROOT / 'include'}",
                    str(d / "rules.cpp"), "-o", str(d / "rules")], check=True)

    def ask(cases):
        out = subprocess.run([str(d / "rules")], input="\n".join(" ".join(map(str, c)) for c in cases), check=True,
                             capture_output=True, text=True)
        return [tuple(int(v) for v in line.split()) for line in out.stdout.splitlines()]

    return ask


KS = (1, 2, 9, 17, 31, 32, 33, 48, 64, 65, 100, 128, 129, 192, 200, 218, 255, 256)


@pytest.mark.parametrize("elem", [2, 4])
@pytest.mark.parametrize("rows", [1, 100, 4096])
def test_the_bounding_waves_have_lanes_to_bound_with(rule, rows, elem):
    cases = [(rows, cols, elem, k) for cols in [*range(1, 6000, 3), *range(6000, 70000, 997)] for k in KS]
    for (_, cols, _, k), (threads, kept, holders, spread) in zip(cases, rule(cases)):
        assert 1 <= holders <= threads // 64 or spread
        if spread:
            assert cols <= 256 * spread and holders == min(4, -(-cols // 64))
        elif cols > 128 and not (rows >= 1024 and cols <= 400 and k <= 64):
            lanes, c = min(64, cols * elem // 16 - 64 * (holders - 1)), -(-k // holders)
            assert c <= lanes, (rows, cols, elem, k, threads, kept, holders)


@pytest.mark.parametrize("case,holders,spread", [((100, 1290, 4, 128), 5, 0), ((100, 2060, 2, 128), 4, 0), ((100, 1280, 4, 128), 5, 0),
                                                 ((100, 300, 4, 64), 4, 4), ((4096, 900, 4, 128), 3, 0), ((1, 4168, 4, 218), 7, 0)])
def test_sizes_around_a_full_wave(rule, case, holders, spread):
    got = rule([case])[0]
    assert got[2:] == (holders, spread), got


# Rows of normal logits, as the kernel bounds them: the c-th largest of the lanes' largest, the least over the waves.
@pytest.mark.parametrize("rows,cols,elem,k", [(100, 1290, 4, 128), (100, 2060, 2, 128), (100, 500, 4, 64), (100, 900, 4, 20),
                                              (4096, 560, 4, 64), (4096, 3000, 2, 100), (100, 1111, 2, 64), (100, 4168, 4, 218)])
def test_the_lists_hold_what_passes(rule, rows, cols, elem, k):
    threads, kept, holders, spread = rule([(rows, cols, elem, k)])[0]
    assert not spread
    n, c, rng = 16 // elem, -(-k // holders), np.random.default_rng(cols)
    waves = threads // 64
    for _ in range(50):
        z = rng.normal(size=cols)
        piece = np.arange(cols) // n
        whole = piece < cols // n
        lane = np.where(whole, piece % threads, 0)
        top = np.full(threads, -np.inf)
        np.maximum.at(top, lane, z)
        bound = min(np.sort(top[64 * w: 64 * w + 64])[-c] for w in range(holders))
        found = np.bincount(lane[z >= bound] // 64, minlength=waves)
        assert found.sum() >= k and found.max() <= 128
