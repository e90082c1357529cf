"""The read-out loss's host rules, compiled from the library's own header with g++ (no GPU): what they promise the kernels, over
sizes from one row and column to the largest."""

import pathlib
import random
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
CSRC = ROOT / "alpha-fly_amd" / "csrc"
HIP_INCLUDE = pathlib.Path("/opt/rocm/include")

PROGRAM = r"""
#include "readout_rules.hpp"
#include <cstdio>
using namespace fly;
int main() {
  long long rows, d, v;
  int planes, gx, gw;
  while (scanf("%lld %lld %lld %d %d %d", &rows, &d, &v, &planes, &gx, &gw) == 6) {
    const Call c{planes == 2 ? FLY_F32 : FLY_BF16, rows, d, v, 1, gx != 0, gw != 0, false};
    const Shape l = logits_shape(planes, rows, v), g = grad_shape(planes, c, rows);
    const Splits s = splits_of(planes, c, rows);
    const long long padded = (v + 31) / 32 * 32;
    printf("%d %d %d %d %d %d %d %d\n", l, parts_of(planes, l, padded), parts_of(planes, kSmall, padded), part_shift(planes, l), g, s.x,
           s.w, few_rows(c));
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


def _cases(n):
    r = random.Random(4)
    size = lambda top: max(1, int(2 ** r.uniform(0, top)))
    for _ in range(n):
        gx = r.randrange(2)
        yield size(19), size(16), size(20), r.choice((1, 2)), gx, 1 if not gx else r.randrange(2)


def test_parts_of_columns_fit_their_space(rule):
    """A row's parts cover its columns and are no more than the space that the smallest tile's, rounded up to 4, give."""
    cases = list(_cases(4000))
    for (_, _, v, _, _, _), (_, parts, small, shift, *_) in zip(cases, rule(cases)):
        assert parts << shift >= (v + 31) // 32 * 32 and parts <= (small + 3) // 4 * 4


def test_parts_of_k_fit_theirs(rule):
    """Sums of parts fit 32 MiB each; a part has 16 blocks of k, but for rounding; few enough jobs for a launch."""
    cases = list(_cases(4000))
    for (rows, d, v, _, gx, gw), (_, _, _, _, _, x, w, _) in zip(cases, rule(cases)):
        for wanted, m, k, parts in ((gx, rows, v, x), (gw, v, rows, w)):
            assert parts >= 1 and (wanted or parts == 1)
            if parts > 1:
                assert parts * m * ((d + 31) // 32 * 128) <= 32 << 20 and (k + 31) // 32 / parts > 7.5


def test_few_rows_are_few(rule):
    cases = [(rows, d, v, p, 1, 1) for rows in (1, 32, 33, 64, 65, 96, 97) for d in (1, 3, 4, 8, 300, 3000) for v in (1, 500, 50_000)
             for p in (1, 2)]
    for (rows, d, v, p, _, _), got in zip(cases, rule(cases)):
        few = got[-1]
        assert not few or (rows <= 96 and d >= (4 if p == 2 else 8))      # rows have a whole piece
        assert few or rows > 32 or d < 8


def test_listed_shapes(rule):
    """The shapes that the comments name, by their measurements."""
    small, medium, large = range(3)
    logits = {(256, 2333, 4168, 1): small, (1120, 2333, 4168, 1): medium, (4096, 2333, 4168, 1): medium, (10000, 2333, 4168, 1): large,
              (4096, 1024, 32000, 1): large, (256, 2333, 4168, 2): small, (543, 2333, 4168, 2): medium, (1120, 2333, 4168, 2): large,
              (256, 1024, 32000, 2): medium}
    grads = {(100, 1024, 32000, 1): small, (1120, 1024, 32000, 1): large, (4096, 2333, 4168, 1): medium, (4096, 2333, 4168, 2): medium,
             (4096, 512, 2000, 2): small}
    assert [g[0] for g in rule([(*k, 1, 1) for k in logits])] == list(logits.values())
    assert [g[4] for g in rule([(*k, 1, 1) for k in grads])] == list(grads.values())
