"""The read-out loss's workspace, compiled from the library's own header with g++ (no GPU): how many rows a piece has, and that what the
kernels of a piece write lies apart and inside, over sizes from one row and column to the largest."""

from __future__ import annotations

import random
import shutil
import subprocess

import pytest

from test_readout_rules import CSRC, HIP_INCLUDE, ROOT

# For each piece that a call may have (a whole one, and what is left at the end) the bytes from each part's start up to the last one that
# a kernel writes, by the kernels' own indexes.
PROGRAM = r"""
#include "readout_rules.hpp"
#include <cstdio>
using namespace fly;
int main() {
  long long rows, d, v, k;
  int planes, wanted;
  while (scanf("%lld %lld %lld %lld %d %d", &rows, &d, &v, &k, &planes, &wanted) == 6) {
    const Call c{planes == 2 ? FLY_F32 : FLY_BF16, rows, d, v, k, (wanted & 1) != 0, (wanted & 2) != 0, (wanted & 4) != 0};
    const Space s(c, planes);
    printf("%lld %zu", (long long)s.piece, s.bytes);
    auto part = [&](size_t from, long long bytes) { if (bytes) printf(" %zu %lld", from, bytes); };
    const long long rest = rows % s.piece ? rows % s.piece : s.piece, padded = s.vb * 32;
    for (long long n : {std::min<long long>(s.piece, rows), rest}) {
      const long long rb = (n + 31) / 32, tiles = (n + 63) / 64;
      auto block = [&](long long r, long long of, long long b) { return ((r * of + b) * planes + planes - 1) * 1024 + 1024; };
      printf(" :");
      part(s.x, block(2 * rb - 1, s.db, s.db - 1));
      part(s.w, block(2 * s.vb - 1, s.db, s.db - 1));
      if (c.gw) part(s.xt, block(2 * s.db - 1, rb, rb - 1));
      if (c.gx) part(s.wt, block(2 * s.db - 1, s.vb, s.vb - 1));
      if (c.gx) part(s.g, block(2 * rb - 1, s.vb, s.vb - 1));
      if (c.gw) part(s.gt, block(2 * s.vb - 1, rb, rb - 1));
      if (c.grads()) part(s.z, ((n + 15) / 16) * (padded / 16) * 64 * (planes == 2 ? 16 : 8));
      part(s.unit_x, rb * 32 * 4);
      part(s.unit_w, padded * 4);
      part(s.bias, padded * 4);
      part(s.stat, ((n - 1) * s.parts + parts_of(planes, logits_shape(planes, n, v), padded)) * 8);
      part(s.info, n * 16);
      part(s.factor, n * 4);
      part(s.turned, n * 8);
      part(s.column, ((k - 1) * s.piece + n) * 4);
      part(s.weight, ((k - 1) * s.piece + n) * 4);
      part(s.logit, ((k - 1) * s.piece + n) * 4);
      part(s.list_sums, n * 8);
      if (c.grads()) part(s.maxima, sizeof(Maxima));
      if (c.gb) part(s.sums, ((tiles - 1) * padded + v) * 4);
      if (s.piece < rows && c.gw) part(s.acc_w, v * s.db * 128);
      if (s.piece < rows && c.gb) part(s.acc_b, v * 4);
      const Splits p = splits_of(planes, c, n);
      if (c.gx && p.x > 1) part(s.share_x, p.x * n * s.db * 128);
      if (c.gw && p.w > 1) part(s.share_w, p.w * v * s.db * 128);
    }
    printf("\n");
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def space(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None or not (HIP_INCLUDE / "hip" / "hip_runtime.h").exists():
        pytest.skip("g++ or the HIP headers are not installed")
    d = tmp_path_factory.mktemp("space")
    (d / "space.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-D__HIP_PLATFORM_AMD__", f"-I{HIP_INCLUDE}", f"-I{CSRC}", f"-I{ROOT / 'include'}",
                    str(d / "space.cpp"), "-o", str(d / "space")], check=True)

    def ask(cases):
        out = subprocess.run([str(d / "space")], input="\n".join(" ".join(map(str, c)) for c in cases), check=True,
                             capture_output=True, text=True).stdout
        for line in out.splitlines():
            head, *pieces = line.split(":")
            piece, total = map(int, head.split())
            yield piece, total, [list(zip(*[iter(map(int, p.split()))] * 2)) for p in pieces]

    return ask


def _cases(n):
    r = random.Random(5)
    size = lambda top: max(1, int(2 ** r.uniform(0, top)))
    for _ in range(n):
        yield size(24), size(16), size(20), size(10), r.choice((1, 2)), r.randrange(8)


def test_parts_of_the_workspace_lie_apart(space):
    cases = list(_cases(3000)) + [(rows, 4, 1 << 20, 3, p, 7) for rows in (320, 321, 400, 640, 641, 700) for p in (1, 2)]
    for case, (_, total, pieces) in zip(cases, space(cases)):
        for spans in pieces:
            at = 0
            for start, size in sorted(spans):
                assert start >= at and start % 256 == 0, case
                at = start + size
            assert at <= total, case


def test_rows_of_a_piece(space):
    """Multiples of 64 rows, one piece where everything fits 4 GiB, and never more than tiles can count."""
    cases = list(_cases(3000))
    for (rows, d, v, k, planes, wanted), (piece, total, _) in zip(cases, space(cases)):
        assert piece % 64 == 0 and 64 <= piece <= 1 << 19 and piece < rows + 64
        logit = 2 * planes * (bool(wanted) + bool(wanted & 1) + bool(wanted & 2))
        row = (v + 31) // 32 * 32 * logit + (d + 31) // 32 * 64 * planes * (1 + bool(wanted & 2)) + 12 * k
        assert piece == 64 or piece * row <= 1 << 32
        assert piece >= min(rows, 1 << 19) or (piece + 64) * (row + 8 * ((v + 63) // 64 * 2)) > 1 << 32


def test_known_pieces(space):
    """float32 with all gradients takes 12 bytes of a logit, 16-bit types 6: with 2^20 columns that is 320 and 640 rows."""
    cases = [(400, 4, 1 << 20, 3, 2, 7), (700, 4, 1 << 20, 3, 1, 7), (300, 4, 1 << 20, 1, 1, 7), ((1 << 19) + 100, 8, 5, 2, 2, 7)]
    assert [p for p, *_ in space(cases)] == [320, 640, 320, 1 << 19]
