"""How the tiles of a sequence are cut into pieces, up to the longest sequence that is accepted: no GPU is needed."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mesh-transformer-jax_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "mtj_cache_kernels.h"
int main() {
  long long tiles;
  int n;
  int first, last;
  if (scanf("%d", &n) == 1)
    for (int left = n; left > 0 && scanf("%d %d %d", &first, &last, &n) == 3; --left) printf("%d\n", mtj::unit_blocks_of(first, last, n));
  while (scanf("%lld %d", &tiles, &n) == 2) {
    long long before = 0, least = tiles, most = 0;
    bool good = mtj::unit_piece_begin(static_cast<int>(tiles), n, 0) == 0 && mtj::unit_piece_begin(static_cast<int>(tiles), n, n) == tiles;
    for (int k = 1; k <= n; ++k) {
      const long long at = mtj::unit_piece_begin(static_cast<int>(tiles), n, k);
      good = good && at >= before && at == tiles * k / n;
      least = at - before < least ? at - before : least;
      most = at - before > most ? at - before : most;
      before = at;
    }
    printf("%d\n", good && most - least <= 1);
  }
}
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    import __graft_entry__ as ge
    build = ge._load_build_module()
    d = tmp_path_factory.mktemp("pieces")
    (d / "pieces.cu").write_text(PROGRAM)
    subprocess.run([build.NVCC, *build.FLAGS, "-I", CSRC, str(d / "pieces.cu"), "-o", str(d / "pieces")], check=True)
    return lambda cases, units=(): subprocess.run(
        [str(d / "pieces")], input="\n".join([str(len(units)), *("%d %d %d" % u for u in units), *("%d %d" % c for c in cases)]), text=True, check=True,
        capture_output=True).stdout.split()


def test_pieces_cover_a_unit_of_any_length(run):
    # 2^30 slots are 2^26 tiles of 16 keys; two blocks on each of 148 SMs
    tiles = [1, 2, 3, 295, 296, 297, 1000, 7255013, 7255014, 2 ** 23, 2 ** 23 + 1, 2 ** 24 - 1, 2 ** 26 - 1, 2 ** 26]
    cases = [(t, n) for t in tiles for n in (1, 2, 7, 100, 147, 148, 149, 255, 256, 257, 295, 296)]
    got = run(cases)
    assert len(got) == len(cases) and all(g == "1" for g in got), [c for c, g in zip(cases, got) if g != "1"]


def test_units_whose_blocks_are_not_known_have_none(run):
    """What the second kernel takes for an index: entries that were not both written (scratch that holds anything) are not."""
    good = {(0, 0, 1): 1, (0, 295, 296): 296, (7, 9, 10): 3, (295, 295, 296): 1}
    bad = [(-1, 0, 296), (0, -1, 296), (5, 4, 296), (0, 296, 296), (296, 296, 296), (3, 10, 10), (-2 ** 31, 2 ** 31 - 1, 296), (2 ** 31 - 1, -2 ** 31, 296),
           (0, 2 ** 31 - 1, 296), (-2 ** 31, -2 ** 31, 296), (2 ** 31 - 1, 2 ** 31 - 1, 296), (0x7fc00000, 0x7fc00000, 1), (-1, -1, 296)]
    got = run([], [*good, *bad])
    assert [int(x) for x in got] == [*good.values(), *[0] * len(bad)]
