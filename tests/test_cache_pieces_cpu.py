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
    return lambda cases: subprocess.run([str(d / "pieces")], input="\n".join("%d %d" % c for c in cases), text=True, check=True,
                                        capture_output=True).stdout.split()


def test_pieces_cover_a_unit_of_any_length(run):
    # 2^30 slots are 2^26 tiles of 16 keys; two blocks on each of 148 SMs
    tiles = [1, 2, 3, 295, 296, 297, 1000, 7255013, 7255014, 2 ** 23, 2 ** 23 + 1, 2 ** 24 - 1, 2 ** 26 - 1, 2 ** 26]
    cases = [(t, n) for t in tiles for n in (1, 2, 7, 100, 147, 148, 149, 255, 256, 257, 295, 296)]
    got = run(cases)
    assert len(got) == len(cases) and all(g == "1" for g in got), [c for c, g in zip(cases, got) if g != "1"]
