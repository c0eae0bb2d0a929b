"""How the delta rule's scans share out their chunks (``csrc/kda_delta_ranges.h``), replayed on the CPU:
each chunk belongs to one piece, and a piece that waits for a state waits for one that the range
before it publishes.  A wait without a publisher runs until its limit and leaves wrong results."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "simpletrain_b200", "csrc")
PROGRAM = r"""
#include "kda_delta_ranges.h"
using namespace kda::delta;
// pieces of every range, in order, as rows of (range, n, h, p0, p1, nc); returns their number
extern "C" int pieces(const int *first, int per_seq, int nseq, int H, int ranges, int *out, int most) {
  const Streams s{first, per_seq, nseq, H};
  int rows = 0;
  for (int r = 0; r < ranges + 2; ++r) {  // tickets past the last range are drawn too
    int lo, hi;
    range_of(s.total(), ranges, r, &lo, &hi);
    Pieces p;
    Piece pc;
    p.begin(s, lo, hi);
    while (p.next(s, &pc)) {
      if (rows == most) return -1;
      int *o = out + 6 * rows++;
      o[0] = r; o[1] = pc.n; o[2] = pc.h; o[3] = pc.p0; o[4] = pc.p1; o[5] = pc.nc;
    }
  }
  return rows;
}
"""


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("ranges")
    (d / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(d / "p.cpp"), "-o", str(d / "p.so")], check=True)
    fn = ctypes.CDLL(str(d / "p.so")).pieces

    def call(lens, H, ranges, packed=True):
        chunks = [-(-n // 64) for n in lens]
        first = (ctypes.c_int * (len(lens) + 1))(*[sum(chunks[:i]) for i in range(len(lens) + 1)])
        most = 2 * ranges + 2 * len(lens) * H + 8
        out = (ctypes.c_int * (6 * most))()
        rows = fn(first if packed else None, chunks[0] if chunks else 0, len(lens), H, ranges, out, most)
        assert rows >= 0
        return [tuple(out[6 * i:6 * i + 6]) for i in range(rows)]
    return call


def check(rows, lens, H, ranges):
    chunks = [-(-n // 64) for n in lens]
    seen = {}
    published, waited = set(), set()
    for r, n, h, p0, p1, nc in rows:
        assert r < ranges and nc == chunks[n] and 0 <= p0 < p1 <= nc
        for c in range(p0, p1):
            assert seen.setdefault((n, h, c), r) == r
        if p0 > 0:
            waited.add((r, n, h, p0))
        if p1 < nc:
            published.add((r + 1, n, h, p1))
    assert len(seen) == H * sum(chunks)
    assert len({r for r, *_ in published}) == len(published)  # a slot and a flag a range
    assert waited == published


def sm_ranges(lens, H, sms=148):
    return max(1, min(len(lens) * H, sms))


@pytest.mark.parametrize("lens,H", [
    ([128] + [0] * 31, 8), ([200] + [0] * 15, 10), ([0] * 31 + [128], 8), ([0] * 20 + [65] + [0] * 20, 4), ([700], 1),
    ([0, 0, 0], 5), ([], 3), ([64] * 200, 1), ([1] * 147 + [10000], 1), ([900, 0, 64, 130] + [65] * 20, 4),
])
def test_every_wait_has_its_publisher(pieces, lens, H):
    check(pieces(lens, H, sm_ranges(lens, H)), lens, H, sm_ranges(lens, H))


def test_random_batches(pieces):
    rng = random.Random(5)
    for _ in range(400):
        n = rng.choice([1, 2, 5, 30, 200])
        top = rng.choice([1, 64, 200, 5000])
        lens = [rng.choice([0, 0, rng.randint(0, top)]) for _ in range(n)]
        H = rng.choice([1, 2, 5, 8, 28, 40])
        check(pieces(lens, H, sm_ranges(lens, H)), lens, H, sm_ranges(lens, H))
        equal = [rng.randint(1, top)] * n
        check(pieces(equal, H, sm_ranges(equal, H), packed=False), equal, H, sm_ranges(equal, H))
