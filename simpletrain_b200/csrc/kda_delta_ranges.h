// How the delta rule's scans share out their chunks: plain arithmetic, for the kernels
// and for the host (tests replay it on the CPU).
//
// The chunks of all streams (sequence, head), stream after stream, are cut into equal
// ranges.  A range's CTA runs its pieces in this order: the last stream's part, which begins that
// stream unless the whole range lies inside one; the streams between; the first stream's part.
// A piece whose stream began in an earlier range (p0 > 0) starts from the state that the range
// just before published; a piece whose stream goes on (p1 < nc) publishes for the range just behind.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define KDA_HD __host__ __device__ __forceinline__
#else
#define KDA_HD inline
#endif

namespace kda {
namespace delta {

struct Streams {
  const int *first;  // [nseq + 1] first chunk of each sequence; NULL: per_seq chunks each
  int per_seq, nseq, H;
  KDA_HD int chunks(int n) const { return first == nullptr ? per_seq : first[n + 1] - first[n]; }
  KDA_HD int64_t total() const { return (int64_t)H * (first == nullptr ? (int64_t)per_seq * nseq : first[nseq]); }
};

// Chunks [*lo, *hi) of range `range` of `ranges`.  Where there are fewer chunks than ranges (many empty
// sequences), the first `total` ranges hold one each and the others none: an empty range
// between two others would hand no state on.
KDA_HD void range_of(int64_t total, int ranges, int range, int *lo, int *hi) {
  const int used = total < ranges ? (int)total : ranges;
  *lo = range < used ? (int)(total * range / used) : 0;
  *hi = range < used ? (int)(total * (range + 1) / used) : 0;
}

// A part of a stream: positions [p0, p1) of its nc chunks (position 0 is the last chunk in reverse).
struct Piece {
  int n, h, p0, p1, nc;
};

struct Pieces {
  int n0, h0, c0, nc0, n1, h1, c1;  // streams and positions of the first and the last chunk
  int turn, n, h;
  static KDA_HD void locate(const Streams &s, int x, int *sn, int *sh, int *sc) {
    if (s.first == nullptr) {
      const int i = x / s.per_seq;
      *sn = i / s.H;
      *sh = i % s.H;
      *sc = x % s.per_seq;
      return;
    }
    int l = 0, r = s.nseq;  // H first[l] <= x < H first[r]
    while (r - l > 1) {
      const int mid = (l + r) >> 1;
      if ((int64_t)s.first[mid] * s.H <= x) l = mid; else r = mid;
    }
    const int nc = s.chunks(l), rem = x - s.first[l] * s.H;
    *sn = l;
    *sh = rem / nc;
    *sc = rem % nc;
  }
  KDA_HD void begin(const Streams &s, int lo, int hi) {
    turn = lo < hi ? 0 : 3;
    if (turn == 3) return;
    locate(s, lo, &n0, &h0, &c0);
    locate(s, hi - 1, &n1, &h1, &c1);
    nc0 = s.chunks(n0);
  }
  KDA_HD bool next(const Streams &s, Piece *p) {
    if (turn == 0) {
      const bool one = n0 == n1 && h0 == h1;
      *p = {n1, h1, one ? c0 : 0, c1 + 1, s.chunks(n1)};
      turn = one ? 3 : 1;
      n = n0;
      h = h0;
      return true;
    }
    if (turn == 1) {  // the next stream that has chunks; the range's last one is not behind us
      if (++h == s.H) {
        h = 0;
        do ++n; while (s.chunks(n) == 0);
      }
      if (n != n1 || h != h1) {
        const int nc = s.chunks(n);
        *p = {n, h, 0, nc, nc};
        return true;
      }
      turn = 2;
    }
    if (turn == 2) {
      *p = {n0, h0, c0, nc0, nc0};
      turn = 3;
      return true;
    }
    return false;
  }
};

}  // namespace delta
}  // namespace kda
