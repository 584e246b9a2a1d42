// How the one-token attention over 16-bit pages is cut into runs, and what each run owes to the others.
// Plain integer arithmetic, the same on the host (where it is tested) and in the kernels.
//
// A "unit" is what one warp attends with: up to 16 query heads of one KV head of one sequence.  `side` units
// of a sequence stand side by side (they are given to warps that run at the same time, so that the heads of a
// token, which are adjacent in a page, are read together).  The tiles of 16 tokens of all unit groups of all
// sequences form one list of `total` entries, cut into runs whatever the bounds between sequences are: a ragged
// batch is balanced.  Where a warp's share is long enough, thirteen sixteenths of the list
// are dealt out beforehand and the rest in runs of a sixteenth, then a thirty-second, of a share that warps take
// when they are free: SMs do not get
// the same share of the memory's bandwidth (8 sequences of 32k - 131k tokens, equal runs: the first SM was
// through after 345 us, the last after 483).  Where the cuts are never depends on who takes a run.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define FQ_HD __host__ __device__ __forceinline__
#else
#define FQ_HD inline
#endif

namespace fq {

constexpr int kDenseTile = 16;  // tokens

// The tiles of a sequence that are read: of `len` tokens (at most `room`, what its block-table row holds; a
// negative length is none) the last `window` (0: all).
struct DenseSpan {
  int len;         // tokens of the sequence
  int begin;       // first token that is seen
  int first_tile;  // begin / 16
  int tiles;
};
FQ_HD DenseSpan dense_span(int len, int64_t room, int window) {
  DenseSpan s;
  s.len = len < 0 ? 0 : (len > room ? int(room) : len);
  s.begin = window > 0 && window < s.len ? s.len - window : 0;
  s.first_tile = s.begin / kDenseTile;
  s.tiles = (s.len + kDenseTile - 1) / kDenseTile - s.first_tile;
  return s;
}

struct DenseCut {
  int total;             // entries of the list
  int fixed;             // runs that are dealt out beforehand
  int length, bound;     // of such a run; fixed * length, or total if that is all
  int medium, length2;   // runs behind `bound`, then
  int bound2, length3;   // runs behind bound2 to the end
  FQ_HD int run_of(int at) const {
    return at < bound ? at / length
                      : (at < bound2 ? fixed + (at - bound) / length2 : fixed + medium + (at - bound2) / length3);
  }
  FQ_HD int begin(int run) const {
    const int64_t x = run < fixed ? int64_t(run) * length
                                  : (run < fixed + medium ? bound + int64_t(run - fixed) * length2
                                                          : bound2 + int64_t(run - fixed - medium) * length3);
    return x < total ? int(x) : total;
  }
  FQ_HD int end(int run) const { return begin(run + 1); }
  FQ_HD int taken() const { return medium + (total - bound2 + length3 - 1) / length3; }
};
constexpr int kDenseShare = 32;   // tiles of a share from which on a part of the list is taken
constexpr int kDenseTaken = 6;    // runs taken per share, at most
constexpr int kDenseShortest = 2; // tiles of a run at least, where there are enough
FQ_HD DenseCut dense_cut(int total, int fixed) {
  DenseCut c;
  const int share = (total + fixed - 1) / fixed;  // (total below 2^30)
  c.total = total;
  c.fixed = fixed;
  c.length = share < kDenseShortest ? kDenseShortest : share;
  c.bound = c.bound2 = total;
  c.medium = 0;
  c.length2 = c.length3 = 1;
  if (share < kDenseShare) return c;
  c.length2 = (share + 15) / 16;
  c.length3 = (share + 31) / 32;
  c.length = share - 3 * c.length2;
  const int64_t bound = int64_t(c.length) * fixed;
  if (bound >= total) return c;
  c.bound = int(bound);
  const int fits = (total - c.bound) / c.length2;
  c.medium = fits < 2 * fixed ? fits : 2 * fixed;
  c.bound2 = c.bound + c.medium * c.length2;
  return c;
}

// A unit group takes the entries [a, b) of the list.  A run that holds all of them writes its result; the
// others leave a piece.  A run has at most two pieces: of the group that was begun before it (slot 0) and of the
// one that goes on behind it (slot 1).  The pieces of a group are those of its runs, run_of(a) to run_of(b - 1).
FQ_HD int dense_slot(const DenseCut& c, int run, int a) { return a < c.begin(run) ? 0 : 1; }

}  // namespace fq
