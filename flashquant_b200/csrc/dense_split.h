// How the one-token attention over 16-bit pages is cut into runs, and what each run owes to the others.
// Plain integer arithmetic, the same on the host (where it is tested) and in the kernels.
//
// A "unit" is what one warp attends with: up to 16 query heads of one KV head of one sequence.  `side` units
// of a sequence stand side by side (they are given to warps that run at the same time, so that the heads of a
// token, which are adjacent in a page, are read together).  The tiles of 16 tokens of all unit groups of all
// sequences form one list of `total` entries, cut into runs whatever the bounds between sequences are: a ragged
// batch is balanced.  Where a warp's share is long, some of every sixteen entries (the "tail") are not dealt out
// beforehand but in short runs that warps take when they are free: SMs do not get the same share of the memory's
// bandwidth (8 sequences of 32k - 131k tokens, equal runs: the first warp was through after 350 us, the last after 456).
// Every sequence has its part of the tail, since short runs are pieces to join.  Where the cuts are never depends on
// who takes a run.
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
  s.tiles = s.len > 0 ? (s.len - 1) / kDenseTile + 1 - s.first_tile : 0;
  return s;
}

// Tiles of a share from which on there is a tail.  Queries, pieces and their join cost more than the balance gives below:
// 32 x 4096 tokens (a share of 55) 94 us without, 94 with one; 64 x 2000, head_dim 256 (108) 166, 170; ragged 8 x 131072
// (300) 452 without, 433 with one.
constexpr int kDenseShare = 192;
constexpr int kDenseMain = 14;    // entries of sixteen that are not in the tail
constexpr int kDenseTaken = 4;    // runs taken per share, at most
constexpr int kDenseShortest = 1; // tiles of a run at least
constexpr int kDenseGroups = 4;   // unit groups to a share from which on there is none (a piece of each is kept room for)

struct DenseCut {
  int total;                  // entries of the list (below 2^30)
  bool split;                 // there is a tail
  int fixed;                  // runs that are dealt out beforehand, of the others
  int mains, length;          // entries of these, of one of them
  int tails, shorter;         // entries of the tail, of one of its runs

  // entries of the main kind before entry x of the list, and back from either kind
  FQ_HD int main_of(int x) const {
    return split ? x / 16 * kDenseMain + (x % 16 < kDenseMain ? x % 16 : kDenseMain) : x;
  }
  FQ_HD int kind_of(bool tail, int x) const { return tail ? x - main_of(x) : main_of(x); }
  FQ_HD int entry(bool tail, int i) const {
    return tail ? i / (16 - kDenseMain) * 16 + kDenseMain + i % (16 - kDenseMain)
                : (split ? i / kDenseMain * 16 + i % kDenseMain : i);
  }
  // runs count through; the entries of a run are of its own kind
  FQ_HD bool is_tail(int run) const { return run >= fixed; }
  FQ_HD int run_of(bool tail, int i) const { return tail ? fixed + i / shorter : i / length; }
  FQ_HD int begin(int run) const {
    const int64_t x = is_tail(run) ? int64_t(run - fixed) * shorter : int64_t(run) * length;
    const int most = is_tail(run) ? tails : mains;
    return x < most ? int(x) : most;
  }
  FQ_HD int end(int run) const {
    const int64_t x = int64_t(begin(run)) + (is_tail(run) ? shorter : length);
    const int most = is_tail(run) ? tails : mains;
    return x < most ? int(x) : most;
  }
  FQ_HD int taken() const { return (tails + shorter - 1) / shorter; }
};
// `groups`: unit groups of all sequences
FQ_HD DenseCut dense_cut(int total, int fixed, int groups) {
  DenseCut c;
  const int share = (total + fixed - 1) / fixed;
  c.total = total;
  c.fixed = fixed;
  c.split = share >= kDenseShare && groups <= kDenseGroups * fixed;
  c.mains = c.main_of(total);
  c.tails = total - c.mains;
  c.length = c.split ? (c.mains + fixed - 1) / fixed : share;
  if (c.length < kDenseShortest) c.length = kDenseShortest;
  c.shorter = share / 24 + 1;
  return c;
}

// A unit group takes the entries [a, b) of the list.  A run that holds all of them writes its result; the others
// leave a piece.  The pieces of a group are those of its runs, the tail's behind the others.
struct DensePieces {
  int main0, mains, tail0, tails;  // first run and number of either kind
  FQ_HD int count() const { return mains + tails; }
  FQ_HD int run(int i) const { return i < mains ? main0 + i : tail0 + i - mains; }
};
FQ_HD DensePieces dense_pieces(const DenseCut& c, int a, int b) {
  DensePieces p{0, 0, 0, 0};
  const int m0 = c.main_of(a), m1 = c.main_of(b), t0 = a - m0, t1 = b - m1;
  if (m1 > m0) {
    p.main0 = c.run_of(false, m0);
    p.mains = c.run_of(false, m1 - 1) - p.main0 + 1;
  }
  if (t1 > t0) {
    p.tail0 = c.run_of(true, t0);
    p.tails = c.run_of(true, t1 - 1) - p.tail0 + 1;
  }
  return p;
}
// whether `run`, which holds some of them, holds all
FQ_HD bool dense_whole(const DenseCut& c, int run, int a, int b) {
  const bool tail = c.is_tail(run);
  return c.kind_of(!tail, a) == c.kind_of(!tail, b) && c.kind_of(tail, a) >= c.begin(run) &&
         c.kind_of(tail, b) <= c.end(run);
}
// Where the piece of the `nth` group, which takes the entries from `a` on, stands that a run leaves.  Without a tail a run
// has at most two: of the group that was begun before it and of the one that goes on behind it.  With one, a group that
// the run has the main entries of is no whole either; but along the list of either kind each next piece is of a later
// run or of a later group, so that the sum of the two counts them.
FQ_HD int dense_slot(const DenseCut& c, int run, int nth, int groups, int a) {
  if (!c.split) return 2 * run + (a < c.begin(run) ? 0 : 1);
  return run + nth + (c.is_tail(run) ? groups : 0);
}
// Slots in all, whatever the lengths are.
FQ_HD int dense_slots(int fixed) { return fixed * (1 + kDenseTaken + 2 * kDenseGroups); }

}  // namespace fq
