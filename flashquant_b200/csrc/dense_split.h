// How the one-token attention over 16-bit pages is cut into runs, and what each run owes to the others.
// Plain integer arithmetic, the same on the host (where it is tested) and in the kernel.
//
// A "unit" is what one warp attends with: up to 16 query heads of one KV head of one sequence.  `side` units
// of a sequence stand side by side in a CTA (adjacent warps read adjacent heads of the same tokens, so the
// rows of a page are read whole); the CTA has `teams` = warps / side such rows of warps.  The tiles of 16
// tokens of all unit groups of all sequences form one list of `total` entries, cut into runs of `length`, run
// i for team i % teams of CTA i / teams.  Ragged batches are balanced whatever their lengths.
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
  int total;   // entries of the list
  int length;  // of a run
  int teams;   // runs of a CTA
  FQ_HD int run_of(int at) const { return at / length; }
  FQ_HD int begin(int run) const {
    const int64_t x = int64_t(run) * length;
    return x < total ? int(x) : total;
  }
  FQ_HD int end(int run) const { return begin(run + 1); }
};
// At least `shortest` tiles to a run (a short list is not cut finer: its parts have to be joined again).
FQ_HD DenseCut dense_cut(int total, int ctas, int teams, int shortest) {
  const int64_t runs = int64_t(ctas) * teams;
  int length = int((total + runs - 1) / runs);
  if (length < shortest) length = shortest;
  return DenseCut{total, length, teams};
}

// A unit group takes the entries [a, b) of the list.  A run that holds all of them writes its result; the
// others leave a piece.  A run has at most two pieces: the one that was begun before it (slot 0) and the one
// that goes on behind it (slot 1).
FQ_HD int dense_slot(const DenseCut& c, int run, int a) { return a < c.begin(run) ? 0 : 1; }
// The teams of a CTA that are all inside one unit group merge first and leave one piece.
FQ_HD bool dense_cta_merges(const DenseCut& c, int cta, int a, int b) {
  const int first = cta * c.teams, last = first + c.teams - 1;
  return c.begin(first) >= a && c.begin(last) < b && c.end(last) <= b;
}
// The pieces of a unit group, in the order of the list: `before` runs, `whole` merging CTAs that count once
// each, then runs again.
struct DensePieces {
  int first, before, cta, whole, count;
};
FQ_HD DensePieces dense_pieces(const DenseCut& c, int a, int b) {
  DensePieces p;
  const int last = c.run_of(b - 1);
  p.first = c.run_of(a);
  const int inner = (a + c.length - 1) / c.length;                 // the first run that begins inside
  const int after = b == c.total ? last + 1 : b / c.length;        // behind the last one that ends inside
  p.cta = (inner + c.teams - 1) / c.teams;
  p.whole = after / c.teams - p.cta;
  if (c.teams == 1 || p.whole < 0) p.whole = 0;
  p.before = p.whole ? p.cta * c.teams - p.first : 0;
  p.count = last - p.first + 1 - p.whole * (c.teams - 1);
  return p;
}
// the run whose slots hold piece i (of a merging CTA: its first)
FQ_HD int dense_piece_run(const DenseCut& c, const DensePieces& p, int i) {
  if (p.whole == 0 || i < p.before) return p.first + i;
  if (i < p.before + p.whole) return (p.cta + i - p.before) * c.teams;
  return (p.cta + p.whole) * c.teams + i - p.before - p.whole;
}

}  // namespace fq
