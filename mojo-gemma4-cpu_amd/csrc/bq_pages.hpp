// bq_pages.hpp -- the page table of the 16-bit cache and of the page operators,
// in plain C++ so that the same lines run in the kernels and in a CPU build.
//
// base_rows [num_seqs, max_pages] int32: the first cache row (slot) of the page
// that holds a sequence's positions [j << shift, (j + 1) << shift), or -1.  The
// table is device memory that the host does not read, so every use of an entry
// checks it here: what does not name rows inside the cache is no page.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define BQ_HD __host__ __device__ inline
#else
#define BQ_HD inline
#endif

namespace bq {

constexpr int kMaxPageShift = 20;

// whether an entry's whole page lies in the cache's num_slots rows
BQ_HD bool page_in(int32_t base, int shift, int64_t num_slots) {
  return base >= 0 && (int64_t)base + ((int64_t)1 << shift) <= num_slots;
}

// the cache row of position p of a sequence, -1 if there is none
BQ_HD int64_t page_slot(const int32_t* rows, int max_pages, int shift, int64_t num_slots,
                        int64_t p) {
  if (p < 0 || (p >> shift) >= max_pages) return -1;
  const int32_t base = rows[p >> shift];
  return page_in(base, shift, num_slots) ? (int64_t)base + (p & (((int64_t)1 << shift) - 1)) : -1;
}

// the page number of an entry, -1 if it names none of the pool's pages
BQ_HD int32_t page_number(int32_t base, int shift, int32_t num_pages) {
  if (base < 0 || (base & (((int32_t)1 << shift) - 1))) return -1;
  return (base >> shift) < num_pages ? base >> shift : -1;
}

// The attention shares its num_seqs s_max slots per kv head out by length: a sequence
// gets `share` of a workgroup for each of its tiles, rounded up or down (`round`), and
// one at least; none takes fewer than kMinTiles tiles.  Rounded down, shares of
// units / all tiles fill at most units + num_seqs - 1 slots (units, of one sequence);
// rounded up, shares of (units - num_seqs) / all tiles fill at most units.
constexpr int kMinTiles = 6;
BQ_HD int attn_units(int num_seqs, int s_max) {
  return num_seqs > 1 ? num_seqs * (s_max - 1) : s_max;
}
// whether the largest share that rounded up fits the units is looked for
BQ_HD bool attn_rounds_up(int num_seqs, int units) {
  return num_seqs > 1 && num_seqs <= 64 && units > num_seqs;
}
// 1e-6: the product of whole numbers may be a little off
constexpr double kRoundDown = 1e-6, kRoundUp = 1.0 - 1e-6;
BQ_HD int attn_splits(int tiles, double share, double round, int most) {
  const double n = (double)tiles * share + round;
  const int whole = n < most ? (int)n : most, room = tiles / kMinTiles;
  return whole < 1 || room < 1 ? 1 : whole < room ? whole : room;
}

// How sequence i goes on after a reorder, from its parent's length: `full`
// whole pages that are shared, then pages [full, end) that are its own (the
// first of them may hold len % page_rows positions already).
struct SeqPlan {
  int32_t parent;  // -1: an empty sequence
  int32_t len;     // positions it holds
  int32_t full, end;
};

BQ_HD SeqPlan seq_plan(int32_t parent, int32_t num_seqs, int32_t parent_len, int32_t grow,
                       int max_pages, int shift) {
  SeqPlan s;
  s.parent = parent >= 0 && parent < num_seqs ? parent : -1;
  const int64_t room = (int64_t)max_pages << shift;
  int64_t len = s.parent >= 0 && parent_len > 0 ? parent_len : 0;
  len = len < room ? len : room;
  const int64_t want = len + (grow > 0 ? grow : 0) + (((int64_t)1 << shift) - 1);
  const int64_t end = want >> shift;
  s.len = (int32_t)len;
  s.full = (int32_t)(len >> shift);
  s.end = (int32_t)(end < max_pages ? end : max_pages);
  return s;
}

// what of its parent's table a sequence keeps
BQ_HD bool seq_keeps(const SeqPlan& s, int j) {
  return s.parent >= 0 && (j < s.full || (j == s.full && j < s.end));
}

}  // namespace bq
