// Where a step's row goes in a paged cache (rope_append.cu); plain C++ too, for the tests on the host.
#pragma once
#ifdef __CUDACC__
#define MA_HD __host__ __device__ __forceinline__
#else
#define MA_HD inline
#endif

namespace ma {

// One round of the search for the last of `n` sequences that starts at or before a row: 32 probes,
// `step` apart, of which `hits` (the first ones, as the starts ascend; at least the first counts) are at
// or before it.  Leaves the range [lo, lo + n) that the next round looks at; it is found when n is 1.
MA_HD int search_step(int n) { return (n + 31) / 32; }
MA_HD void search_take(int hits, int* lo, int* n) {
  const int step = search_step(*n), j = (hits > 1 ? hits : 1) - 1, rest = *n - j * step;
  *lo += j * step;
  *n = step < rest ? step : rest;
}

// A batch that fits a warp: lane i has the start of sequence i, lanes from the last one on where that ends (so that
// lane b + 1 has the end of sequence b), and its number of keys.  Of the sequences `hits` start at or before the row.
constexpr int kSmallBatch = 31;
MA_HD int small_start(int lane, int num_batch) { return lane < num_batch ? lane : num_batch; }
MA_HD int small_keys(int lane, int num_batch) { return lane < num_batch ? lane : num_batch - 1; }
MA_HD int small_take(int hits) { return (hits > 1 ? hits : 1) - 1; }

// Row t of the sequence [q0, q1) with `len` keys, the new ones counted: its position, and -1 for a row
// that is not one of the sequence's or lies before its first key.
MA_HD int position_of(int t, int q0, int q1, int len) {
  if (t < q0 || t >= q1 || len < 1 || q1 - t > len) return -1;
  return len - (q1 - t);
}

// The page that holds position `pos` (-1: none), from the sequence's row of the page table.
MA_HD int page_of(int pos, const int* row, int width, int num_pages) {
  if (pos < 0 || (pos >> 7) >= width) return -1;
  const int page = row[pos >> 7];
  return page >= 0 && page < num_pages ? page : -1;
}

}  // namespace ma
