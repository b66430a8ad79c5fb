// The paged cache's allocator: parameter blocks and the split of its work (fhog_pages.hip).
#pragma once

#include "fhog_paged.h"

namespace fhog {

// A cache as bytes: page p of tensor i is rows [p * kv_heads, (p + 1) * kv_heads) of `row` bytes.
struct PageBytes {
  char* at[5];    // keys, values, their scales, key means; null: none
  long row[5];    // bytes of one head in a page (2^31 and more with large pages)
  int token[5];   // bytes of one token of one head (0: not by token)
};

struct PagesParams {
  int* table;  // (batch, width)
  int* lengths;
  const int* parents;     // null: each row its own
  const int* new_tokens;  // null: new_each
  int new_each;
  int batch, width, pages, page_shift, kv_heads;
  int list_used;  // whether the used pages are listed instead of the free ones
  // workspace
  int* state;      // (pages) PageState, where LDS is too small
  int* listed;     // (pages) the free (used) pages, lowest first
  int* place;      // (pages) a used page's place in that list (list_used)
  int* entries;    // (batch, width) the rows' entries before they grow (with parents)
  int* held;       // (batch) lengths before
  int* begin;      // (batch) first column that gets a new page
  int* first;      // (batch) how many new pages the rows before get
  int* source;     // (batch) page to copy to the first new one, or -1
  int* chunks;     // listed pages before each chunk of kPageChunk
  int* totals;     // [0] pages listed, [1] pages asked for
};

constexpr int kPageChunk = 4096;
// Up to this many pages, entries and rows one workgroup does the bookkeeping, with the pages' states in LDS: six launches
// become two. The limits are LDS' (pages), a thread a row (rows), and 128 entries a thread. (us a step of one token a row,
// page of 16 and one head, one workgroup / launches: 128 rows of 34 columns 10 / 25, 64 of 128 13 / 26, 64 of 256 16 / 26, 16 of
// 1024 18 / 26, 64 of 512 33 / 27, 256 of 128 32 / 27, 64 of 1024 45 / 27, 256 of 512 76 / 27, 1024 of 128 82 / 28: the two cross at
// about 25000 entries, and from there to the limit one workgroup is the slower way.)
constexpr int kFewPages = 32768, kFewEntries = 1 << 17, kFewRows = 1024;
// And one, if the copies are no more than this at most, a wave a row and head. (us, two launches / one, without / with a copy a
// row: 1 row of 4 heads of 64, pages of 16 5.0 / 3.9, 4 5.6 / 4.3 and 6.0 / 4.9, 8, 128 KB 5.8 / 4.9 and 6.0 / 6.3, 16 6.2 / 6.5
// and 6.5 / 9.2; 2 of 8 heads of 128, pages of 64, 512 KB 5.8 / 4.0 and 6.3 / 7.0, 4 5.7 / 4.6 and 6.1 / 11.6.)
constexpr long kFewBytes = 128l << 10, kFewHeads = 32;
inline bool few_pages(int batch, int width, int pages) {
  return pages <= kFewPages && (long)batch * width <= kFewEntries && batch <= kFewRows;
}
inline long pages_workspace_ints(int batch, int width, int pages) {
  return 3l * pages + (long)batch * width + 4l * batch + pages / kPageChunk + 2 + 2;
}
inline void pages_workspace(PagesParams& p, int* ws) {
  p.totals = ws;
  p.listed = p.totals + 2;
  p.state = p.listed + p.pages;
  p.place = p.state + p.pages;
  p.held = p.place + p.pages;
  p.begin = p.held + p.batch;
  p.first = p.begin + p.batch;
  p.source = p.first + p.batch;
  p.chunks = p.source + p.batch;
  p.entries = p.chunks + p.pages / kPageChunk + 2;
}

// Extends the rows and copies the shared pages' held rows; *free_pages = free pages left, less those that
// were lacking.
hipError_t launch_pages_extend(const PagesParams& p, const PageBytes& cache, int* free_pages, hipStream_t s);
// The used pages to the front of `out`, of out_pages pages, zeros behind; the table for it to table_out.
hipError_t launch_pages_compact(const PagesParams& p, const PageBytes& cache, const PageBytes& out, int out_pages,
                                int* table_out, hipStream_t s);

}  // namespace fhog
