// The paged cache's allocator on the device: rows of a page table go on from their parents and grow, and
// the used pages of a cache move to the front of another (fhog_pages.h).
//
// The table and the lengths are all there is to know: a page is used if some row has it among its first
// ceil(length / page_size) entries, else free. A row that grows within its last page must have that page for
// itself: it keeps it if every other user grows in it too and has a higher index, else it gets a copy. So
// one number a page is enough, the smallest that its users give: -1 from a user that goes on
// reading it as it is, its index from a row that grows in it, and none from nobody (PageState).
//
// New pages are the free ones, lowest first, to the rows in their order, each row's columns in theirs:
// sums over rows and pages give every row its place, whatever order the atomics ran in.
//
// The bookkeeping is bound by latency (a few dependent round trips), the copies by memory.
#include "fhog_pages.h"

namespace fhog {

namespace {

constexpr int kFree = 0x7fffffff, kRead = -1;  // PageState: else the lowest row that grows in the page

struct PageRow {
  int from;         // the parent, or -1: an empty row
  long held, more;  // tokens held and new
  int used;         // entries in use, of the table's
  bool grows;       // within its last page
  __device__ __forceinline__ PageRow(const PagesParams& p, int b) {
    from = p.parents ? p.parents[b] : b;
    if ((unsigned)from >= (unsigned)p.batch) from = -1;
    held = from < 0 ? 0 : max(0, p.lengths[from]);
    more = max(0, p.new_tokens ? p.new_tokens[b] : p.new_each);
    const long pages = (held + (1l << p.page_shift) - 1) >> p.page_shift;
    used = (int)min(pages, (long)p.width);
    grows = more > 0 && pages <= p.width && (held & ((1l << p.page_shift) - 1)) != 0;
  }
  __device__ __forceinline__ int end(const PagesParams& p) const {
    return (int)min((held + more + (1l << p.page_shift) - 1) >> p.page_shift, (long)p.width);
  }
};

// Entry i of all rows: kept for later with parents, and what it says about its page.
template <typename State> __device__ __forceinline__ void mark_entry(const PagesParams& p, State* state, long i) {
  const int b = (int)(i / p.width), c = (int)(i - (long)b * p.width);
  const PageRow row(p, b);
  if (c >= row.used) return;
  const int page = p.table[(long)row.from * p.width + c];
  if (p.parents) p.entries[i] = page;
  if ((unsigned)page < (unsigned)p.pages) atomicMin(&state[page], row.grows && c == row.used - 1 ? b : kRead);
}

// What row b asks for: how many pages; notes which column is the first and which page it copies.
__device__ __forceinline__ int ask(const PagesParams& p, const int* state, int b) {
  const PageRow row(p, b);
  int begin = row.used, source = -1;
  if (row.grows) {
    const int page = p.table[(long)row.from * p.width + row.used - 1];
    if ((unsigned)page < (unsigned)p.pages && state[page] != b) {
      source = page;
      --begin;
    }
  }
  p.held[b] = (int)row.held;
  p.begin[b] = begin;
  p.source[b] = source;
  return max(0, row.end(p) - begin);
}

__device__ __forceinline__ bool is_listed(const PagesParams& p, int state) { return (state == kFree) != (p.list_used != 0); }

// Lists pages [from, to), `first` of which come before; by one wave.
template <typename State>
__device__ __forceinline__ void list_pages(const PagesParams& p, const State* state, int from, int to, int first) {
  const int lane = threadIdx.x & 63;
  for (int at = from; at < to; at += 64) {
    const int page = at + lane;
    const bool mine = page < to && is_listed(p, state[page]);
    const unsigned long all = __ballot(mine);
    if (mine) {
      const int place = first + __popcll(all & ((1ul << lane) - 1));
      p.listed[place] = page;
      if (p.list_used) p.place[page] = place;
    }
    first += __popcll(all);
  }
}
template <typename State>
__device__ __forceinline__ int count_pages(const PagesParams& p, const State* state, int from, int to) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int at = from; at < to; at += 64) sum += __popcll(__ballot(at + lane < to && is_listed(p, state[min(at + lane, to - 1)])));
  return sum;
}

// All of the bookkeeping in one workgroup.
__global__ void __launch_bounds__(1024) pages_few_kernel(PagesParams p) {
  __shared__ int state[kFewPages];
  __shared__ int box[16];
  for (int i = threadIdx.x; i < p.pages; i += 1024) state[i] = kFree;
  __syncthreads();
  const long entries = (long)p.batch * p.width;
  for (long i = threadIdx.x; i < entries; i += 1024) mark_entry(p, state, i);
  __syncthreads();
  int asked = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 1024) {
    const int b = b0 + (int)threadIdx.x;
    int sum;
    const int before = group_scan<1024>(b < p.batch ? ask(p, state, b) : 0, sum, box);
    if (b < p.batch) p.first[b] = asked + before;
    asked += sum;
  }
  // Each wave lists a run of pages.
  const int wave = threadIdx.x >> 6, run = ((p.pages + 16 * 64 - 1) / (16 * 64)) * 64;
  const int from = min(p.pages, wave * run), to = min(p.pages, from + run);
  const int mine = count_pages(p, state, from, to);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) box[wave] = mine;
  __syncthreads();
  int first = 0, total = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) first += box[w];
    total += box[w];
  }
  list_pages(p, state, from, to, first);
  if (threadIdx.x == 0) {
    p.totals[0] = total;
    p.totals[1] = asked;
  }
}

// The same in steps, for more.
__global__ void __launch_bounds__(256) pages_clear_kernel(PagesParams p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < p.pages) p.state[i] = kFree;
}
__global__ void __launch_bounds__(256) pages_mark_kernel(PagesParams p) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i < (long)p.batch * p.width) mark_entry(p, p.state, i);
}
__global__ void __launch_bounds__(256) pages_count_kernel(PagesParams p) {
  __shared__ int box[4];
  const int wave = threadIdx.x >> 6;
  const int from = blockIdx.x * kPageChunk + wave * (kPageChunk / 4), to = min(p.pages, from + kPageChunk / 4);
  const int sum = from < to ? count_pages(p, p.state, from, to) : 0;
  if ((threadIdx.x & 63) == 0) box[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) p.chunks[blockIdx.x] = box[0] + box[1] + box[2] + box[3];
}
__global__ void __launch_bounds__(1024) pages_scan_kernel(PagesParams p) {
  __shared__ int box[16];
  int asked = 0, listed = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 1024) {
    const int b = b0 + (int)threadIdx.x;
    int sum;
    const int before = group_scan<1024>(b < p.batch ? ask(p, p.state, b) : 0, sum, box);
    if (b < p.batch) p.first[b] = asked + before;
    asked += sum;
  }
  const int chunks = (p.pages + kPageChunk - 1) / kPageChunk;
  for (int c0 = 0; c0 < chunks; c0 += 1024) {
    const int c = c0 + (int)threadIdx.x;
    int sum;
    const int before = group_scan<1024>(c < chunks ? p.chunks[c] : 0, sum, box);
    if (c < chunks) p.chunks[c] = listed + before;
    listed += sum;
  }
  if (threadIdx.x == 0) {
    p.totals[0] = listed;
    p.totals[1] = asked;
  }
}
__global__ void __launch_bounds__(256) pages_list_kernel(PagesParams p) {
  __shared__ int box[4];
  const int wave = threadIdx.x >> 6;
  const int from = blockIdx.x * kPageChunk + wave * (kPageChunk / 4), to = min(p.pages, from + kPageChunk / 4);
  const int sum = from < to ? count_pages(p, p.state, from, to) : 0;
  if ((threadIdx.x & 63) == 0) box[wave] = sum;
  __syncthreads();
  int first = p.chunks[blockIdx.x];
  for (int w = 0; w < wave; ++w) first += box[w];
  if (from < to) list_pages(p, p.state, from, to, first);
}

hipError_t bookkeeping(const PagesParams& p, hipStream_t stream) {
  if (few_pages(p.batch, p.width, p.pages)) {
    hipLaunchKernelGGL(pages_few_kernel, dim3(1), dim3(1024), 0, stream, p);
    return hipGetLastError();
  }
  const long entries = (long)p.batch * p.width;
  const int chunks = (p.pages + kPageChunk - 1) / kPageChunk;
  hipLaunchKernelGGL(pages_clear_kernel, dim3((p.pages + 255) / 256), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(pages_mark_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(pages_count_kernel, dim3(chunks), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(pages_scan_kernel, dim3(1), dim3(1024), 0, stream, p);
  hipLaunchKernelGGL(pages_list_kernel, dim3(chunks), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// `bytes` bytes (a multiple of 16, both ends aligned to it) by the workgroup; null source: zeros. kPast: stored past the
// caches, for copies larger than these (230 MB of e4m3 pages 82 us where they went to them in 106; after other work, with the
// bookkeeping, 116 and 121).
template <bool kPast> __device__ __forceinline__ void copy_bytes(char* to, const char* from, int bytes) {
  for (int i = 16 * (int)threadIdx.x; i < bytes; i += 16 * 256) {
    const u32x4 x = from ? *reinterpret_cast<const u32x4*>(from + i) : u32x4{0, 0, 0, 0};
    if constexpr (kPast)
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to + i));
    else
      *reinterpret_cast<u32x4*>(to + i) = x;
  }
}

// A workgroup a row and key/value head, whose rows of a shared page it copies if there are any; the
// first of a row's writes its entries and length too.
__global__ void __launch_bounds__(256) pages_extend_kernel(PagesParams p, PageBytes cache, int* free_pages) {
  const int b = blockIdx.x, hk = blockIdx.y;
  const int begin = p.begin[b], first = p.first[b], source = p.source[b], listed = p.totals[0];
  const long held = p.held[b];
  if (hk == 0) {
    const long more = max(0, p.new_tokens ? p.new_tokens[b] : p.new_each);
    const long pages = (held + more + (1l << p.page_shift) - 1) >> p.page_shift;
    const int end = (int)min(pages, (long)p.width);
    int* const row = p.table + (long)b * p.width;
    for (int c = threadIdx.x; c < p.width; c += 256) {
      if (c < begin) {
        if (p.parents) row[c] = p.entries[(long)b * p.width + c];
      } else {
        const int place = first + c - begin;
        row[c] = c < end && place < listed ? p.listed[place] : -1;
      }
    }
    if (threadIdx.x == 0) {
      p.lengths[b] = (int)min(held + more, 0x7fffffffl);
      if (b == 0) *free_pages = listed - p.totals[1];
    }
  }
  if (source < 0 || first >= listed) return;
  const int target = p.listed[first], rows = (int)(held & ((1l << p.page_shift) - 1));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!cache.at[i]) continue;
    char* to = cache.at[i] + ((long)target * p.kv_heads + hk) * cache.row[i];
    const char* from = cache.at[i] + ((long)source * p.kv_heads + hk) * cache.row[i];
    if (i < 2)
      copy_bytes<false>(to, from, rows * cache.token[i]);
    else  // a byte a token
      for (int r = threadIdx.x; r < rows; r += 256) to[r] = from[r];
  }
}

// Workgroups y take the tensors' pieces of a page in turn, the last of y the table.
__global__ void __launch_bounds__(256) pages_compact_kernel(PagesParams p, PageBytes cache, PageBytes out, int out_pages,
                                                            int* table_out, int pieces) {
  if ((int)blockIdx.y == pieces) {
    const long entries = (long)p.batch * p.width;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < entries; i += (long)gridDim.x * 256) {
      const int b = (int)(i / p.width), c = (int)(i - (long)b * p.width);
      int to = -1;
      if (c < PageRow(p, b).used) {
        const int page = p.table[i];
        if ((unsigned)page < (unsigned)p.pages) to = p.place[page];
        if (to >= out_pages) to = -1;
      }
      table_out[i] = to;
    }
    return;
  }
  const int page = blockIdx.x;
  const long from = page < p.totals[0] ? p.listed[page] : -1;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    if (!cache.at[i]) continue;
    const long size = (long)p.kv_heads * cache.row[i];  // of a page
    const long piece = (size / 16 + pieces - 1) / pieces * 16;
    const long at = piece * blockIdx.y, left = size - at;
    if (left > 0)
      copy_bytes<true>(out.at[i] + page * size + at, from < 0 ? nullptr : cache.at[i] + from * size + at,
                 (int)(left < piece ? left : piece));
  }
}

}  // namespace

hipError_t launch_pages_extend(const PagesParams& p, const PageBytes& cache, int* free_pages, hipStream_t stream) {
  const hipError_t e = bookkeeping(p, stream);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pages_extend_kernel, dim3(p.batch, p.kv_heads), dim3(256), 0, stream, p, cache, free_pages);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesParams& p, const PageBytes& cache, const PageBytes& out, int out_pages,
                                int* table_out, hipStream_t stream) {
  const hipError_t e = bookkeeping(p, stream);
  if (e != hipSuccess) return e;
  // about 16 KB of a tensor a workgroup
  const long page = (long)p.kv_heads * cache.row[0];
  const int pieces = (int)(page >= 16384 * 64l ? 64 : page > 16384 ? page / 16384 : 1);
  hipLaunchKernelGGL(pages_compact_kernel, dim3(out_pages, pieces + 1), dim3(256), 0, stream, p, cache, out, out_pages,
                     table_out, pieces);
  return hipGetLastError();
}

}  // namespace fhog
