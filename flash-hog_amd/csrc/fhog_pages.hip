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
// The bookkeeping is bound by latency, four dependent round trips: 5.8 us for 128 rows of 34 entries, of which the launch is
// two. The copies are bound by memory.
#include "fhog_pages.h"

namespace fhog {

namespace {

constexpr int kFree = 0x7fffffff, kRead = -1;  // PageState: else the lowest row that grows in the page

struct PageRow {
  int from = -1;             // the parent, or -1: an empty row
  long held = 0, more = 0;  // tokens held and new
  int used = 0;             // entries in use, of the table's
  bool grows = false;       // within its last page
  __device__ PageRow() = default;
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

// Entry c of row b, from what is known of it: kept for later with parents, and what it says about its page.
template <typename State, typename Row>
__device__ __forceinline__ int mark_entry(const PagesParams& p, State* state, int b, int c, const Row& row) {
  const int page = p.table[(long)row.from * p.width + c];
  if (p.parents) p.entries[(long)b * p.width + c] = page;
  if ((unsigned)page < (unsigned)p.pages) atomicMin(&state[page], row.grows && c == row.used - 1 ? b : kRead);
  return page;
}

// What row b, whose last page is `last`, asks for: how many pages; notes which column is the first and which page it copies.
template <typename State> __device__ __forceinline__ int ask(const PagesParams& p, const State* state, int b, const PageRow& row, int last) {
  const bool copies = row.grows && (unsigned)last < (unsigned)p.pages && state[last] != b;
  const int begin = row.used - copies;
  p.held[b] = (int)row.held;
  p.begin[b] = begin;
  p.source[b] = copies ? last : -1;
  return max(0, row.end(p) - begin);
}
__device__ __forceinline__ int ask(const PagesParams& p, int b) {
  const PageRow row(p, b);
  return ask(p, p.state, b, row, row.grows ? p.table[(long)row.from * p.width + row.used - 1] : -1);
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

// `bytes` bytes (a multiple of 16, both ends aligned to it) by kThreads threads; null source: zeros. kPast: stored past the
// caches, for copies larger than these (230 MB of e4m3 pages 82 us where they went to them in 106; after other work, with the
// bookkeeping, 116 and 121).
template <bool kPast, int kThreads> __device__ __forceinline__ void copy_bytes(char* to, const char* from, long bytes, int thread) {
  for (long i = 16 * thread; i < bytes; i += 16 * kThreads) {
    const u32x4 x = from ? *reinterpret_cast<const u32x4*>(from + i) : u32x4{0, 0, 0, 0};
    if constexpr (kPast)
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to + i));
    else
      *reinterpret_cast<u32x4*>(to + i) = x;
  }
}

// After the bookkeeping, by kThreads threads: row b's entries and length, by the first key/value head's, and this head's
// rows of a shared page, if it copies one.
template <int kThreads>
__device__ __forceinline__ void extend_row(const PagesParams& p, const PageBytes& cache, int* free_pages, int b, int hk, int thread) {
  const int begin = p.begin[b], first = p.first[b], source = p.source[b], listed = p.totals[0];
  const long held = p.held[b];
  if (hk == 0) {
    const long more = max(0, p.new_tokens ? p.new_tokens[b] : p.new_each);
    const long pages = (held + more + (1l << p.page_shift) - 1) >> p.page_shift;
    const int end = (int)min(pages, (long)p.width);
    int* const row = p.table + (long)b * p.width;
    for (int c = thread; c < p.width; c += kThreads) {
      if (c < begin) {
        if (p.parents) row[c] = p.entries[(long)b * p.width + c];
      } else {
        const int place = first + c - begin;
        row[c] = c < end && place < listed ? p.listed[place] : -1;
      }
    }
    if (thread == 0) {
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
      copy_bytes<false, kThreads>(to, from, (long)rows * cache.token[i], thread);
    else  // a byte a token
      for (int r = thread; r < rows; r += kThreads) to[r] = from[r];
  }
}

// All of the bookkeeping in one workgroup, a thread a row; kExtend: and what follows it.
struct FewRow {
  int from, used, grows, last;
};
template <bool kExtend> __global__ void __launch_bounds__(1024) pages_few_kernel(PagesParams p, PageBytes cache, int* free_pages) {
  __shared__ int state[kFewPages];
  __shared__ FewRow s_row[kFewRows];
  __shared__ int box[16];
  static_assert(kFewRows == 1024);
  const int b = threadIdx.x;
  PageRow row;
  if (b < p.batch) row = PageRow(p, b);
  s_row[b] = {row.from, row.used, row.grows, -1};
  for (int i = threadIdx.x; i < p.pages; i += 1024) state[i] = kFree;
  __syncthreads();
  const int entries = p.batch * p.width;
  for (int i = threadIdx.x; i < entries; i += 1024) {
    const int r = i / p.width, c = i - r * p.width;
    FewRow& of = s_row[r];
    if (c >= of.used) continue;
    const int page = mark_entry(p, state, r, c, of);
    if (c == of.used - 1) of.last = page;
  }
  __syncthreads();
  int asked;
  const int before = group_scan<1024>(b < p.batch ? ask(p, state, b, row, s_row[b].last) : 0, asked, box);
  if (b < p.batch) p.first[b] = before;
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
  if constexpr (kExtend) {
    __syncthreads();  // (what this workgroup wrote it reads)
    for (int i = wave; i < p.batch * p.kv_heads; i += 16) extend_row<64>(p, cache, free_pages, i / p.kv_heads, i % p.kv_heads, threadIdx.x & 63);
  }
}

// The same in steps, for more.
__global__ void __launch_bounds__(256) pages_clear_kernel(PagesParams p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < p.pages) p.state[i] = kFree;
}
__global__ void __launch_bounds__(256) pages_mark_kernel(PagesParams p) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)p.batch * p.width) return;
  const int b = (int)(i / p.width), c = (int)(i - (long)b * p.width);
  const PageRow row(p, b);
  if (c < row.used) mark_entry(p, p.state, b, c, row);
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
    const int before = group_scan<1024>(b < p.batch ? ask(p, b) : 0, sum, box);
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
    hipLaunchKernelGGL((pages_few_kernel<false>), dim3(1), dim3(1024), 0, stream, p, PageBytes{}, nullptr);
    return hipGetLastError();
  }
  const long entries = (long)p.batch * p.width;
  const int chunks = (p.pages + kPageChunk - 1) / kPageChunk;
  hipLaunchKernelGGL(pages_clear_kernel, dim3((p.pages + 255) / 256), dim3(256), 0, stream, p);
  if (entries > 0)  // (a cache without rows may be compacted)
    hipLaunchKernelGGL(pages_mark_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(pages_count_kernel, dim3(chunks), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(pages_scan_kernel, dim3(1), dim3(1024), 0, stream, p);
  hipLaunchKernelGGL(pages_list_kernel, dim3(chunks), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// A workgroup a row and key/value head.
__global__ void __launch_bounds__(256) pages_extend_kernel(PagesParams p, PageBytes cache, int* free_pages) {
  extend_row<256>(p, cache, free_pages, blockIdx.x, blockIdx.y, threadIdx.x);
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
    const long size = p.kv_heads * cache.row[i];  // of a page
    const long piece = (size / 16 + pieces - 1) / pieces * 16;
    const long at = piece * blockIdx.y, left = size - at;
    if (left > 0)
      copy_bytes<true, 256>(out.at[i] + page * size + at, from < 0 ? nullptr : cache.at[i] + from * size + at,
                            left < piece ? left : piece, threadIdx.x);
  }
}

}  // namespace

hipError_t launch_pages_extend(const PagesParams& p, const PageBytes& cache, int* free_pages, hipStream_t stream) {
  const long most = (long)p.batch * p.kv_heads * (cache.row[0] + cache.row[1]);  // bytes that the rows copy
  if (few_pages(p.batch, p.width, p.pages) && most <= kFewBytes && (long)p.batch * p.kv_heads <= kFewHeads) {
    hipLaunchKernelGGL((pages_few_kernel<true>), dim3(1), dim3(1024), 0, stream, p, cache, free_pages);
    return hipGetLastError();
  }
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
  const long page = p.kv_heads * cache.row[0];
  const int pieces = (int)(page >= 16384 * 64l ? 64 : page > 16384 ? page / 16384 : 1);
  hipLaunchKernelGGL(pages_compact_kernel, dim3(out_pages, pieces + 1), dim3(256), 0, stream, p, cache, out, out_pages,
                     table_out, pieces);
  return hipGetLastError();
}

}  // namespace fhog
