// Pages of a paged cache (gfx950): sequences that continue others, room for
// their next tokens, and live pages moved together.  No state is kept: a page is
// held while a row's first ceil(len / page_size) table entries, or `keep`, name
// it, so an ended or replaced row frees its pages by itself.  Free pages are
// given lowest first, in row order, so the result is the same on every run.
//
// A plan (who holds each page, which pages go where) and the copies it asks for.
// The copies are bound by memory.  The plan is a chain of short steps over little
// data, bound by latency and launches: in small caches (is_small) one work-group makes
// all of it, holders as two bits of each page in LDS (held; held twice), rows in LDS, a
// page's place from the held pages before its word of bits.  Larger ones count holders
// in memory with the whole chip; the steps between stay with one work-group.
//
// us, plan + copies: fork of 4 rows in 320 pages 4.8 + 2.5, of 128 rows in 2,048 pages of
// 12 planes 8.2 + 8.0 (31 MB); compaction of 300 pages 4.3 + 6.6, of 2,048 (395 MB read
// and written) 7.0 + 82, 4.8 TB/s, a large copy's rate.
#include "bt_common.h"
#include "bt_kernels.h"

namespace bt {

namespace {

constexpr int kThreads = 1024;
constexpr int kAhead = 8;  // table entries a thread has on their way at a time
constexpr int kSmallPages = 1 << 18, kSmallRows = 2048;  // what LDS holds

// A row of the result: where it comes from, its tokens, the entries it will have,
// and the rank among the pages given of its first one.
struct Row {
  int from, n, need, at;  // from: its sign bit is set where the last page is copied
};

__device__ __forceinline__ int pages_of(const PageOpParams& p, int tokens) { return (tokens + p.page_size - 1) >> p.page_shift; }

// The row that new row r continues, its tokens, and (fork) the entries needed; `over`: entries the table lacks,
// at most so many that their sum over the rows fits 31 bits.
__device__ __forceinline__ Row read_row(const PageOpParams& p, int r, int& over) {
  const int from = p.parent ? p.parent[r] : r;
  const int cap = p.pages_per_seq * p.page_size;
  Row row{0, 0, 0, 0};
  if (from >= 0 && from < p.rows) {
    const int n = p.lens[from];
    row.from = from;
    row.n = n < 0 ? 0 : (n > cap ? cap : n);
  }
  const int add = p.add && p.add[r] > 0 ? p.add[r] : 0;
  const int64_t want = ((int64_t)row.n + add + p.page_size - 1) >> p.page_shift;
  row.need = (int)(want < p.pages_per_seq ? want : p.pages_per_seq);
  const int64_t lacking = want - row.need, most = (1 << 30) / p.rows_out;
  over = (int)(lacking < most ? lacking : most);
  // Rows without new tokens write nowhere: marked by need = -1 - need.
  if (add == 0) row.need = -1 - row.need;
  return row;
}
// A live entry of a row, -1 outside the cache.
__device__ __forceinline__ int read_entry(const PageOpParams& p, const Row& row, int c) {
  const int id = p.table[(row.from & 0x7fffffff) * p.pages_per_seq + c];
  return id >= 0 && id < p.num_pages ? id : -1;
}

// Exclusive sum of v over the work-group's threads, and the total.
__device__ __forceinline__ int block_scan(int v, int& total, int* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int x = wave_scan(v);
  __syncthreads();  // the sums of the scan before are read
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  const int s = wave_scan(lane < kThreads / 64 ? lds[lane] : 0);
  total = __builtin_amdgcn_readlane(s, kThreads / 64 - 1);
  return x - v + (wave > 0 ? __builtin_amdgcn_readlane(s, wave - 1) : 0);
}

// Holders of the pages, 0, 1 or more: bits in LDS, or counts in memory.
template <bool SMALL>
struct Holders {
  uint32_t* once;
  uint32_t* twice;
  const int* count;
  template <int N>
  __device__ __forceinline__ void mark(const int (&id)[N]) {  // those that are not negative
    uint32_t old[N];
#pragma unroll
    for (int j = 0; j < N; ++j) old[j] = id[j] >= 0 ? atomicOr(once + (id[j] >> 5), 1u << (id[j] & 31)) : 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (id[j] >= 0 && old[j] >> (id[j] & 31) & 1) atomicOr(twice + (id[j] >> 5), 1u << (id[j] & 31));
  }
  __device__ __forceinline__ bool held(int id) const {
    if constexpr (SMALL) return once[id >> 5] >> (id & 31) & 1;
    else return count[id] != 0;
  }
  __device__ __forceinline__ bool shared(int id) const {
    if constexpr (SMALL) return twice[id >> 5] >> (id & 31) & 1;
    else return count[id] > 1;
  }
};

// Held pages before each word of a small cache's bits, by the whole work-group; all of them in `held`.
__device__ __forceinline__ void words_before(const PageOpParams& p, const Holders<true>& h, int* before, int& held, int* lds) {
  const int words = (p.num_pages + 31) / 32, run = (words + kThreads - 1) / kThreads, first = (int)threadIdx.x * run;
  int mine = 0;
  for (int i = first; i < first + run && i < words; ++i) mine += __popc(h.once[i]);
  int at = block_scan(mine, held, lds);
  for (int i = first; i < first + run && i < words; ++i) {
    before[i] = at;
    at += __popc(h.once[i]);
  }
  __syncthreads();
}
__device__ __forceinline__ int held_before(const Holders<true>& h, const int* before, int id) {
  return before[id >> 5] + __popc(h.once[id >> 5] & ((1u << (id & 31)) - 1));
}

// A thread's walk over the (row, column) cells t, t + kThreads, ...: one work-group does
// all of a small cache's, so a division for each would be most of the work.
struct Walk {
  int r, c, dr, dc, per_row;
  __device__ __forceinline__ explicit Walk(int columns)
      : r((int)threadIdx.x / columns), c((int)threadIdx.x % columns), dr(kThreads / columns), dc(kThreads % columns), per_row(columns) {}
  __device__ __forceinline__ void step() {
    r += dr;
    c += dc;
    if (c >= per_row) {
      c -= per_row;
      ++r;
    }
  }
};

// Rows and holders of a small cache, by one work-group.
__device__ __forceinline__ void small_holders(const PageOpParams& p, Holders<true>& h, Row* rows, int& over_sum) {
  const int t = threadIdx.x;
  for (int i = t; i < (p.num_pages + 31) / 32; i += kThreads) h.once[i] = h.twice[i] = 0;
  over_sum = 0;
  for (int r = t; r < p.rows_out; r += kThreads) {
    int over;
    rows[r] = read_row(p, r, over);
    over_sum += over;
    if (p.lens_out) p.lens_out[r] = rows[r].n;
  }
  __syncthreads();
  const int cells = p.rows_out * p.pages_per_seq;
  Walk cell(p.pages_per_seq);
  for (int i0 = t; i0 < cells; i0 += kAhead * kThreads) {
    int id[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j, cell.step()) {
      id[j] = -1;
      if (cell.r < p.rows_out) {
        const Row row = rows[cell.r];
        if (cell.c * p.page_size < row.n) id[j] = read_entry(p, row, cell.c);
      }
    }
    h.mark(id);
  }
  for (int i = t; i < p.num_keep; i += kThreads) {
    const int id = p.keep[i];
    const int one[1] = {id < p.num_pages ? id : -1};
    h.mark(one);
  }
  __syncthreads();
}

// The same for a large one, over the whole chip; rows in the workspace.
struct Layout {
  int* count;   // (num_pages)
  int* list;    // (num_pages) free pages; compact: holes
  int* copies;  // {number}, then {from, to, tokens, -} each
  Row* rows;    // (rows_out)
};
__host__ __device__ __forceinline__ Layout layout_of(const PageOpParams& p) {
  Layout l;
  const int64_t most = p.num_pages > p.rows_out ? p.num_pages : p.rows_out;
  l.copies = p.ws;
  l.rows = reinterpret_cast<Row*>(p.ws + 4 + 4 * most);
  l.count = p.ws + 4 + 4 * most + 4 * (int64_t)p.rows_out;
  l.list = l.count + p.num_pages;
  return l;
}

__global__ void pages_clear_kernel(PageOpParams p) {
  const Layout l = layout_of(p);
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < p.num_pages) l.count[i] = 0;
}

__global__ void pages_count_kernel(PageOpParams p) {
  const Layout l = layout_of(p);
  const int64_t cells = (int64_t)p.rows_out * p.pages_per_seq;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  int id = -1;
  if (i < cells) {
    const int r = (int)(i / p.pages_per_seq), c = (int)(i % p.pages_per_seq);
    int over;
    const Row row = read_row(p, r, over);
    if (c < pages_of(p, row.n)) id = read_entry(p, row, c);
    if (c == 0) {
      l.rows[r] = row;
      if (p.lens_out) p.lens_out[r] = row.n;
    }
  } else if (i < cells + p.num_keep) {
    id = p.keep[i - cells];
  }
  if (id >= 0 && id < p.num_pages) atomicAdd(l.count + id, 1);
}

template <bool SMALL>
__global__ __launch_bounds__(kThreads) void fork_plan_kernel(PageOpParams p) {
  __shared__ uint32_t bits[SMALL ? 2 * (kSmallPages / 32) : 1];
  __shared__ int before[SMALL ? kSmallPages / 32 : 1];
  __shared__ Row small_rows[SMALL ? kSmallRows : 1];
  __shared__ int lds[kThreads / 64];
  const Layout l = layout_of(p);
  const int t = threadIdx.x;
  Holders<SMALL> h{bits, bits + kSmallPages / 32, l.count};
  Row* rows = SMALL ? small_rows : l.rows;
  __shared__ int over_sum;
  if (t == 0) over_sum = 0;
  int total, over = 0;
  if constexpr (SMALL) {
    small_holders(p, h, rows, over);
  } else {
    for (int r = t; r < p.rows_out; r += kThreads) {
      int o;
      read_row(p, r, o);
      over += o;
    }
  }
  // Pages each row is given: a copy's first, then those of its new tokens.
  int given = 0;
  for (int base = 0; base < p.rows_out; base += kThreads) {
    const int r = base + t;
    int mine = 0;
    Row row{0, 0, 0, 0};
    if (r < p.rows_out) {
      row = rows[r];
      const int used = pages_of(p, row.n);
      if (row.need < 0) {
        row.need = -1 - row.need;
      } else if ((row.n & (p.page_size - 1))) {
        const int last = read_entry(p, row, used - 1);
        if (last >= 0 && h.shared(last)) row.from |= (int)0x80000000;
      }
      mine = row.need - used + (row.from < 0);
    }
    row.at = given + block_scan(mine, total, lds);
    if (r < p.rows_out) rows[r] = row;
    given += total;
  }
  // Free pages in order, as many as are given.
  int free_pages;
  if constexpr (SMALL) {
    int held;
    words_before(p, h, before, held, lds);
    free_pages = p.num_pages - held;
    for (int base = 0; base < p.num_pages && base - before[base >> 5] < given; base += kThreads) {
      const int id = base + t, rank = id < p.num_pages ? id - held_before(h, before, id) : given;
      if (rank < given && !h.held(id)) l.list[rank] = id;
    }
  } else {  // a thread takes a run of pages
    const int run = (p.num_pages + kThreads - 1) / kThreads;
    const int64_t first = (int64_t)t * run;
    int mine = 0;
    for (int i = 0; i < run && first + i < p.num_pages; ++i) mine += !h.held((int)first + i);
    int at = block_scan(mine, free_pages, lds);
    for (int i = 0; i < run && first + i < p.num_pages && at < given; ++i)
      if (!h.held((int)first + i)) l.list[at++] = (int)first + i;
  }
  if (over) atomicAdd(&over_sum, over);
  __syncthreads();  // also: the list and the rows are written
  if (t == 0) {
    l.copies[0] = p.rows_out;
    l.copies[1] = free_pages;
    p.status[0] = given < free_pages ? free_pages - given : 0;
    const int64_t missing = (int64_t)over_sum + (given > free_pages ? given - free_pages : 0);
    p.status[1] = (int)(missing < INT32_MAX ? missing : INT32_MAX);
  }
  for (int r = t; r < p.rows_out; r += kThreads) {
    const Row row = rows[r];
    int* copy = l.copies + 4 + 4 * (int64_t)r;
    copy[1] = -1;
    if (row.from < 0) {
      const int last = pages_of(p, row.n) - 1, to = row.at < free_pages ? l.list[row.at] : -1;
      copy[0] = read_entry(p, row, last);
      copy[1] = to;
      copy[2] = (row.n & (p.page_size - 1));
    }
    if constexpr (SMALL) l.rows[r] = row;
  }
}

template <bool SMALL>
__global__ __launch_bounds__(kThreads) void compact_plan_kernel(PageOpParams p) {
  __shared__ uint32_t bits[SMALL ? 2 * (kSmallPages / 32) : 1];
  __shared__ int before[SMALL ? kSmallPages / 32 : 1];
  __shared__ Row small_rows[SMALL ? kSmallRows : 1];
  __shared__ int lds[kThreads / 64];
  const Layout l = layout_of(p);
  const int t = threadIdx.x;
  Holders<SMALL> h{bits, bits + kSmallPages / 32, l.count};
  int over;
  if constexpr (SMALL) small_holders(p, h, small_rows, over);
  // The free places below the number of live pages (holes) and the held pages at or past it (movers)
  // are as many; with n held pages before page i, i - n holes come before it, or n - (held pages
  // before page `live`) movers.
  int live, below;  // held pages before page `live`
  auto place = [&](int id, bool held, int n) {
    if (held && id >= live) l.copies[4 + 4 * (int64_t)(n - below)] = id;
    else p.where[id] = held ? id : -1;
    if (!held && id < live) l.list[id - n] = id;
  };
  if constexpr (SMALL) {
    words_before(p, h, before, live, lds);
    below = live < p.num_pages ? held_before(h, before, live) : live;
    for (int id = t; id < p.num_pages; id += kThreads) place(id, h.held(id), held_before(h, before, id));
  } else {  // a thread takes a run of pages
    __shared__ int below_live;
    const int run = (p.num_pages + kThreads - 1) / kThreads;
    const int64_t first = (int64_t)t * run;
    int mine = 0;
    for (int i = 0; i < run && first + i < p.num_pages; ++i) mine += h.held((int)first + i);
    int n = block_scan(mine, live, lds);
    if (live < p.num_pages && first <= live && live < first + run) {  // one thread
      int m = n;
      for (int i = 0; first + i < live; ++i) m += h.held((int)first + i);
      below_live = m;
    }
    __syncthreads();
    below = live < p.num_pages ? below_live : live;
    for (int i = 0; i < run && first + i < p.num_pages; ++i) {
      const bool held = h.held((int)first + i);
      place((int)first + i, held, n);
      n += held;
    }
  }
  const int total = live - below;
  __syncthreads();
  for (int m = t; m < total; m += kThreads) {
    int* copy = l.copies + 4 + 4 * (int64_t)m;
    const int to = l.list[m];
    copy[1] = to;
    copy[2] = p.page_size;
    p.where[copy[0]] = to;
  }
  if (t == 0) {
    l.copies[0] = total;
    p.status[0] = live;
  }
}

// What a plan asks for, over the whole chip: the copies, and the new table's entries.
// A copy is the first `tokens` tokens of page `from` to page `to`, in every plane; no page
// is both copied and copied to, so their order does not matter.
constexpr int kApplyThreads = 256, kCopyLoads = 4;
template <bool FORK>
__global__ __launch_bounds__(kApplyThreads) void pages_apply_kernel(PageOpParams p, int copy_groups) {
  const Layout l = layout_of(p);
  if ((int)blockIdx.x < copy_groups * p.planes) {
    const int n = l.copies[0];
    const int64_t plane = (int64_t)(blockIdx.x / copy_groups) * p.plane_stride;
    for (int c = blockIdx.x % copy_groups; c < n; c += copy_groups) {
      const int* copy = l.copies + 4 + 4 * (int64_t)c;
      if (copy[1] < 0) continue;
      const u32x4* src = reinterpret_cast<const u32x4*>(p.pages + plane + copy[0] * p.page_stride);
      u32x4* dst = reinterpret_cast<u32x4*>(p.pages + plane + copy[1] * p.page_stride);
      const int units = copy[2] * (p.token_elems / 8);
      int u = threadIdx.x;
      for (; u + (kCopyLoads - 1) * kApplyThreads < units; u += kCopyLoads * kApplyThreads) {
        u32x4 x[kCopyLoads];
#pragma unroll
        for (int i = 0; i < kCopyLoads; ++i) x[i] = src[u + i * kApplyThreads];
#pragma unroll
        for (int i = 0; i < kCopyLoads; ++i) dst[u + i * kApplyThreads] = x[i];
      }
      for (; u < units; u += kApplyThreads) dst[u] = src[u];
    }
    return;
  }
  const int64_t i = (int64_t)(blockIdx.x - copy_groups * p.planes) * kApplyThreads + threadIdx.x;
  if (i >= (int64_t)p.rows_out * p.pages_per_seq) return;
  const int r = (int)(i / p.pages_per_seq), c = (int)(i % p.pages_per_seq);
  int id = -1;
  if constexpr (FORK) {
    const Row row = l.rows[r];
    const int used = pages_of(p, row.n);
    if (c == used - 1 && row.from < 0) {
      id = l.copies[4 + 4 * (int64_t)r + 1];
    } else if (c < used) {
      id = read_entry(p, row, c);
    } else if (c < row.need) {
      const int rank = row.at + (row.from < 0) + c - used;
      if (rank < l.copies[1]) id = l.list[rank];
    }
  } else {
    int over;
    const Row row = read_row(p, r, over);
    if (c < pages_of(p, row.n)) {
      id = read_entry(p, row, c);
      if (id >= 0) id = p.where[id];
    }
  }
  p.table_out[i] = id;
}

// One work-group reads 2^16 table entries in 22 us; the whole chip needs two more launches, and the one
// work-group of its other steps time for each page.  us of a fork (a compaction), one work-group / the chip: 128
// rows of 128 entries in 8,192 pages 13.5 (13.3) / 17.7 (20.7), of 256 18.9 (17.6) / 18.4 (20.4), of 512 29.6
// (26.8) / 20.6 (21.4); 256 of 512 in 32,768 pages 49 (52) / 37 (76); 1,024 of 512 in 2^18 169 (339) / 184 (565).
bool is_small(const PageOpParams& p) {
  return p.num_pages <= kSmallPages && p.rows_out <= kSmallRows &&
         (int64_t)p.rows_out * p.pages_per_seq + p.num_keep <= (1 << 15) + 2 * p.num_pages;
}

dim3 per_cell(int64_t n) { return dim3((unsigned)((n + 255) / 256)); }

void launch_count(const PageOpParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(pages_clear_kernel, per_cell(p.num_pages), dim3(256), 0, stream, p);
  const int64_t items = (int64_t)p.rows_out * p.pages_per_seq + p.num_keep;
  if (items) hipLaunchKernelGGL(pages_count_kernel, per_cell(items), dim3(256), 0, stream, p);
}

template <bool FORK>
void launch_apply(const PageOpParams& p, int copies, hipStream_t stream) {
  const int groups = copies < 1024 ? copies : 1024;
  const int64_t cells = (int64_t)p.rows_out * p.pages_per_seq;
  const int64_t grid = (int64_t)groups * p.planes + (cells + kApplyThreads - 1) / kApplyThreads;
  if (grid) hipLaunchKernelGGL(pages_apply_kernel<FORK>, dim3((unsigned)grid), dim3(kApplyThreads), 0, stream, p, groups);
}

}  // namespace

int64_t page_ws_ints(int64_t num_pages, int64_t rows_out) {
  const int64_t most = num_pages > rows_out ? num_pages : rows_out;
  return 4 + 4 * most + 4 * rows_out + 2 * num_pages;
}

hipError_t launch_fork_pages(const PageOpParams& p, hipStream_t stream) {
  if (is_small(p)) {
    hipLaunchKernelGGL(fork_plan_kernel<true>, dim3(1), dim3(kThreads), 0, stream, p);
  } else {
    launch_count(p, stream);
    hipLaunchKernelGGL(fork_plan_kernel<false>, dim3(1), dim3(kThreads), 0, stream, p);
  }
  launch_apply<true>(p, p.add ? p.rows_out : 0, stream);  // without new tokens nothing is written, so nothing copied
  return hipGetLastError();
}

hipError_t launch_compact_pages(const PageOpParams& p, hipStream_t stream) {
  if (is_small(p)) {
    hipLaunchKernelGGL(compact_plan_kernel<true>, dim3(1), dim3(kThreads), 0, stream, p);
  } else {
    launch_count(p, stream);
    hipLaunchKernelGGL(compact_plan_kernel<false>, dim3(1), dim3(kThreads), 0, stream, p);
  }
  launch_apply<false>(p, p.num_pages, stream);
  return hipGetLastError();
}

}  // namespace bt
