// Pages of a paged cache (gfx950): sequences that continue others, room for
// their next tokens, and live pages moved together.  No state is kept: a page is
// held while a row's first ceil(len / page_size) table entries, or `keep`, name
// it, so an ended or replaced row frees its pages by itself.  Free pages are
// given lowest first, in row order, so the result is the same on every run.
#include "bt_common.h"
#include "bt_kernels.h"

namespace bt {

namespace {

constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int row_len(const PageOpParams& p, int row) {
  if (row < 0 || row >= p.rows) return 0;
  const int64_t cap = (int64_t)p.pages_per_seq * p.page_size;
  const int64_t n = p.lens[row];
  return (int)(n < 0 ? 0 : (n > cap ? cap : n));
}
__device__ __forceinline__ int parent_of(const PageOpParams& p, int i) { return p.parent ? p.parent[i] : i; }

__global__ void pages_clear_kernel(PageOpParams p) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < p.num_pages) p.ws[i] = 0;
}

// Holders of every page, over the new rows' live entries and `keep`.
__global__ void pages_count_kernel(PageOpParams p) {
  const int64_t cells = (int64_t)p.rows_out * p.pages_per_seq;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  int id = -1;
  if (i < cells) {
    const int r = (int)(i / p.pages_per_seq), c = (int)(i % p.pages_per_seq);
    const int from = parent_of(p, r), n = row_len(p, from);
    if (c < (n + p.page_size - 1) / p.page_size) {
      id = p.table[(int64_t)from * p.pages_per_seq + c];
      if (id < 0 || id >= p.num_pages) id = -1;
    }
    p.table_out[i] = id;
    if (c == 0 && p.lens_out) p.lens_out[r] = n;
  } else if (i < cells + p.num_keep) {
    id = p.keep[i - cells];
  }
  if (id >= 0 && id < p.num_pages) atomicAdd(p.ws + id, 1);
}

// Exclusive sum of v over the work-group's threads, and the total.
__device__ int block_scan(int v, int& total, int* lds) {
  const int t = threadIdx.x;
  __syncthreads();
  lds[t] = v;
  __syncthreads();
  for (int o = 1; o < kPlanThreads; o <<= 1) {
    const int x = t >= o ? lds[t - o] : 0;
    __syncthreads();
    lds[t] += x;
    __syncthreads();
  }
  total = lds[kPlanThreads - 1];
  return lds[t] - v;
}

__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(PageOpParams p) {
  __shared__ int lds[kPlanThreads];
  int* held = p.ws;
  int* list = p.ws + p.num_pages;
  int* copies = p.ws + 2 * (int64_t)p.num_pages;
  const int t = threadIdx.x;
  int free_pages = 0, total;
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {
    const int i = base + t;
    const int is_free = i < p.num_pages && held[i] == 0;
    const int at = free_pages + block_scan(is_free, total, lds);
    if (is_free) list[at] = i;
    free_pages += total;
  }
  __syncthreads();
  int given = 0, missing = 0;
  for (int base = 0; base < p.rows_out; base += kPlanThreads) {
    const int r = base + t;
    int n = 0, used = 0, need = 0, fork = 0, over = 0;
    int32_t* row = p.table_out + (int64_t)r * p.pages_per_seq;
    if (r < p.rows_out) {
      n = row_len(p, parent_of(p, r));
      const int add = p.add && p.add[r] > 0 ? p.add[r] : 0;
      used = (n + p.page_size - 1) / p.page_size;
      const int64_t want = ((int64_t)n + add + p.page_size - 1) / p.page_size;
      need = (int)(want < p.pages_per_seq ? want : p.pages_per_seq);
      over = (int)(want - need);
      if (add > 0 && n % p.page_size) {
        const int last = row[used - 1];
        fork = last >= 0 && held[last] > 1;
      }
    }
    const int mine = need - used + fork;
    int at = given + block_scan(mine, total, lds);
    given += total;
    if (fork) {
      const int from = row[used - 1], to = at < free_pages ? list[at] : -1;
      ++at;
      row[used - 1] = to;
      copies[4 + 4 * r] = from;
      copies[4 + 4 * r + 1] = to;
      copies[4 + 4 * r + 2] = n % p.page_size;
    } else if (r < p.rows_out) {
      copies[4 + 4 * r + 1] = -1;
    }
    for (int c = used; c < need; ++c, ++at) row[c] = at < free_pages ? list[at] : -1;
    block_scan(over, total, lds);
    missing += total;
  }
  if (t == 0) {
    copies[0] = p.rows_out;
    p.status[0] = given < free_pages ? free_pages - given : 0;
    p.status[1] = missing + (given > free_pages ? given - free_pages : 0);
  }
}

__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PageOpParams p) {
  __shared__ int lds[kPlanThreads];
  int* held = p.ws;
  int* copies = p.ws + 2 * (int64_t)p.num_pages;
  const int t = threadIdx.x;
  int live = 0, total;
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {
    const int i = base + t;
    block_scan(i < p.num_pages && held[i] != 0, total, lds);
    live += total;
  }
  // Hole h (a free page below `live`) takes mover h (a held page at or past it).
  int holes = 0, movers = 0;
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {
    const int i = base + t;
    const bool in = i < p.num_pages, is_held = in && held[i] != 0;
    const int hole = in && !is_held && i < live, mover = is_held && i >= live;
    int at = holes + block_scan(hole, total, lds);
    holes += total;
    if (hole) copies[4 + 4 * at + 1] = i;
    at = movers + block_scan(mover, total, lds);
    movers += total;
    if (mover) {
      copies[4 + 4 * at] = i;
      copies[4 + 4 * at + 2] = p.page_size;
    }
    if (in && !mover) p.where[i] = is_held ? i : -1;
  }
  __syncthreads();
  for (int m = t; m < movers; m += kPlanThreads) p.where[copies[4 + 4 * m]] = copies[4 + 4 * m + 1];
  if (t == 0) {
    copies[0] = movers;
    p.status[0] = live;
  }
}

__global__ void compact_table_kernel(PageOpParams p) {
  const int64_t cells = (int64_t)p.rows_out * p.pages_per_seq;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= cells) return;
  const int id = p.table_out[i];
  if (id >= 0) p.table_out[i] = p.where[id];
}

// The plan's copies: the first `tokens` tokens of page `from` to page `to`, in every plane.
__global__ void pages_copy_kernel(PageOpParams p) {
  const int* copies = p.ws + 2 * (int64_t)p.num_pages;
  const int n = copies[0];
  const int plane = blockIdx.y;
  for (int c = blockIdx.x; c < n; c += gridDim.x) {
    const int from = copies[4 + 4 * c], to = copies[4 + 4 * c + 1], tokens = copies[4 + 4 * c + 2];
    if (to < 0) continue;
    const u32x4* src = reinterpret_cast<const u32x4*>(p.pages + plane * p.plane_stride + from * p.page_stride);
    u32x4* dst = reinterpret_cast<u32x4*>(p.pages + plane * p.plane_stride + to * p.page_stride);
    const int units = tokens * (p.token_elems / 8);
    for (int u = threadIdx.x; u < units; u += blockDim.x) dst[u] = src[u];
  }
}

hipError_t launch_count(const PageOpParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(pages_clear_kernel, dim3((p.num_pages + 255) / 256), dim3(256), 0, stream, p);
  const int64_t items = (int64_t)p.rows_out * p.pages_per_seq + p.num_keep;
  if (items) hipLaunchKernelGGL(pages_count_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fork_pages(const PageOpParams& p, hipStream_t stream) {
  hipError_t e = launch_count(p, stream);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  if (p.rows_out) hipLaunchKernelGGL(pages_copy_kernel, dim3(p.rows_out < 1024 ? p.rows_out : 1024, p.planes), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_compact_pages(const PageOpParams& p, hipStream_t stream) {
  hipError_t e = launch_count(p, stream);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  const int64_t cells = (int64_t)p.rows_out * p.pages_per_seq;
  if (cells) hipLaunchKernelGGL(compact_table_kernel, dim3((unsigned)((cells + 255) / 256)), dim3(256), 0, stream, p);
  hipLaunchKernelGGL(pages_copy_kernel, dim3(p.num_pages < 1024 ? p.num_pages : 1024, p.planes), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace bt
