// The C ABI of the paged cache's operators: argument checks and launches.
// Declarations and documentation live in include/breezetoken_amd.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "../../include/breezetoken_amd.h"
#include "bt_kernels.h"

namespace {

constexpr double kLog2e = 1.4426950408889634;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
inline bool dtype_known(int32_t t) { return t == BT_DTYPE_F32 || t == BT_DTYPE_BF16; }
inline int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }
inline int hip_rc(hipError_t e) { return e == hipSuccess ? BT_OK : (int)e; }
inline int log2_of(int32_t x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

// Pages and table of a cache.
int check_paged(const void* k, const void* v, int64_t stride_page, int64_t stride_tok, int64_t stride_head,
                int32_t num_pages, int32_t page_size, int32_t head_dim, const int32_t* table, int64_t table_stride,
                int32_t pages_per_seq) {
  if (!k || !v || !table || !aligned16(k) || !aligned16(v) || !aligned4(table)) return BT_EINVAL;
  if (num_pages < 1 || pages_per_seq < 1 || table_stride < pages_per_seq) return BT_EINVAL;
  if (stride_page < head_dim || stride_tok < head_dim || stride_head < head_dim || stride_page % 8 || stride_tok % 8 || stride_head % 8)
    return BT_EINVAL;
  if (!bt::page_size_served(page_size)) return BT_ENOTSUP;
  if ((int64_t)pages_per_seq * page_size > INT32_MAX - bt::kMaxPageSize) return BT_ENOTSUP;
  if (stride_tok > (int64_t)(INT32_MAX / 2) / page_size) return BT_ENOTSUP;  // a page's rows of one head within 2 GiB
  return BT_OK;
}

bt::PagedLayout paged_layout(int64_t stride_page, int64_t stride_tok, int64_t stride_head, int32_t num_pages,
                             int32_t page_size, const int32_t* table, int64_t table_stride, int32_t pages_per_seq) {
  bt::PagedLayout l{};
  l.stride_page = stride_page;
  l.stride_tok = stride_tok;
  l.stride_head = stride_head;
  l.num_pages = num_pages;
  l.page_shift = log2_of(page_size);
  l.table = table;
  l.table_stride = table_stride;
  l.pages_per_seq = pages_per_seq;
  return l;
}

// Compute units of the current device.
int device_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  static std::atomic<int> cache[64];
  if (dev >= 0 && dev < 64 && (n = cache[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
  if (dev >= 0 && dev < 64) cache[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Decode workspace, each part 256-byte aligned: the parts' LSEs, the parts, and
// each sequence's first slot and count.
struct PagedWorkspace {
  int32_t runs;
  int64_t part, base, count, bytes;
};
PagedWorkspace paged_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t max_tokens) {
  PagedWorkspace w{};
  w.runs = bt::paged_runs(batch, kv_heads, head_dim, max_tokens, device_cus());
  if (w.runs == 0) return w;
  const int64_t slots = (int64_t)heads * (w.runs + batch);
  w.part = align256(slots * 4);
  w.base = w.part + align256(slots * head_dim * 4);
  w.count = w.base + align256((int64_t)batch * 4);
  w.bytes = w.count + align256((int64_t)batch * 4);
  return w;
}

}  // namespace

extern "C" {

int64_t bt_paged_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t max_tokens) {
  if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_tokens < 1) return 0;
  return paged_workspace(batch, heads, kv_heads, head_dim, max_tokens).bytes;
}

static int decode_params(bt::PagedDecodeParams& p, const void* q, int32_t q_dtype, int64_t q_stride_seq, const void* k,
                         const void* v, int64_t stride_page, int64_t stride_tok, int64_t stride_head, int32_t num_pages,
                         int32_t page_size, const int32_t* table, int64_t table_stride, int32_t pages_per_seq,
                         const int32_t* lens, int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, float scale,
                         void* workspace, int64_t workspace_bytes, void* out, int32_t out_dtype, int64_t out_stride_seq) {
  if (!q || !lens || !out || !aligned16(q) || !aligned16(out) || !aligned4(lens)) return BT_EINVAL;
  if (batch < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || heads % kv_heads) return BT_EINVAL;
  if (!dtype_known(q_dtype) || !dtype_known(out_dtype)) return BT_EINVAL;
  if (q_stride_seq < (int64_t)heads * head_dim || q_stride_seq % 8) return BT_EINVAL;
  if (out_stride_seq < (int64_t)heads * head_dim || out_stride_seq % 8) return BT_EINVAL;
  int rc = check_paged(k, v, stride_page, stride_tok, stride_head, num_pages, page_size, head_dim, table, table_stride,
                       pages_per_seq);
  if (rc) return rc;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return BT_ENOTSUP;
  if (heads / kv_heads > 8 || batch > bt::kPagedMaxBatch || kv_heads > 65535) return BT_ENOTSUP;
  if ((int64_t)batch * heads > INT32_MAX / 512) return BT_ENOTSUP;  // work-items of a launch
  const int64_t max_tokens = (int64_t)pages_per_seq * page_size;
  if (batch * (max_tokens / 16) > INT32_MAX / 2) return BT_ENOTSUP;  // tiles are numbered through the batch
  const PagedWorkspace ws = paged_workspace(batch, heads, kv_heads, head_dim, max_tokens);
  if (ws.bytes && (!workspace || !aligned16(workspace) || workspace_bytes < ws.bytes)) return BT_ENOSPC;
  p.q = q;
  p.q_stride_seq = q_stride_seq;
  p.q_bf16 = q_dtype == BT_DTYPE_BF16;
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.pg = paged_layout(stride_page, stride_tok, stride_head, num_pages, page_size, table, table_stride, pages_per_seq);
  p.lens = lens;
  p.batch = batch;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.scale_log2 = (float)((double)scale * kLog2e);
  p.runs = ws.runs;
  if (ws.bytes) {
    char* at = static_cast<char*>(workspace);
    p.lse = reinterpret_cast<float*>(at);
    p.part = reinterpret_cast<float*>(at + ws.part);
    p.part_base = reinterpret_cast<int32_t*>(at + ws.base);
    p.part_count = reinterpret_cast<int32_t*>(at + ws.count);
  }
  p.out = out;
  p.out_bf16 = out_dtype == BT_DTYPE_BF16;
  p.out_stride_seq = out_stride_seq;
  return BT_OK;
}

int bt_gqa_decode_paged(const void* q, int32_t q_dtype, int64_t q_stride_seq, const void* k, const void* v,
                        int64_t stride_page, int64_t stride_tok, int64_t stride_head, int32_t num_pages,
                        int32_t page_size, const int32_t* table, int64_t table_stride, int32_t pages_per_seq,
                        const int32_t* lens, int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim,
                        float scale, void* workspace, int64_t workspace_bytes, void* out, int32_t out_dtype,
                        int64_t out_stride_seq, void* stream) {
  bt::PagedDecodeParams p{};
  const int rc = decode_params(p, q, q_dtype, q_stride_seq, k, v, stride_page, stride_tok, stride_head, num_pages, page_size,
                               table, table_stride, pages_per_seq, lens, batch, heads, kv_heads, head_dim, scale, workspace,
                               workspace_bytes, out, out_dtype, out_stride_seq);
  return rc ? rc : hip_rc(bt::launch_decode_paged(p, head_dim, (hipStream_t)stream));
}

// Workspace of the drafts' attention, as PagedWorkspace.
static PagedWorkspace tree_workspace(int32_t batch, int32_t drafts, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                     int64_t max_tokens) {
  PagedWorkspace w{};
  w.runs = bt::tree_runs(batch, kv_heads, drafts * (heads / kv_heads), max_tokens, device_cus());
  if (w.runs == 0) return w;
  const int64_t slots = (int64_t)drafts * heads * (w.runs + batch);
  w.part = align256(slots * 4);
  w.base = w.part + align256(slots * head_dim * 4);
  w.count = w.base + align256((int64_t)batch * 4);
  w.bytes = w.count + align256((int64_t)batch * 4);
  return w;
}

int64_t bt_tree_workspace_bytes(int32_t batch, int32_t drafts, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                int32_t max_tokens) {
  if (batch < 1 || drafts < 1 || drafts > bt::kMaxDrafts || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_tokens < 1)
    return 0;
  return tree_workspace(batch, drafts, heads, kv_heads, head_dim, max_tokens).bytes;
}

int bt_gqa_decode_tree(const void* q, int32_t q_dtype, int64_t q_stride_seq, const void* k, const void* v,
                       int64_t stride_page, int64_t stride_tok, int64_t stride_head, int32_t num_pages,
                       int32_t page_size, const int32_t* table, int64_t table_stride, int32_t pages_per_seq,
                       const int32_t* lens, const int32_t* parents, int32_t batch, int32_t drafts, int32_t heads,
                       int32_t kv_heads, int32_t head_dim, float scale, void* workspace, int64_t workspace_bytes,
                       void* out, int32_t out_dtype, int64_t out_stride_seq, void* stream) {
  if (!q || !lens || !parents || !out || !aligned16(q) || !aligned16(out) || !aligned4(lens) || !aligned4(parents)) return BT_EINVAL;
  if (batch < 1 || drafts < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || heads % kv_heads) return BT_EINVAL;
  if (!dtype_known(q_dtype) || !dtype_known(out_dtype)) return BT_EINVAL;
  if (drafts > bt::kMaxDrafts) return BT_ENOTSUP;
  const int64_t row = (int64_t)drafts * heads * head_dim;
  if (q_stride_seq < row || q_stride_seq % 8 || out_stride_seq < row || out_stride_seq % 8) return BT_EINVAL;
  int rc = check_paged(k, v, stride_page, stride_tok, stride_head, num_pages, page_size, head_dim, table, table_stride,
                       pages_per_seq);
  if (rc) return rc;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return BT_ENOTSUP;
  if (heads / kv_heads > 8 || batch > bt::kPagedMaxBatch || kv_heads > 65535) return BT_ENOTSUP;
  if ((int64_t)batch * drafts * heads > INT32_MAX / 512) return BT_ENOTSUP;  // work-items of a launch
  const int64_t max_tokens = (int64_t)pages_per_seq * page_size;
  if (batch * (max_tokens / 16) > INT32_MAX / 2) return BT_ENOTSUP;  // tiles are numbered through the batch
  const PagedWorkspace ws = tree_workspace(batch, drafts, heads, kv_heads, head_dim, max_tokens);
  if (ws.bytes && (!workspace || !aligned16(workspace) || workspace_bytes < ws.bytes)) return BT_ENOSPC;
  bt::TreeParams p{};
  p.q = q;
  p.q_stride_seq = q_stride_seq;
  p.q_bf16 = q_dtype == BT_DTYPE_BF16;
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.pg = paged_layout(stride_page, stride_tok, stride_head, num_pages, page_size, table, table_stride, pages_per_seq);
  p.lens = lens;
  p.parents = parents;
  p.batch = batch;
  p.drafts = drafts;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.row_blocks = bt::tree_row_blocks(drafts * p.group);
  p.scale_log2 = (float)((double)scale * kLog2e);
  p.places = bt::tree_places(kv_heads, drafts * p.group, device_cus());
  p.runs = ws.runs;
  if (ws.bytes) {
    char* at = static_cast<char*>(workspace);
    p.lse = reinterpret_cast<float*>(at);
    p.part = reinterpret_cast<float*>(at + ws.part);
    p.part_base = reinterpret_cast<int32_t*>(at + ws.base);
    p.part_count = reinterpret_cast<int32_t*>(at + ws.count);
  }
  p.out = out;
  p.out_bf16 = out_dtype == BT_DTYPE_BF16;
  p.out_stride_seq = out_stride_seq;
  return hip_rc(bt::launch_decode_tree(p, head_dim, (hipStream_t)stream));
}

int bt_accept_drafts(void* pages, int64_t plane_stride, int64_t page_stride, int32_t planes, int32_t num_pages,
                     int32_t page_size, int32_t token_elems, const int32_t* table, const int32_t* lens, int32_t rows,
                     int32_t pages_per_seq, const int32_t* parents, const int32_t* tokens, const int32_t* first,
                     const int32_t* best, int32_t drafts, int32_t* lens_out, int32_t* path_out, int32_t* following_out,
                     void* stream) {
  if (!pages || !aligned16(pages) || planes < 1 || num_pages < 1 || token_elems < 8 || token_elems % 8) return BT_EINVAL;
  if (!table || !lens || !parents || !tokens || !first || !best || !lens_out || !path_out || !following_out) return BT_EINVAL;
  for (const int32_t* x : {table, lens, parents, tokens, first, best, (const int32_t*)lens_out, (const int32_t*)path_out, (const int32_t*)following_out})
    if (!aligned4(x)) return BT_EINVAL;
  if (rows < 1 || pages_per_seq < 1 || drafts < 1 || lens_out == lens || following_out == first) return BT_EINVAL;
  if (path_out == parents || path_out == tokens || path_out == best) return BT_EINVAL;
  if (!bt::page_size_served(page_size) || drafts > bt::kMaxDrafts) return BT_ENOTSUP;
  if (token_elems > INT32_MAX / page_size) return BT_ENOTSUP;
  const int64_t page = (int64_t)page_size * token_elems;
  if (page_stride % 8 || plane_stride % 8 || page_stride < page || plane_stride < page) return BT_EINVAL;
  if (planes > 1 && plane_stride / num_pages < page_stride && page_stride / planes < plane_stride) return BT_EINVAL;
  if ((int64_t)pages_per_seq * page_size > INT32_MAX - bt::kMaxPageSize) return BT_ENOTSUP;
  const int64_t groups = ((int64_t)planes * (token_elems / 8) + 255) / 256;
  if (groups > 65535 || rows > INT32_MAX / 256) return BT_ENOTSUP;
  bt::AcceptParams p{};
  p.pages = static_cast<uint16_t*>(pages);
  p.plane_stride = plane_stride;
  p.page_stride = page_stride;
  p.planes = planes;
  p.num_pages = num_pages;
  p.page_shift = log2_of(page_size);
  p.token_elems = token_elems;
  p.table = table;
  p.lens = lens;
  p.rows = rows;
  p.pages_per_seq = pages_per_seq;
  p.drafts = drafts;
  p.parents = parents;
  p.tokens = tokens;
  p.first = first;
  p.best = best;
  p.lens_out = lens_out;
  p.path_out = path_out;
  p.following_out = following_out;
  return hip_rc(bt::launch_accept_drafts(p, (hipStream_t)stream));
}

int bt_key_bounds(const void* k, int64_t stride_page, int64_t stride_tok, int64_t stride_head, int32_t num_pages,
                  int32_t page_size, const int32_t* table, int64_t table_stride, int32_t pages_per_seq,
                  const int32_t* lens, const int32_t* first, int32_t batch, int32_t kv_heads, int32_t head_dim,
                  void* bounds, void* stream) {
  if (!lens || !bounds || !aligned16(bounds) || !aligned4(lens) || !aligned4(first)) return BT_EINVAL;
  if (batch < 1 || kv_heads < 1 || head_dim < 1) return BT_EINVAL;
  const int rc = check_paged(k, k, stride_page, stride_tok, stride_head, num_pages, page_size, head_dim, table, table_stride,
                             pages_per_seq);
  if (rc) return rc;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return BT_ENOTSUP;
  if (batch > bt::kPagedMaxBatch || kv_heads > 65535) return BT_ENOTSUP;
  if ((int64_t)batch * pages_per_seq > INT32_MAX) return BT_ENOTSUP;  // pages are numbered through the batch
  bt::BoundsParams p{};
  p.k = static_cast<const uint16_t*>(k);
  p.pg = paged_layout(stride_page, stride_tok, stride_head, num_pages, page_size, table, table_stride, pages_per_seq);
  p.lens = lens;
  p.first = first;
  p.batch = batch;
  p.kv_heads = kv_heads;
  p.head_dim = head_dim;
  p.bounds = static_cast<uint16_t*>(bounds);
  return hip_rc(bt::launch_key_bounds(p, (hipStream_t)stream));
}

int64_t bt_select_workspace_bytes(int32_t batch, int32_t kv_heads, int32_t pages_per_seq, int32_t count) {
  if (batch < 1 || kv_heads < 1 || pages_per_seq < 1 || !bt::needs_scores(pages_per_seq, count)) return 0;
  return align256((int64_t)batch * kv_heads * pages_per_seq * 8);
}

static int select_params(bt::SelectParams& p, const void* q, int32_t q_dtype, int64_t q_stride_seq, const void* bounds,
                         int32_t num_pages, int32_t page_size, const int32_t* table, int64_t table_stride,
                         int32_t pages_per_seq, const int32_t* lens, int32_t batch, int32_t heads, int32_t kv_heads,
                         int32_t head_dim, int32_t count) {
  if (!q || !bounds || !table || !lens) return BT_EINVAL;
  if (!aligned16(q) || !aligned16(bounds) || !aligned4(table) || !aligned4(lens)) return BT_EINVAL;
  if (batch < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || heads % kv_heads || !dtype_known(q_dtype)) return BT_EINVAL;
  if (q_stride_seq < (int64_t)heads * head_dim || q_stride_seq % 8) return BT_EINVAL;
  if (num_pages < 1 || pages_per_seq < 1 || table_stride < pages_per_seq || count < 1) return BT_EINVAL;
  if (!bt::page_size_served(page_size)) return BT_ENOTSUP;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return BT_ENOTSUP;
  if (heads / kv_heads > 8 || batch > bt::kPagedMaxBatch || kv_heads > 65535) return BT_ENOTSUP;
  if ((int64_t)pages_per_seq * page_size > INT32_MAX - bt::kMaxPageSize || (int64_t)count * page_size > INT32_MAX - bt::kMaxPageSize)
    return BT_ENOTSUP;
  // Work-items of a launch: of the choice, and of the scores.
  if ((int64_t)batch * kv_heads > INT32_MAX / 1024 || (int64_t)batch * kv_heads * ((pages_per_seq + 127) / 128) > INT32_MAX / 256)
    return BT_ENOTSUP;
  p.q = q;
  p.q_stride_seq = q_stride_seq;
  p.q_bf16 = q_dtype == BT_DTYPE_BF16;
  p.bounds = static_cast<const uint16_t*>(bounds);
  p.pg = paged_layout(0, 0, 0, num_pages, page_size, table, table_stride, pages_per_seq);
  p.lens = lens;
  p.batch = batch;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.head_dim = head_dim;
  p.count = count;
  return BT_OK;
}

int bt_select_pages(const void* q, int32_t q_dtype, int64_t q_stride_seq, const void* bounds, int32_t num_pages,
                    int32_t page_size, const int32_t* table, int64_t table_stride, int32_t pages_per_seq,
                    const int32_t* lens, int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim,
                    int32_t count, int32_t* chosen, int32_t* chosen_lens, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  if (!chosen || !chosen_lens || chosen_lens == lens || chosen == table || !aligned4(chosen) || !aligned4(chosen_lens)) return BT_EINVAL;
  bt::SelectParams p{};
  const int rc = select_params(p, q, q_dtype, q_stride_seq, bounds, num_pages, page_size, table, table_stride, pages_per_seq,
                               lens, batch, heads, kv_heads, head_dim, count);
  if (rc) return rc;
  const int64_t bytes = bt_select_workspace_bytes(batch, kv_heads, pages_per_seq, count);
  if (bytes && (!workspace || !aligned16(workspace) || workspace_bytes < bytes)) return BT_ENOSPC;
  p.score = bytes ? static_cast<double*>(workspace) : nullptr;
  p.chosen = chosen;
  p.chosen_len = chosen_lens;
  return hip_rc(bt::launch_select_pages(p, (hipStream_t)stream));
}

// Workspace of the sparse attention, each part 256-byte aligned: the scores, the choice, its lengths, and what
// the attention over it needs.
struct SparseWorkspace {
  int64_t chosen, lens, attention, bytes;
};
static SparseWorkspace sparse_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t pages_per_seq,
                                        int32_t page_size, int32_t count) {
  SparseWorkspace w{};
  w.chosen = bt_select_workspace_bytes(batch, kv_heads, pages_per_seq, count);
  w.lens = w.chosen + align256((int64_t)batch * kv_heads * count * 4);
  w.attention = w.lens + align256((int64_t)batch * 4);
  w.bytes = w.attention + paged_workspace(batch, heads, kv_heads, head_dim, (int64_t)count * page_size).bytes;
  return w;
}

int64_t bt_sparse_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t pages_per_seq,
                                  int32_t page_size, int32_t count) {
  if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || pages_per_seq < 1 || page_size < 1 || count < 1) return 0;
  return sparse_workspace(batch, heads, kv_heads, head_dim, pages_per_seq, page_size, count).bytes;
}

int bt_gqa_decode_sparse(const void* q, int32_t q_dtype, int64_t q_stride_seq, const void* k, const void* v,
                         int64_t stride_page, int64_t stride_tok, int64_t stride_head, int32_t num_pages,
                         int32_t page_size, const void* bounds, const int32_t* table, int64_t table_stride,
                         int32_t pages_per_seq, const int32_t* lens, int32_t batch, int32_t heads, int32_t kv_heads,
                         int32_t head_dim, int32_t count, float scale, void* workspace, int64_t workspace_bytes,
                         void* out, int32_t out_dtype, int64_t out_stride_seq, void* stream) {
  if (!(scale > 0.f)) return BT_EINVAL;  // the pages are chosen for one
  bt::SelectParams p{};
  int rc = select_params(p, q, q_dtype, q_stride_seq, bounds, num_pages, page_size, table, table_stride, pages_per_seq, lens,
                         batch, heads, kv_heads, head_dim, count);
  if (rc) return rc;
  const SparseWorkspace ws = sparse_workspace(batch, heads, kv_heads, head_dim, pages_per_seq, page_size, count);
  if (!workspace || !aligned16(workspace) || workspace_bytes < ws.bytes) return BT_ENOSPC;
  char* at = static_cast<char*>(workspace);
  p.score = ws.chosen ? reinterpret_cast<double*>(at) : nullptr;
  p.chosen = reinterpret_cast<int32_t*>(at + ws.chosen);
  p.chosen_len = reinterpret_cast<int32_t*>(at + ws.lens);
  bt::PagedDecodeParams d{};
  rc = decode_params(d, q, q_dtype, q_stride_seq, k, v, stride_page, stride_tok, stride_head, num_pages, page_size, p.chosen,
                     (int64_t)kv_heads * count, count, p.chosen_len, batch, heads, kv_heads, head_dim, scale, at + ws.attention,
                     workspace_bytes - ws.attention, out, out_dtype, out_stride_seq);
  if (rc) return rc;
  d.table_stride_head = count;
  rc = hip_rc(bt::launch_select_pages(p, (hipStream_t)stream));
  return rc ? rc : hip_rc(bt::launch_decode_paged(d, head_dim, (hipStream_t)stream));
}

int bt_attn_prep_drafts(const void* qkv, int32_t qkv_dtype, int64_t qkv_stride, int32_t tokens, int32_t heads,
                        int32_t kv_heads, int32_t head_dim, int32_t gated, const float* q_norm, const float* k_norm,
                        float eps, const float* cos, const float* sin, int32_t rope_dim, int32_t rope_cap,
                        int32_t interleaved, const int32_t* pos, const int32_t* angles, const int32_t* rows, void* q_out,
                        int32_t q_dtype, void* k, void* v, int64_t stride_page, int64_t stride_tok, int64_t stride_head,
                        int32_t num_pages, int32_t page_size, const int32_t* table, int64_t table_stride,
                        int32_t table_rows, int32_t pages_per_seq, void* stream) {
  if (!qkv || !pos || !q_out || !aligned16(qkv) || !aligned16(q_out) || !aligned4(angles)) return BT_EINVAL;
  if (tokens < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || table_rows < 1) return BT_EINVAL;
  if (!dtype_known(qkv_dtype) || !dtype_known(q_dtype)) return BT_EINVAL;
  const int64_t row = (int64_t)heads * head_dim * (gated ? 2 : 1) + 2 * (int64_t)kv_heads * head_dim;
  if (qkv_stride < row || qkv_stride % 8) return BT_EINVAL;
  if ((q_norm == nullptr) != (k_norm == nullptr) || (cos == nullptr) != (sin == nullptr)) return BT_EINVAL;
  if (q_norm && (!aligned16(q_norm) || !aligned16(k_norm))) return BT_EINVAL;
  if (cos && (rope_dim < 2 || rope_dim % 2 || rope_dim > head_dim || rope_cap < 1)) return BT_EINVAL;
  if (!(eps >= 0.f)) return BT_EINVAL;
  int rc = check_paged(k, v, stride_page, stride_tok, stride_head, num_pages, page_size, head_dim, table, table_stride,
                       pages_per_seq);
  if (rc) return rc;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512) return BT_ENOTSUP;
  if ((int64_t)tokens * (heads + 2 * (int64_t)kv_heads) > INT32_MAX / 64) return BT_ENOTSUP;
  if (row > INT32_MAX) return BT_ENOTSUP;  // a token's values are numbered in 32 bits
  bt::PagedPrepParams p{};
  p.x = qkv;
  p.x_bf16 = qkv_dtype == BT_DTYPE_BF16;
  p.x_stride = qkv_stride;
  p.tokens = tokens;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.gated = gated ? 1 : 0;
  p.wq = q_norm;
  p.wk = k_norm;
  p.eps = eps;
  p.cos = cos;
  p.sin = sin;
  p.rope_dim = cos ? rope_dim : 0;
  p.rope_cap = rope_cap;
  p.interleaved = interleaved ? 1 : 0;
  p.pos = pos;
  p.angle = angles;
  p.rows = rows;
  p.table_rows = table_rows;
  p.q_out = q_out;
  p.q_out_bf16 = q_dtype == BT_DTYPE_BF16;
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  p.pg = paged_layout(stride_page, stride_tok, stride_head, num_pages, page_size, table, table_stride, pages_per_seq);
  return hip_rc(bt::launch_paged_prep(p, head_dim, (hipStream_t)stream));
}

int bt_attn_prep_paged(const void* qkv, int32_t qkv_dtype, int64_t qkv_stride, int32_t tokens, int32_t heads,
                       int32_t kv_heads, int32_t head_dim, int32_t gated, const float* q_norm, const float* k_norm,
                       float eps, const float* cos, const float* sin, int32_t rope_dim, int32_t rope_cap,
                       int32_t interleaved, const int32_t* pos, const int32_t* rows, void* q_out, int32_t q_dtype,
                       void* k, void* v, int64_t stride_page, int64_t stride_tok, int64_t stride_head,
                       int32_t num_pages, int32_t page_size, const int32_t* table, int64_t table_stride,
                       int32_t table_rows, int32_t pages_per_seq, void* stream) {
  return bt_attn_prep_drafts(qkv, qkv_dtype, qkv_stride, tokens, heads, kv_heads, head_dim, gated, q_norm, k_norm, eps, cos,
                             sin, rope_dim, rope_cap, interleaved, pos, nullptr, rows, q_out, q_dtype, k, v, stride_page,
                             stride_tok, stride_head, num_pages, page_size, table, table_stride, table_rows, pages_per_seq,
                             stream);
}

int64_t bt_pages_workspace_bytes(int32_t num_pages, int32_t rows) {
  if (num_pages < 1 || rows < 0) return 0;
  return 4 * bt::page_ws_ints(num_pages, rows);
}

static int page_params(bt::PageOpParams& p, void* pages, int64_t plane_stride, int64_t page_stride, int32_t planes,
                       int32_t num_pages, int32_t page_size, int32_t token_elems, const int32_t* table,
                       const int32_t* lens, int32_t rows, int32_t pages_per_seq, int32_t rows_out, const int32_t* keep,
                       int32_t num_keep, int32_t* table_out, void* workspace, int64_t workspace_bytes) {
  if (!pages || !aligned16(pages) || planes < 1 || num_pages < 1 || token_elems < 8 || token_elems % 8) return BT_EINVAL;
  if (!bt::page_size_served(page_size)) return BT_ENOTSUP;
  if (token_elems > INT32_MAX / page_size) return BT_ENOTSUP;
  const int64_t page = (int64_t)page_size * token_elems;
  if (page_stride % 8 || plane_stride % 8 || page_stride < page || plane_stride < page) return BT_EINVAL;
  // Planes and pages lie apart: planes of pages, or pages of planes.
  if (planes > 1 && plane_stride / num_pages < page_stride && page_stride / planes < plane_stride) return BT_EINVAL;
  if (rows < 0 || rows_out < 0 || pages_per_seq < 1 || num_keep < 0 || (num_keep && !keep)) return BT_EINVAL;
  if ((rows && (!table || !lens)) || (rows_out && !table_out) || (table_out && table_out == table)) return BT_EINVAL;
  if ((int64_t)pages_per_seq * page_size > INT32_MAX - bt::kMaxPageSize) return BT_ENOTSUP;
  // Work-items of a launch: 1,024 work-groups of 256 a plane, and one per entry.
  if ((int64_t)planes * (1024 * 256) + (int64_t)rows_out * pages_per_seq + num_keep > INT32_MAX) return BT_ENOTSUP;
  if ((int64_t)rows * pages_per_seq > INT32_MAX) return BT_ENOTSUP;
  if (!workspace || !aligned16(workspace) || workspace_bytes < bt_pages_workspace_bytes(num_pages, rows_out))
    return BT_ENOSPC;
  p.pages = static_cast<uint16_t*>(pages);
  p.plane_stride = plane_stride;
  p.page_stride = page_stride;
  p.planes = planes;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.page_shift = log2_of(page_size);
  p.token_elems = token_elems;
  p.table = table;
  p.lens = lens;
  p.rows = rows;
  p.pages_per_seq = pages_per_seq;
  p.rows_out = rows_out;
  p.keep = keep;
  p.num_keep = num_keep;
  p.table_out = table_out;
  p.ws = static_cast<int32_t*>(workspace);
  return BT_OK;
}

int bt_fork_pages(void* pages, int64_t plane_stride, int64_t page_stride, int32_t planes, int32_t num_pages,
                  int32_t page_size, int32_t token_elems, const int32_t* table, const int32_t* lens, int32_t rows,
                  int32_t pages_per_seq, const int32_t* parent, const int32_t* add, int32_t rows_out,
                  const int32_t* keep, int32_t num_keep, int32_t* table_out, int32_t* lens_out, int32_t* status,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (!status || (rows_out && !lens_out) || (lens_out && lens_out == lens) || (!parent && rows_out && rows_out != rows)) return BT_EINVAL;
  bt::PageOpParams p{};
  const int rc = page_params(p, pages, plane_stride, page_stride, planes, num_pages, page_size, token_elems, table, lens,
                             rows, pages_per_seq, rows_out, keep, num_keep, table_out, workspace, workspace_bytes);
  if (rc) return rc;
  p.parent = parent;
  p.add = add;
  p.lens_out = lens_out;
  p.status = status;
  return hip_rc(bt::launch_fork_pages(p, (hipStream_t)stream));
}

int bt_compact_pages(void* pages, int64_t plane_stride, int64_t page_stride, int32_t planes, int32_t num_pages,
                     int32_t page_size, int32_t token_elems, const int32_t* table, const int32_t* lens, int32_t rows,
                     int32_t pages_per_seq, const int32_t* keep, int32_t num_keep, int32_t* table_out, int32_t* where,
                     int32_t* live, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!where || !live) return BT_EINVAL;
  bt::PageOpParams p{};
  const int rc = page_params(p, pages, plane_stride, page_stride, planes, num_pages, page_size, token_elems, table, lens,
                             rows, pages_per_seq, rows, keep, num_keep, table_out, workspace, workspace_bytes);
  if (rc) return rc;
  p.where = where;
  p.status = live;
  return hip_rc(bt::launch_compact_pages(p, (hipStream_t)stream));
}

int64_t bt_beam_workspace_bytes(int32_t batch, int32_t width, int32_t vocab, int32_t beams) {
  if (batch < 1 || width < 1 || vocab < 1 || beams < 1) return 0;
  return bt::beam_ws_bytes(batch, width, vocab, beams);
}

int bt_beam_select(const void* logits, int32_t dtype, int64_t stride_batch, int64_t stride_beam, const float* scores,
                   int32_t batch, int32_t width, int32_t vocab, int32_t beams, float* scores_out, int32_t* parent_out,
                   int32_t* token_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!logits || !scores || !scores_out || !parent_out || !token_out) return BT_EINVAL;
  if (batch < 1 || width < 1 || vocab < 1 || beams < 1 || !dtype_known(dtype)) return BT_EINVAL;
  if (stride_batch < 0 || stride_beam < 0 || (int64_t)beams > (int64_t)width * vocab) return BT_EINVAL;
  if (vocab > (1 << 30) || width > bt::kMaxBeamWidth || beams > bt::kMaxBeams || (int64_t)batch * width > INT32_MAX / 1024) return BT_ENOTSUP;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == BT_DTYPE_BF16 ? 2 : 4)) return BT_EINVAL;
  if (!workspace || !aligned16(workspace) || workspace_bytes < bt_beam_workspace_bytes(batch, width, vocab, beams))
    return BT_ENOSPC;
  bt::BeamParams p{};
  p.logits = logits;
  p.bf16 = dtype == BT_DTYPE_BF16;
  p.stride_batch = stride_batch;
  p.stride_beam = stride_beam;
  p.scores = scores;
  p.batch = batch;
  p.width = width;
  p.vocab = vocab;
  p.beams = beams;
  p.ws = workspace;
  p.scores_out = scores_out;
  p.parent_out = parent_out;
  p.token_out = token_out;
  return hip_rc(bt::launch_beam_select(p, (hipStream_t)stream));
}

}  // extern "C"
