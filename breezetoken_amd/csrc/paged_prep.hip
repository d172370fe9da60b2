// Preparation of an attention layer over a paged cache, any number of tokens in
// one launch (gfx950): per token, from the fused projection output
// [H x q (| gate) | Hkv x k | Hkv x v],
//
//   n(x) = x * rsqrt(mean(x^2) + eps) * w                            (optional)
//   rotary position, c_i / s_i = columns i < rope_dim / 2 of row pos of the
//   tables (rows clamped to the table):
//     half layout:        (n_i, n_{i+h}) -> (n_i c_i - n_{i+h} s_i, n_{i+h} c_i + n_i s_i), h = rope_dim / 2
//     interleaved layout: the same on (n_{2i}, n_{2i+1})
//   q -> q_out, k and v -> bf16 at the token's slot of the pages.
//
// Tokens without a slot (position or row outside the table, page id outside the
// cache) write no key and no value.
#include "bt_common.h"
#include "bt_kernels.h"

namespace bt {

namespace {

// One wave per (token, row): rows 0 .. H - 1 are q heads, then k heads, then v heads.
template <int D>
__global__ __launch_bounds__(64) void paged_prep_kernel(PagedPrepParams p) {
  constexpr int E = D / 64;
  __shared__ float row[D];
  const int rows = p.heads + 2 * p.kv_heads;
  const int t = (int)(blockIdx.x / (unsigned)rows), r = (int)(blockIdx.x % (unsigned)rows);
  const int lane = threadIdx.x;
  const bool is_q = r < p.heads, is_v = r >= p.heads + p.kv_heads;
  const int step = p.gated ? 2 * D : D;
  const int64_t src = (int64_t)t * p.x_stride + (is_q ? (int64_t)r * step : (int64_t)p.heads * step + (int64_t)(r - p.heads) * D);
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int64_t at = src + lane * E + e;
    x[e] = p.x_bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p.x)[at]) : reinterpret_cast<const float*>(p.x)[at];
  }
  const int pos = p.pos[t];
  const float* w = is_q ? p.wq : p.wk;
  if (!is_v && w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(x[e], x[e], ss);
    ss = wave_sum(ss);
    const float f = 1.0f / sqrtf(ss / (float)D + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * f * w[lane * E + e];
  }
  if (!is_v && p.cos != nullptr) {
#pragma unroll
    for (int e = 0; e < E; ++e) row[lane * E + e] = x[e];
    __syncthreads();
    const int pr = pos < 0 ? 0 : (pos >= p.rope_cap ? p.rope_cap - 1 : pos);
    const float* c = p.cos + (int64_t)pr * p.rope_dim;
    const float* s = p.sin + (int64_t)pr * p.rope_dim;
    const int half = p.rope_dim / 2;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane * E + e;
      if (d < p.rope_dim) {
        const bool first = p.interleaved ? (d & 1) == 0 : d < half;
        const int i = p.interleaved ? d >> 1 : (first ? d : d - half);
        const float other = row[p.interleaved ? d ^ 1 : (first ? d + half : d - half)];
        x[e] = first ? x[e] * c[i] - other * s[i] : x[e] * c[i] + other * s[i];
      }
    }
  }
  if (is_q) {
    const int64_t at = ((int64_t)t * p.heads + r) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (p.q_out_bf16) reinterpret_cast<uint16_t*>(p.q_out)[at + e] = (uint16_t)f32_to_bf16_bits(x[e]);
      else reinterpret_cast<float*>(p.q_out)[at + e] = x[e];
    }
    return;
  }
  const int seq = p.rows ? p.rows[t] : t;
  if (seq < 0 || seq >= p.table_rows || pos < 0 || (pos >> p.pg.page_shift) >= p.pg.pages_per_seq) return;
  const int page = p.pg.table[(int64_t)seq * p.pg.table_stride + (pos >> p.pg.page_shift)];
  if (page < 0 || page >= p.pg.num_pages) return;
  const int g = is_v ? r - p.heads - p.kv_heads : r - p.heads;
  const int64_t at = (int64_t)page * p.pg.stride_page + (int64_t)(pos & ((1 << p.pg.page_shift) - 1)) * p.pg.stride_tok +
                     (int64_t)g * p.pg.stride_head + lane * E;
  uint16_t* dst = is_v ? p.v : p.k;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[at + e] = (uint16_t)f32_to_bf16_bits(x[e]);
}

}  // namespace

hipError_t launch_paged_prep(const PagedPrepParams& p, int head_dim, hipStream_t stream) {
  const dim3 grid((unsigned)p.tokens * (unsigned)(p.heads + 2 * p.kv_heads));
  switch (head_dim) {
    case 64: hipLaunchKernelGGL(paged_prep_kernel<64>, grid, dim3(64), 0, stream, p); break;
    case 128: hipLaunchKernelGGL(paged_prep_kernel<128>, grid, dim3(64), 0, stream, p); break;
    case 256: hipLaunchKernelGGL(paged_prep_kernel<256>, grid, dim3(64), 0, stream, p); break;
    case 512: hipLaunchKernelGGL(paged_prep_kernel<512>, grid, dim3(64), 0, stream, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace bt
