// Decode attention over a paged bf16 KV cache for gfx950: one new token per
// sequence, keys 0 .. lens[b] - 1 found through the page table.
//
//   x_j = q . k_j * scale * log2e,  m = max_j x_j,  l = sum_j exp2(x_j - m)
//   out = sum_j exp2(x_j - m) v_j / l,  zeros for a sequence without keys
//
// A table entry outside [0, num_pages) holds no keys.
#include "bt_common.h"
#include "bt_kernels.h"

namespace bt {

namespace {

// One work-group of four waves per (sequence, query head); wave w takes the
// tokens w, w + 4, ...; lane l holds the dims l, l + 64, ...
template <int D, bool QBF16>
__global__ __launch_bounds__(256) void gqa_paged_kernel(PagedDecodeParams p) {
  constexpr int E = D / 64;
  const int h = (int)blockIdx.x % p.heads, b = (int)blockIdx.x / p.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kvh = h / p.group;
  const int64_t cap = (int64_t)p.pg.pages_per_seq << p.pg.page_shift;
  int64_t valid = p.lens[b];
  if (valid > cap) valid = cap;
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int64_t at = (int64_t)b * p.q_stride_seq + (int64_t)h * D + e * 64 + lane;
    q[e] = QBF16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p.q)[at]) : reinterpret_cast<const float*>(p.q)[at];
    q[e] *= p.scale_log2;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = wave; j < valid; j += 4) {
    const int page = p.pg.table[(int64_t)b * p.pg.table_stride + (j >> p.pg.page_shift)];
    if (page < 0 || page >= p.pg.num_pages) continue;
    const int64_t row = (int64_t)page * p.pg.stride_page + (j & ((1 << p.pg.page_shift) - 1)) * p.pg.stride_tok +
                        (int64_t)kvh * p.pg.stride_head;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x = fmaf(q[e], bf16_bits_to_f32(p.k[row + e * 64 + lane]), x);
    x = wave_sum(x);
    const float mn = fmax_nc(m, x);  // a NaN score makes the row NaN
    const float a = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(x - mn);
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(w, bf16_bits_to_f32(p.v[row + e * 64 + lane]), o[e] * a);
  }
  __shared__ float ms[4], ls[4], os[4][D];
  if (lane == 0) {
    ms[wave] = m;
    ls[wave] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) os[wave][e * 64 + lane] = o[e];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < 4; ++w) top = fmax_nc(top, ms[w]);
  for (int w = 0; w < 4; ++w) sum += ms[w] == -INFINITY ? 0.f : ls[w] * exp2f(ms[w] - top);
  for (int d = threadIdx.x; d < D; d += 256) {
    float y = 0.f;
    for (int w = 0; w < 4; ++w) y += ms[w] == -INFINITY ? 0.f : os[w][d] * exp2f(ms[w] - top);
    y = sum == 0.f ? 0.f : y / sum;
    const int64_t at = (int64_t)b * p.out_stride_seq + (int64_t)h * D + d;
    if (p.out_bf16) reinterpret_cast<uint16_t*>(p.out)[at] = (uint16_t)f32_to_bf16_bits(y);
    else reinterpret_cast<float*>(p.out)[at] = y;
  }
}

template <int D>
hipError_t launch_dim(const PagedDecodeParams& p, hipStream_t stream) {
  const dim3 grid(p.batch * p.heads);
  if (p.q_bf16) hipLaunchKernelGGL((gqa_paged_kernel<D, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((gqa_paged_kernel<D, false>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_decode_paged(const PagedDecodeParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_dim<64>(p, stream);
    case 128: return launch_dim<128>(p, stream);
    case 256: return launch_dim<256>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bt
