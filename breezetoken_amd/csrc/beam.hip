// Beam search's selection for gfx950: of the batch's width x vocab candidates
//   score[b, w] + logit[b, w, v] - log sum_u exp(logit[b, w, u])
// the best `beams` of each batch item, with the beam they continue and their token.
//
// Candidates are ordered by their value in 64 bits, equal ones by their place
// w * vocab + v.  A NaN logit counts as -inf, a beam without a finite logit has
// only candidates of -inf.  A logit of +inf makes its beam's others -inf and its
// own candidate score[b, w] less the log of the number of them.
#include "bt_common.h"
#include "bt_kernels.h"

namespace bt {

namespace {

constexpr int kBeamThreads = 256;

// Order-preserving bits of a float (-0 as +0); NaN is taken as -inf by the caller.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* x, int64_t i) {
  const float f = BF16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(x)[i]) : reinterpret_cast<const float*>(x)[i];
  return f != f ? -INFINITY : f;
}

__device__ uint64_t block_max(uint64_t v, uint64_t* lds) {
  __syncthreads();
  lds[threadIdx.x] = v;
  __syncthreads();
  for (int o = kBeamThreads / 2; o; o >>= 1) {
    if ((int)threadIdx.x < o && lds[threadIdx.x + o] > lds[threadIdx.x]) lds[threadIdx.x] = lds[threadIdx.x + o];
    __syncthreads();
  }
  return lds[0];
}
__device__ double block_sum(double v, double* lds) {
  __syncthreads();
  lds[threadIdx.x] = v;
  __syncthreads();
  for (int o = kBeamThreads / 2; o; o >>= 1) {
    if ((int)threadIdx.x < o) lds[threadIdx.x] += lds[threadIdx.x + o];
    __syncthreads();
  }
  return lds[0];
}

// Per (batch item, beam): the best `beams` tokens as (logit order, ~token), and the
// amount to add to a logit.
template <bool BF16>
__global__ __launch_bounds__(kBeamThreads) void beam_rows_kernel(BeamParams p) {
  __shared__ uint64_t lds[kBeamThreads];
  const int row = blockIdx.x, b = row / p.width, w = row % p.width;
  const int64_t base = b * p.stride_batch + w * p.stride_beam;
  uint64_t* best = reinterpret_cast<uint64_t*>(p.ws) + (int64_t)row * (p.beams + 2);
  uint64_t last = ~0ull, top = 0;
  for (int k = 0; k < p.beams; ++k) {
    uint64_t mine = 0;  // below every key: no candidate left
    for (int v = threadIdx.x; v < p.vocab; v += kBeamThreads) {
      const uint64_t key = (uint64_t)order_bits(load_logit<BF16>(p.logits, base + v)) << 32 | (uint32_t)~v;
      if (key < last && key > mine) mine = key;
    }
    last = block_max(mine, lds);
    if (k == 0) top = last;
    if (threadIdx.x == 0) best[k] = last;
    __syncthreads();
  }
  const float m = from_order((uint32_t)(top >> 32));
  double sum = 0;
  for (int v = threadIdx.x; v < p.vocab; v += kBeamThreads) {
    const float x = load_logit<BF16>(p.logits, base + v);
    sum += x == m ? 1.0 : exp((double)x - (double)m);
  }
  sum = block_sum(sum, reinterpret_cast<double*>(lds));
  if (threadIdx.x == 0) {
    reinterpret_cast<double*>(best)[p.beams] = (double)m;
    reinterpret_cast<double*>(best)[p.beams + 1] = (double)p.scores[row] - log(sum);
  }
}

// A candidate's value: the logit relative to the beam's largest, first.
__device__ __forceinline__ double candidate(uint64_t key, double m, double add) {
  const float x = from_order((uint32_t)(key >> 32));
  const double v = (double)x == m && x != -INFINITY ? add : (double)x - m + add;
  return v != v ? -(double)INFINITY : v;
}

__global__ __launch_bounds__(64) void beam_join_kernel(BeamParams p) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const bool mine = lane < p.width;
  const uint64_t* best = reinterpret_cast<const uint64_t*>(p.ws) + ((int64_t)b * p.width + (mine ? lane : 0)) * (p.beams + 2);
  const double m = reinterpret_cast<const double*>(best)[p.beams], add = reinterpret_cast<const double*>(best)[p.beams + 1];
  int at = 0;
  for (int k = 0; k < p.beams; ++k) {
    const uint64_t key = mine && at < p.beams ? best[at] : 0;
    double v = key ? candidate(key, m, add) : -(double)INFINITY;
    int from = key ? lane : 64;  // without a candidate behind every beam
    for (int o = 32; o; o >>= 1) {
      const double ov = __shfl_xor(v, o);
      const int of = __shfl_xor(from, o);
      if (of < 64 && (from == 64 || ov > v || (ov == v && of < from))) {
        v = ov;
        from = of;
      }
    }
    if (lane == from) {
      const int64_t out = (int64_t)b * p.beams + k;
      p.scores_out[out] = (float)v;
      p.parent_out[out] = b * p.width + lane;
      p.token_out[out] = (int)~(uint32_t)key;
      ++at;
    }
  }
}

}  // namespace

int64_t beam_ws_bytes(int batch, int width, int vocab, int beams) { return (int64_t)batch * width * (beams + 2) * 8; }

hipError_t launch_beam_select(const BeamParams& p, hipStream_t stream) {
  const dim3 rows(p.batch * p.width);
  if (p.bf16) hipLaunchKernelGGL(beam_rows_kernel<true>, rows, dim3(kBeamThreads), 0, stream, p);
  else hipLaunchKernelGGL(beam_rows_kernel<false>, rows, dim3(kBeamThreads), 0, stream, p);
  hipLaunchKernelGGL(beam_join_kernel, dim3(p.batch), dim3(64), 0, stream, p);
  return hipGetLastError();
}

}  // namespace bt
