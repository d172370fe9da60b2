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
//
// Bound by memory: 8,192 tokens of H = 8, Hkv = 2, D = 256 (f32, gated, norm) take
// 36 us, 4.8 TB/s, what a large copy reaches.  A wave takes kRows rows of one token
// for each of its row slots (a row of D values lies in D / 4 lanes, 8 values a lane at
// D = 512): the loads of all of them go out together, and the token's position, page
// and angles are read once.  In the half layout a value's partner comes through LDS (16 bytes a lane
// where the half is a multiple of 4), in the interleaved one it is in the lane.
#include "bt_common.h"
#include "bt_kernels.h"

namespace bt {

namespace {

constexpr int kWaves = 4;
// Calls whose rows all fit the chip at once, a row slot a wave (256 CUs hold 8,192 waves), take one row a
// slot: latency counts.  One / four rows, us a graph node, H = 32, Hkv = 8, D = 128 (24 waves a token): 24
// tokens 3.5 / 4.3, 256 4.7 / 5.3, 512 7.5 / 6.6, 2,048 19.3 / 15.2; H = 8, Hkv = 2, D = 256 (12 waves): 24
// tokens 3.3 / 4.1, 512 5.6 / 6.1, 1,024 8.4 / 7.8.
constexpr int64_t kFewWaves = 8192;

enum Rope : int { kNone = 0, kHalf = 1, kHalfOdd = 2, kPairs = 3 };  // kHalfOdd: a half that is no multiple of 4

struct __attribute__((packed, aligned(4))) Loose4 {  // tables need no more than a float's alignment
  float v[4];
};

template <int D, bool XBF16, int ROPE, int kRows>
__global__ __launch_bounds__(kWaves * 64) void paged_prep_kernel(PagedPrepParams p, int groups) {
  constexpr int E = D == 512 ? 8 : 4;  // values of a lane
  constexpr int kLanes = D / E;        // lanes of a row
  constexpr int kSlots = 64 / kLanes;  // rows side by side in a wave
  __shared__ __attribute__((aligned(16))) float lds[ROPE == kHalf || ROPE == kHalfOdd ? kWaves * 64 * E : 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned id = blockIdx.x * kWaves + wave;
  if (id >= (unsigned)p.tokens * (unsigned)groups) return;
  const int t = (int)(id / (unsigned)groups), g = (int)(id % (unsigned)groups);
  const int d0 = lane % kLanes * E;
  const int k0 = p.heads, v0 = p.heads + p.kv_heads, rows = p.heads + 2 * p.kv_heads;
  const int row0 = g * kRows * kSlots + lane / kLanes;
  auto row_of = [&](int j) { return row0 + j * kSlots; };

  // ---- the rows' values ---------------------------------------------------------
  const int step = p.gated ? 2 * D : D;
  const int64_t token = (int64_t)t * p.x_stride;
  float x[kRows][E];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int r = row_of(j);
    if (r < rows) {
      const int64_t at = token + (r < k0 ? r * step : p.heads * step + (r - k0) * D) + d0;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        if constexpr (XBF16) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint16_t*>(p.x) + at + e);
          x[j][e] = __uint_as_float(w[0] << 16);
          x[j][e + 1] = __uint_as_float(w[0] & 0xffff0000u);
          x[j][e + 2] = __uint_as_float(w[1] << 16);
          x[j][e + 3] = __uint_as_float(w[1] & 0xffff0000u);
        } else {
          const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.x) + at + e);
          x[j][e] = w.x;
          x[j][e + 1] = w.y;
          x[j][e + 2] = w.z;
          x[j][e + 3] = w.w;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[j][e] = 0.f;
    }
  }

  // ---- the token's slot and angles -------------------------------------------------
  const int pos = __builtin_amdgcn_readfirstlane(p.pos[t]);
  const int seq = p.rows ? __builtin_amdgcn_readfirstlane(p.rows[t]) : t;
  int page = -1;
  if (seq >= 0 && seq < p.table_rows && pos >= 0 && pos >> p.pg.page_shift < p.pg.pages_per_seq)
    page = __builtin_amdgcn_readfirstlane(p.pg.table[(int64_t)seq * p.pg.table_stride + (pos >> p.pg.page_shift)]);
  const bool slot = page >= 0 && page < p.pg.num_pages;
  const int64_t slot_at = (int64_t)page * p.pg.stride_page + (int64_t)(pos & ((1 << p.pg.page_shift) - 1)) * p.pg.stride_tok;
  float cs[E], sn[E];  // per value (half layouts) or per pair
  const int half = p.rope_dim >> 1;
  const bool turned = ROPE != kNone && d0 < p.rope_dim;
  if constexpr (ROPE != kNone) {
    const int pr = pos < 0 ? 0 : (pos >= p.rope_cap ? p.rope_cap - 1 : pos);
    const float* c = p.cos + (int64_t)pr * p.rope_dim;
    const float* s = p.sin + (int64_t)pr * p.rope_dim;
    if (turned) {
      if constexpr (ROPE == kHalf) {
        const int i0 = d0 < half ? d0 : d0 - half;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          // At D = 512 a lane's second four may lie past the half, or past rope_dim.
          const int d = d0 + e, i = E == 4 ? i0 : (d < half ? d : (d < p.rope_dim ? d - half : 0));
          const Loose4 cc = *reinterpret_cast<const Loose4*>(c + i), ss = *reinterpret_cast<const Loose4*>(s + i);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            cs[e + q] = cc.v[q];
            sn[e + q] = ss.v[q];
          }
        }
      } else if constexpr (ROPE == kHalfOdd) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int d = d0 + e, i = d < half ? d : (d < p.rope_dim ? d - half : 0);
          cs[e] = c[i];
          sn[e] = s[i];
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const int i = d0 + e < p.rope_dim ? (d0 + e) >> 1 : 0;
          cs[e] = c[i];
          sn[e] = s[i];
        }
      }
    }
  }
  float* part = lds + wave * 64 * E;  // this wave's: its LDS operations stay in order

#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int r = row_of(j);
    const bool is_v = r >= v0;
    // ---- norm --------------------------------------------------------------------
    if (p.wq != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(x[j][e], x[j][e], ss);
      ss = xor_sum<8>(xor_sum<4>(xor_sum<2>(xor_sum<1>(ss))));
      if constexpr (kLanes >= 32) ss = rows16_sum(ss);
      if constexpr (kLanes >= 64) ss = halves_sum(ss);
      const float f = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
      if (!is_v) {
        const float* w = (r < k0 ? p.wq : p.wk) + d0;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          const float4 ww = *reinterpret_cast<const float4*>(w + e);
          x[j][e] *= f * ww.x;
          x[j][e + 1] *= f * ww.y;
          x[j][e + 2] *= f * ww.z;
          x[j][e + 3] *= f * ww.w;
        }
      }
    }
    // ---- rotation ------------------------------------------------------------------
    if constexpr (ROPE == kHalf || ROPE == kHalfOdd) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(part + lane * E + e) = float4{x[j][e], x[j][e + 1], x[j][e + 2], x[j][e + 3]};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (turned && !is_v) {
        const float* row = part + lane / kLanes * D;
#pragma unroll
        for (int e = 0; e < E; e += (ROPE == kHalf ? 4 : 1)) {
          const int d = d0 + e;
          if (d < p.rope_dim) {
            const bool first = d < half;
            const float* other = row + (first ? d + half : d - half);
            if constexpr (ROPE == kHalf) {
              const float4 o = *reinterpret_cast<const float4*>(other);
              const float sg = first ? -1.f : 1.f;
              x[j][e] = x[j][e] * cs[e] + sg * o.x * sn[e];
              x[j][e + 1] = x[j][e + 1] * cs[e + 1] + sg * o.y * sn[e + 1];
              x[j][e + 2] = x[j][e + 2] * cs[e + 2] + sg * o.z * sn[e + 2];
              x[j][e + 3] = x[j][e + 3] * cs[e + 3] + sg * o.w * sn[e + 3];
            } else {
              x[j][e] = x[j][e] * cs[e] + (first ? -*other : *other) * sn[e];
            }
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before the next row's values take the place
    } else if constexpr (ROPE == kPairs) {
      if (turned && !is_v) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          if (d0 + e < p.rope_dim) {
            const float a = x[j][e], b = x[j][e + 1];
            x[j][e] = a * cs[e] - b * sn[e];
            x[j][e + 1] = b * cs[e] + a * sn[e];
          }
        }
      }
    }
    // ---- out -----------------------------------------------------------------------
    if (r >= rows) continue;
    if (r < k0 && !p.q_out_bf16) {
      float* dst = reinterpret_cast<float*>(p.q_out) + ((int64_t)t * p.heads + r) * D + d0;
#pragma unroll
      for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(dst + e) = float4{x[j][e], x[j][e + 1], x[j][e + 2], x[j][e + 3]};
    } else {
      if (r >= k0 && !slot) continue;
      uint16_t* dst = r < k0 ? reinterpret_cast<uint16_t*>(p.q_out) + ((int64_t)t * p.heads + r) * D
                             : (is_v ? p.v : p.k) + slot_at + (int64_t)(r - (is_v ? v0 : k0)) * p.pg.stride_head;
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<u32x2*>(dst + d0 + e) = u32x2{f32x2_to_bf16x2_bits(x[j][e], x[j][e + 1]), f32x2_to_bf16x2_bits(x[j][e + 2], x[j][e + 3])};
    }
  }
}

template <int D, bool XBF16, int ROPE>
hipError_t launch_rope(const PagedPrepParams& p, hipStream_t stream) {
  constexpr int kSlots = 64 / (D / (D == 512 ? 8 : 4));
  const int rows = p.heads + 2 * p.kv_heads;
  auto launch = [&](auto kernel, int per) {
    const int groups = (rows + per - 1) / per;
    const dim3 grid((unsigned)(((int64_t)p.tokens * groups + kWaves - 1) / kWaves));
    hipLaunchKernelGGL(kernel, grid, dim3(kWaves * 64), 0, stream, p, groups);
    return hipGetLastError();
  };
  if ((int64_t)p.tokens * ((rows + kSlots - 1) / kSlots) <= kFewWaves) return launch(paged_prep_kernel<D, XBF16, ROPE, 1>, kSlots);
  return launch(paged_prep_kernel<D, XBF16, ROPE, 4>, 4 * kSlots);
}

template <int D, bool XBF16>
hipError_t launch_dim(const PagedPrepParams& p, hipStream_t stream) {
  if (!p.cos) return launch_rope<D, XBF16, kNone>(p, stream);
  if (p.interleaved) return launch_rope<D, XBF16, kPairs>(p, stream);
  return p.rope_dim % 8 == 0 ? launch_rope<D, XBF16, kHalf>(p, stream) : launch_rope<D, XBF16, kHalfOdd>(p, stream);
}

}  // namespace

hipError_t launch_paged_prep(const PagedPrepParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return p.x_bf16 ? launch_dim<64, true>(p, stream) : launch_dim<64, false>(p, stream);
    case 128: return p.x_bf16 ? launch_dim<128, true>(p, stream) : launch_dim<128, false>(p, stream);
    case 256: return p.x_bf16 ? launch_dim<256, true>(p, stream) : launch_dim<256, false>(p, stream);
    case 512: return p.x_bf16 ? launch_dim<512, true>(p, stream) : launch_dim<512, false>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bt
