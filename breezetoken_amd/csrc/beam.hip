// Beam search's selection for gfx950: of the batch's width x vocab candidates
//   score[b, w] + logit[b, w, v] - log sum_u exp(logit[b, w, u])
// the best `beams` of each batch item, with the beam they continue and their token.
//
// A beam's candidates are ordered by their logits, equal ones by token; those of two
// beams by their value in 64 bits, equal ones by beam.  A NaN logit counts as -inf, a
// beam without a finite logit has only candidates of -inf.  A logit of +inf makes its
// beam's others -inf and its own candidate the score less the log of their number.
//
// Every (batch item, beam) row is cut into up to 64 chunks, one wave each, four
// neighbouring chunks a work-group.  A wave holds 4,096 logits in registers at a time.
// The work-group's lanes exchange the largest of theirs: the beams-th largest of these
// 256 values bounds which logits can be chosen, so of 16,384 logits little more than
// `beams` are looked at; they enter the wave's best, sorted 64-bit keys (order of the
// logit, ~token) across its lanes.  The exponentials' reference is a whole number: c, the
// largest's product with log2(e) rounded, so that each is one fused multiply-add
// x log2(e) - c and one v_exp, and sums of any lanes, waves and chunks add after a power
// of two.
//
// The multiply-add rounds to 2^-24 of its result, so far below the reference terms would be
// off by 2^-20, and alike where they are equal.  So c is that of a lane's sixteen logits,
// whose terms weigh the less the more they are off; what is missing from the float over
// log2(e) multiplies their sum.  Eights are added in 32 bits (three levels), the rest in
// 64.  A log-sum is off by 2^-21 at most: 2^-23 of v_exp, 3 x 2^-24 of the eights, and under 2.5 x
// 2^-24 of the exponents and the factor; 0.7 x 2^-22 was the most seen over rows of equal
// logits far below one peak, 1.6 to 2.2 with the work-group's largest as the only reference
// and eights added one by one (2% of the time: 128 rows of bf16 24.7 / 25.1 us, f32 33.5 / 33.7).
// A second kernel, a work-group per batch item, joins the chunks of a row and then the rows.
//
// 128 rows of 248,320 bf16 logits (64 MB): the scan takes 20.5 us, of which its loads alone
// 13 (4.9 TB/s); exponentials and sums, the bound, and the selection add 2 to 3 each, since
// a wave asks for its next logits when it is done with these.  With twice the registers
// and the next ones asked for before the work it took 22: every row is on its way at once
// then.  The join takes 5.6, a chain of dependent steps in a work-group per batch item.
#include "bt_common.h"
#include "bt_kernels.h"

namespace bt {

namespace {

constexpr int kScanWaves = 4;
constexpr int kLoads = 4;    // 16-byte loads of a lane per batch
constexpr int kJoinWaves = 16;
constexpr int kStats = 3;     // of a chunk, behind its keys
constexpr float kLog2e = 1.44269504088896340736f;
// 2^(n kRest) = 1 + n kLog2eRest, kRest what is missing from 1 of the float over log2(e).
constexpr float kLog2eRest = (float)((1.44269504088896340736 / (double)kLog2e - 1.0) * 0.69314718055994530942);

// Order-preserving bits of a float (-0 as +0), and back.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t make_key(float x, int token) {
  return (uint64_t)order_bits(x) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ uint64_t bcast(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// A wave's best keys, sorted: lane i holds the i-th (0: none).
struct Best {
  uint64_t key = 0;
  __device__ __forceinline__ void insert(uint64_t k) {
    const int at = __popcll(__builtin_amdgcn_ballot_w64(key > k));
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)key, 0x138, 0xf, 0xf, false);  // wave_shr:1
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(key >> 32), 0x138, 0xf, 0xf, false);
    const uint64_t up = (uint64_t)hi << 32 | lo;
    key = lane_id() < at ? key : (lane_id() == at ? k : up);
  }
};

// Sum over the wave in 64 bits, in the same order on every run, without an LDS round trip.
template <int MASK>
__device__ __forceinline__ double xor_add64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
  uint64_t a = u, b;
  if constexpr (MASK == 16 || MASK == 32) {
    const auto l = MASK == 16 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto h = MASK == 16 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    a = (uint64_t)h[0] << 32 | l[0];
    b = (uint64_t)h[1] << 32 | l[1];
  } else {
    b = (uint64_t)xor_partner_bits<MASK>(hi) << 32 | xor_partner_bits<MASK>(lo);
  }
  return __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b);
}
__device__ __forceinline__ double wave_sum64(double x) {
  return xor_add64<1>(xor_add64<2>(xor_add64<4>(xor_add64<8>(xor_add64<16>(xor_add64<32>(x))))));
}

// A bound that at least n (1 .. 64) of the wave's 64 N values reach, and not many more than
// 5/4 n where they differ by more than `apart`.  0 is no value: with fewer than n others it is the bound.
// `top`: the largest.
constexpr uint32_t kBf16Apart = 0xfffe;  // order_bits of bf16 values differ by 2^16
template <int N>
__device__ __forceinline__ uint32_t nth_bound(const uint32_t (&x)[N], int n, uint32_t apart, uint32_t& top) {
  uint32_t least = x[0] - 1, most = x[0];
#pragma unroll
  for (int j = 1; j < N; ++j) {
    least = x[j] - 1 < least ? x[j] - 1 : least;
    most = x[j] > most ? x[j] : most;
  }
  uint32_t lo = ~wave_umax(~least) + 1, hi = wave_umax(most);  // `lo`: the smallest value
  top = hi;
  int have = 0;  // reach `lo`
#pragma unroll
  for (int j = 0; j < N; ++j) have += __popcll(__builtin_amdgcn_ballot_w64(x[j] >= lo));
  if (lo == 0 || have < n) return 0;
  // Quarters: three thresholds a step, whose compares do not wait for one another.
#pragma unroll 1
  for (int i = 0; i < 16 && lo < hi && hi - lo > apart && have > n + n / 4; ++i) {
    const uint32_t d = hi - lo, t1 = lo + (d >> 2) + 1, t2 = lo + (d >> 1) + 1, t3 = t2 + (d >> 2);
    int reach1 = 0, reach2 = 0, reach3 = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      reach1 += __popcll(__builtin_amdgcn_ballot_w64(x[j] >= t1));
      reach2 += __popcll(__builtin_amdgcn_ballot_w64(x[j] >= t2));
      reach3 += __popcll(__builtin_amdgcn_ballot_w64(x[j] >= t3));
    }
    if (reach2 >= n) {
      lo = reach3 >= n ? t3 : t2;
      hi = reach3 >= n ? hi : t3 - 1;
      have = reach3 >= n ? reach3 : reach2;
    } else {
      hi = reach1 >= n ? t2 - 1 : t1 - 1;
      lo = reach1 >= n ? t1 : lo;
      have = reach1 >= n ? reach1 : have;
    }
  }
  return lo;
}

// One wave per chunk of a row.
template <bool BF16>
__global__ __launch_bounds__(kScanWaves * 64) void beam_scan_kernel(BeamParams p) {
  constexpr int kVec = BF16 ? 8 : 4;
  constexpr int kElems = kVec * kLoads;      // of a lane per batch
  constexpr int kBatch = 64 * kElems;
  constexpr int kBatches = BF16 ? 2 : 4;     // held in registers: 4,096 logits
  constexpr int kHeld = kBatches * kBatch;
  constexpr int kGroup = 8;                  // logits of a lane tested together
  constexpr int kGroups = kBatches * kElems / kGroup;
  struct __attribute__((packed, aligned(BF16 ? 2 : 4))) Loose { u32x4 v; };  // rows start at any element
  __shared__ uint32_t lane_tops[2][kScanWaves * 64];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = (p.chunks + kScanWaves - 1) / kScanWaves;
  const int row = (int)(blockIdx.x / (unsigned)groups), c = (int)(blockIdx.x % (unsigned)groups) * kScanWaves + wave;
  const char* src = reinterpret_cast<const char*>(p.logits) +
                    (row / p.width * p.stride_batch + row % p.width * p.stride_beam) * (BF16 ? 2 : 4);
  const int v0 = c < p.chunks ? c * p.chunk_size : p.vocab;  // a wave past the last chunk has no logits
  const int v1 = c < p.chunks - 1 ? v0 + p.chunk_size : p.vocab;

  // Logit e of a lane's batch that starts at v is that of token v + token_of(e).
  auto token_of = [&](int e) { return e / kVec * (64 * kVec) + lane * kVec + e % kVec; };
  auto logit = [&](const u32x4 (&raw)[kLoads], int e) -> float {
    if constexpr (BF16) {
      const uint32_t w = raw[e / 8][e % 8 / 2];
      return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    } else {
      return __uint_as_float(raw[e / 4][e % 4]);
    }
  };
  auto load = [&](u32x4 (&raw)[kLoads], int v) {
    if (v + kBatch <= v1) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        raw[j] = reinterpret_cast<const Loose*>(src + (int64_t)(v + token_of(j * kVec)) * (BF16 ? 2 : 4))->v;
    } else {  // the chunk's end: -inf past it
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int t = v + token_of(j * kVec);
        if (t + kVec <= v1) {
          raw[j] = reinterpret_cast<const Loose*>(src + (int64_t)t * (BF16 ? 2 : 4))->v;
        } else if constexpr (BF16) {
          uint32_t x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = t + i < v1 ? reinterpret_cast<const uint16_t*>(src)[t + i] : 0xff80u;
#pragma unroll
          for (int i = 0; i < 4; ++i) raw[j][i] = pack2(x[2 * i], x[2 * i + 1]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) raw[j][i] = t + i < v1 ? reinterpret_cast<const uint32_t*>(src)[t + i] : 0xff800000u;
        }
      }
    }
  };

  const int beams = p.beams;
  Best best;
  float bound = -INFINITY;  // `beams` logits of the work-group's reach it
  float top = -INFINITY;    // the work-group's largest
  float ref = 0.f;          // the sum's reference: 2^ref
  double sum = 0;
  u32x4 raw[kBatches][kLoads];
  for (int s = 0, odd = 0; s < p.chunk_size; s += kHeld, odd ^= 1) {
    const int v = v0 + s;
#pragma unroll
    for (int i = 0; i < kBatches; ++i)
      if (v + i * kBatch < v1) load(raw[i], v + i * kBatch);
    float most[kGroups], mine = -INFINITY;  // fmaxf leaves NaN out
#pragma unroll
    for (int i = 0; i < kBatches; ++i) {
#pragma unroll
      for (int g = 0; g < kElems / kGroup; ++g) {
        float x = -INFINITY;
        if (v + i * kBatch < v1) {
#pragma unroll
          for (int e = 0; e < kGroup; ++e) x = fmaxf(x, logit(raw[i], g * kGroup + e));
        }
        most[i * (kElems / kGroup) + g] = x;
        mine = fmaxf(mine, x);
      }
    }
    // (Two buffers: a wave that is a pass ahead writes the other one.)
    lane_tops[odd][threadIdx.x] = order_bits(mine);
    __syncthreads();
    uint32_t tops[kScanWaves], highest;
#pragma unroll
    for (int j = 0; j < kScanWaves; ++j) tops[j] = lane_tops[odd][j * 64 + lane];
    bound = fmaxf(bound, from_order(nth_bound(tops, beams, BF16 ? kBf16Apart : 0, highest)));
    top = fmaxf(top, from_order(highest));
    if (v >= v1) continue;

    const float now = top == -INFINITY ? 0.f : rintf(top * kLog2e);
    if (sum != 0.0) sum *= (double)fast_exp2(ref - now);  // whole numbers, falling: exact, or past all that counts
    ref = now;
#pragma unroll
    for (int i = 0; i < kBatches; ++i) {
      if (v + i * kBatch >= v1) break;
#pragma unroll
      for (int e0 = 0; e0 < kElems; e0 += 2 * kGroup) {
        const int g = (i * kElems + e0) / kGroup;
        const float own = fmaxf(rintf(fmaxf(most[g], most[g + 1]) * kLog2e), ref - 256.f);
        float part[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[kGroup];
#pragma unroll
          for (int e = 0; e < kGroup; ++e) x[e] = fast_exp2(fmaf(logit(raw[i], e0 + h * kGroup + e), kLog2e, -own));
          part[h] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        }
        sum += ((double)part[0] + (double)part[1]) * (double)(fast_exp2(own - ref) * fmaf(own, kLog2eRest, 1.f));
      }
    }

    uint64_t least = bcast(best.key, beams - 1);
#pragma unroll
    for (int i = 0; i < kBatches; ++i) {
      if (v + i * kBatch >= v1) break;
#pragma unroll
      for (int g = 0; g < kElems / kGroup; ++g) {
        if (!__builtin_amdgcn_ballot_w64(most[i * (kElems / kGroup) + g] >= bound)) continue;
#pragma unroll
        for (int e = g * kGroup; e < (g + 1) * kGroup; ++e) {
          const float x = logit(raw[i], e);
          if (!__builtin_amdgcn_ballot_w64(!(x < bound))) continue;  // NaN counts as -inf
          const int t = v + i * kBatch + token_of(e);
          const uint64_t k = t < v1 ? make_key(fmaxf(x, -INFINITY), t) : 0;
          uint64_t mask = __builtin_amdgcn_ballot_w64(!(x < bound) && k > least);
          if (mask) {
            do {
              const int l = __builtin_ctzll(mask);
              mask &= mask - 1;
              best.insert(bcast(k, l));
            } while (mask);
            least = bcast(best.key, beams - 1);
          }
        }
      }
    }
  }
  if (c >= p.chunks) return;
  // Over the lanes.  Where a logit is NaN or +inf, or so large that the reference's rounding is more than the
  // exponent's, once more with care, relative to the largest.
  const bool careful = __builtin_amdgcn_ballot_w64(sum != sum) || !(fabsf(top) <= 4096.f || top == -INFINITY);
  if (careful) {
    sum = 0;
    for (int t = v0 + lane; t < v1; t += 64) {
      const float x = fmaxf(BF16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(src)[t]) : reinterpret_cast<const float*>(src)[t],
                            -INFINITY);
      sum += x == top ? 1.0 : exp((double)x - (double)top);
    }
  }
  sum = wave_sum64(sum);

  uint64_t* keys = reinterpret_cast<uint64_t*>(p.ws) + (int64_t)row * p.chunks * (beams + kStats);
  if (lane < beams) keys[(int64_t)lane * p.chunks + c] = best.key;  // [place][chunk]
  double* stats = reinterpret_cast<double*>(keys + (int64_t)beams * p.chunks);
  if (lane == 0) {
    stats[c] = (double)top;
    stats[p.chunks + c] = sum;
    stats[2 * p.chunks + c] = careful ? __builtin_nan("") : (double)ref;  // sum * 2^ref, or (NaN) sum * e^top
  }
}

// A wave's candidates in LDS, appended as they come.  Where no more fit, and at the end, each lane
// counts how many are larger than its two (keys differ): its place in order.
constexpr int kListed = 2 * kMaxBeams;  // the best `beams` and 64 more
struct Listed {
  uint64_t* list;
  int beams, n = 0;
  uint64_t least = 0;  // the beams-th best when last sorted
  __device__ __forceinline__ void sort() {
    const int lane = lane_id();
    __builtin_amdgcn_wave_barrier();
    const uint64_t a = lane < n ? list[lane] : 0, b = lane + 64 < n ? list[lane + 64] : 0;
    int before_a = 0, before_b = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const uint64_t x = list[j];
      before_a += x > a;
      before_b += x > b;
    }
    __builtin_amdgcn_wave_barrier();
    if (lane < n && before_a < beams) list[before_a] = a;
    if (lane + 64 < n && before_b < beams) list[before_b] = b;
    __builtin_amdgcn_wave_barrier();
    if (n >= beams) {
      n = beams;
      least = list[beams - 1];
    }
  }
  // The lanes' keys for which `want` holds and that may be among the best (0 is none); whether there were any.
  __device__ __forceinline__ bool add(uint64_t k, bool want) {
    uint64_t mask = __builtin_amdgcn_ballot_w64(want && k > least);
    if (n + __popcll(mask) > kListed) {
      sort();
      mask = __builtin_amdgcn_ballot_w64(want && k > least);
    }
    const int at = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    if (mask >> lane_id() & 1) list[at] = k;
    n += __popcll(mask);
    return mask != 0;
  }
};

__global__ __launch_bounds__(kJoinWaves * 64) void beam_join_kernel(BeamParams p) {
  __shared__ uint64_t lists[kJoinWaves][kListed];
  __shared__ uint64_t row_keys[kMaxBeamWidth * kMaxBeams];
  __shared__ uint64_t order[kMaxBeamWidth * (kMaxBeams | 1)];  // rows of beams | 1: an odd pitch keeps rows' places in banks of their own
  __shared__ int ranks[kMaxBeamWidth * kMaxBeams];
  __shared__ double row_max[kMaxBeamWidth], row_add[kMaxBeamWidth];
  __shared__ uint32_t bound_of_all;
  __shared__ int num_picked;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x, beams = p.beams, chunks = p.chunks;
  for (int w = wave; w < p.width; w += (int)(blockDim.x >> 6)) {
    const uint64_t* keys = reinterpret_cast<const uint64_t*>(p.ws) + ((int64_t)b * p.width + w) * chunks * (beams + kStats);
    const double* stats = reinterpret_cast<const double*>(keys + (int64_t)beams * chunks);
    const bool mine = lane < chunks;
    const double m = mine ? stats[lane] : -(double)INFINITY;
    double sum = mine ? stats[chunks + lane] : 0.0;
    const double ref = mine ? stats[2 * chunks + lane] : 0.0;
    const float score = p.scores[(int64_t)b * p.width + w];
    // The chunks' lists are sorted.  Their first keys, or where those are too few the first four, bound which
    // are looked at, little more than `beams`; the places come one after the other while there are any.  Four
    // are on their way at a time.
    Listed best{lists[wave], beams};
    uint32_t bound = 0;
    bool more = true;
    for (int i0 = 0; i0 < beams && more; i0 += 4) {
      uint64_t k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = mine && i0 + i < beams ? keys[(int64_t)(i0 + i) * chunks + lane] : 0;
      if (i0 == 0) {
        const uint32_t x[4] = {(uint32_t)(k[0] >> 32), (uint32_t)(k[1] >> 32), (uint32_t)(k[2] >> 32), (uint32_t)(k[3] >> 32)};
        const uint32_t first[1] = {x[0]};
        uint32_t unused;
        const uint32_t apart = p.bf16 ? kBf16Apart : 0;
        bound = chunks > beams ? nth_bound(first, beams, apart, unused) : nth_bound(x, beams, apart, unused);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (more) more = best.add(k[i], (uint32_t)(k[i] >> 32) >= bound);
    }
    best.sort();
    if (lane < beams) row_keys[w * beams + lane] = lane < best.n ? best.list[lane] : 0;
    const double top = (double)wave_fmaxf((float)m);
    // Relative to the row's largest.
    const double power = ref != ref ? (m - top) * 1.4426950408889634 : ref - top * 1.4426950408889634;
    sum = wave_sum64(sum == 0.0 || (ref != ref && m == top) ? sum : sum * exp2(power));
    if (lane == 0) {
      row_max[w] = top;
      row_add[w] = (double)score - log(sum);
    }
  }
  __syncthreads();
  // Every row's candidates by their value; where they are many, those that the rows' first four bound (little
  // more than `beams`); then each one's rank: how many of the other rows' sorted lists come before it.  (us of the
  // join, all ranked / the bounded: 8 rows of 8 candidates 5.6 / 6.6, 16 of 8 7.7 / 7.7, 16 of 16 10.5 / 9.1, 32
  // of 32 40 / 19.)
  const int all = p.width * beams, pitch = beams | 1;
  for (int i = threadIdx.x; i < all; i += blockDim.x) {
    const uint64_t key = row_keys[i];
    const double top = row_max[i / beams], add = row_add[i / beams];
    const double x = (double)from_order((uint32_t)(key >> 32));
    double v = x == top && x != -(double)INFINITY ? add : x - top + add;
    v = v != v ? -(double)INFINITY : v + 0.0;
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    order[i / beams * pitch + i % beams] = key ? (u >> 63 ? ~u : u | 1ull << 63) : 0;  // 0: no candidate, behind every other
    ranks[i] = i % beams;
  }
  __syncthreads();
  const bool prune = all * p.width > 2048;
  int* picked = reinterpret_cast<int*>(lists);
  static_assert(sizeof(lists) >= sizeof(ranks), "every candidate may be picked");
  int few = all;
  if (prune) {
    if (wave == 0) {
      uint32_t x[4], unused;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = lane < p.width && j < beams ? (uint32_t)(order[lane * pitch + j] >> 32) : 0;
      const uint32_t bound = nth_bound(x, beams, 0, unused);
      if (lane == 0) {
        bound_of_all = bound;
        num_picked = 0;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < all; i += blockDim.x)
      if ((uint32_t)(order[i / beams * pitch + i % beams] >> 32) >= bound_of_all) picked[atomicAdd(&num_picked, 1)] = i;
    __syncthreads();
    few = num_picked;
  }
  for (int i = threadIdx.x; i < few * p.width; i += blockDim.x) {
    const int j = i % few, c = prune ? picked[j] : j, o = i / few, w = c / beams;
    const uint64_t mine = order[w * pitch + c % beams];
    if (mine == 0 || o == w) continue;
    const uint64_t least = o < w ? mine : mine + 1;  // equal ones of lower rows come before
    int lo = 0, hi = beams;  // places of row o that come before: [0, lo), from hi on none
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (order[o * pitch + mid] >= least) lo = mid + 1;
      else hi = mid;
    }
    if (lo) atomicAdd(ranks + c, lo);
  }
  __syncthreads();
  for (int j = threadIdx.x; j < few; j += blockDim.x) {
    const int i = prune ? picked[j] : j, rank = ranks[i];
    const uint64_t mine = order[i / beams * pitch + i % beams];
    if (mine && rank < beams) {
      const int64_t out = (int64_t)b * beams + rank;
      const uint64_t u = mine >> 63 ? mine & ~(1ull << 63) : ~mine;
      p.scores_out[out] = (float)__builtin_bit_cast(double, u);
      p.parent_out[out] = b * p.width + i / beams;
      p.token_out[out] = (int)~(uint32_t)row_keys[i];
    }
  }
}

}  // namespace

// Chunks of a row, at most 64, and their size (whole wave loads): 4,096 waves in all where
// the rows are long enough, each at least 2,048 logits (a bf16 batch), whole work-groups.  us a call, bf16: 128
// rows of 248,320 26, with 2,048 waves 30; 128 rows of 32,000 13.7 with 1,000 logits a wave,
// 12.3 with 2,000 (before the join's last changes, on both sides).
int beam_chunks(int batch, int width, int vocab, int* size) {
  const int64_t rows = (int64_t)batch * width;
  int64_t want = (4096 + rows - 1) / rows;
  want = (want + kScanWaves - 1) / kScanWaves * kScanWaves;
  want = want < 64 ? want : 64;
  const int64_t most = ((int64_t)vocab + 2047) / 2048;
  want = want < most ? want : most;
  const int64_t per = ((int64_t)vocab + want - 1) / want;
  const int64_t unit = 512;
  *size = (int)((per + unit - 1) / unit * unit);
  return (int)(((int64_t)vocab + *size - 1) / *size);
}

int64_t beam_ws_bytes(int batch, int width, int vocab, int beams) {
  int size;
  return (int64_t)batch * width * beam_chunks(batch, width, vocab, &size) * (beams + kStats) * 8;
}

hipError_t launch_beam_select(const BeamParams& params, hipStream_t stream) {
  BeamParams p = params;
  p.chunks = beam_chunks(p.batch, p.width, p.vocab, &p.chunk_size);
  const dim3 grid((unsigned)((int64_t)p.batch * p.width * ((p.chunks + kScanWaves - 1) / kScanWaves))), block(kScanWaves * 64);
  if (p.bf16) hipLaunchKernelGGL(beam_scan_kernel<true>, grid, block, 0, stream, p);
  else hipLaunchKernelGGL(beam_scan_kernel<false>, grid, block, 0, stream, p);
  const int join = p.width < kJoinWaves ? p.width : kJoinWaves;
  hipLaunchKernelGGL(beam_join_kernel, dim3(p.batch), dim3(join * 64), 0, stream, p);
  return hipGetLastError();
}

}  // namespace bt
