// Which pages a new token attends (gfx950): bounds of the keys of each page, and the
// choice of pages by them.
//
//   low / high[page, g, d] = min / max over the page's tokens of k[token, g, d]   (NaN keys left out)
//   score[b, g, e] = max over the group's heads h of sum_d q_hd (q_hd > 0 ? high_d : low_d)
//     >= every product of those heads with a key of page table[b, e]; -inf where a channel has no number (low > high)
//   chosen[b, g]: the last page, and the best count - 1 of the others (ties: the lower
//     entry), in the order of the table
//
// Scores are sums in 64 bits: the choice is by value, and two pages may lie nearer to each
// other than 32 bits resolve.  (A product of an f32 and a bf16 value is exact in 64 bits.)
//
// Bounds are bound by the one read of K: 241 MB (32 sequences of 256 to 32,768 tokens, pages
// of 32, Hkv = 2, D = 256) in 51 us, 4.7 TB/s where a large copy reaches 4.9; the newest pages
// of 128 sequences take 5.0 us, a chain of loads.  Scores read 35 MB of bounds (32 sequences of
// 8,192 to 32,768 tokens, H = 8) in 13 to 14 us, 2.4 to 2.7 TB/s, between the stream and the 64-bit products;
// the choice of 63 of up to 1,023 pages takes 6 us, of one among 2,047 5, a chain of barriers.
#include "bt_common.h"
#include "bt_decode.h"
#include "bt_kernels.h"

namespace bt {

namespace {

// ---------------------------------------------------------------------- bounds
constexpr int kBoundWaves = 4;
constexpr int kBoundGroups = 2048;  // work-groups of a launch at most (1,024 and 8,192: 52.3 and 51.7 us for 52.1)
// Tokens from which on a page is the work of four waves, not one.  One / four, us, pages of 32, 64, 128, 1,024 (Hkv = 2,
// D = 256): all keys of 32 sequences of 256 to 32,768 tokens 53 / 67, 48 / 53, 46 / 46, 72 / 46; the newest pages of
// 128 sequences 5.3 / 5.1, 6.3 / 5.2, 8.1 / 5.8, and of 512 25.7 / 14.9.
constexpr int kSharedPage = 128;

// Items are the (row, entry) pairs to do, numbered through, times kv heads.  SHARED: a
// work-group takes one, else a wave does.
template <int D, bool SHARED>
__global__ __launch_bounds__(kBoundWaves * 64) void key_bounds_kernel(BoundsParams p) {
  constexpr int kLanes = D / 8;        // of a token's row
  constexpr int kRows = 64 / kLanes;   // tokens of a wave load
  constexpr int kAhead = 8;            // loads on their way
  constexpr int kStep = SHARED ? kBoundWaves : 1;
  extern __shared__ int ends[];  // items up to and with each row
  __shared__ int wsum[64];
  __shared__ float joined[SHARED ? kBoundWaves * 2 * D : 1];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int size = 1 << p.pg.page_shift, cap = p.pg.pages_per_seq << p.pg.page_shift;
  auto tokens_of = [&](int b) {
    const int n = p.lens[b];
    return n < 0 ? 0 : (n > cap ? cap : n);
  };
  auto first_of = [&](int b, int n) -> int {
    const int f = p.first ? p.first[b] : 0;
    return f >= n ? (n + size - 1) >> p.pg.page_shift : (f < 0 ? 0 : f) >> p.pg.page_shift;
  };
  const int windows = (p.batch + 63) >> 6;
  for (int i = wave; i < windows; i += kBoundWaves) {
    const int b = 64 * i + lane;
    int x = 0;
    if (b < p.batch) {
      const int n = tokens_of(b);
      x = ((n + size - 1) >> p.pg.page_shift) - first_of(b, n);
    }
    const int e = wave_scan(x);
    if (b < p.batch) ends[b] = e;
    if (lane == 63) wsum[i] = e;
  }
  __syncthreads();
  const int wends = wave_scan(lane < windows ? wsum[lane] : 0);
  const int total = __builtin_amdgcn_readlane(wends, 63);

  const int64_t items = (int64_t)total * p.kv_heads;
  const int64_t hop = (int64_t)gridDim.x * (kBoundWaves / kStep);
  for (int64_t item = (int64_t)blockIdx.x * (kBoundWaves / kStep) + (SHARED ? 0 : wave); item < items; item += hop) {
    const int t = uniform((int)(item / p.kv_heads)), g = uniform((int)(item % p.kv_heads));
    const int i = __popcll(__builtin_amdgcn_ballot_w64(wends <= t));  // its window
    const int before = i ? __builtin_amdgcn_readlane(wends, i - 1) : 0;
    int at = 64 * i + lane;
    const int in = __popcll(__builtin_amdgcn_ballot_w64(at < p.batch && ends[at < p.batch ? at : 0] <= t - before));
    const int b = uniform(64 * i + in);
    const int row0 = before + (in ? uniform(ends[b - 1]) : 0);
    const int n = uniform(tokens_of(b));
    const int entry = uniform(first_of(b, n)) + t - row0;
    const int page = uniform(p.pg.table[(int64_t)b * p.pg.table_stride + entry]);
    if ((uint32_t)page >= (uint32_t)p.pg.num_pages) continue;
    int fill = n - (entry << p.pg.page_shift);
    if (fill < size) {
      // A partly filled page may be another row's too, with more tokens: every row that holds it in
      // this entry writes the bounds of the most.
      int most = 0;
      for (int r = lane; r < p.batch; r += 64)
        if (p.pg.table[(int64_t)r * p.pg.table_stride + entry] == page) {
          const int m = tokens_of(r) - (entry << p.pg.page_shift);
          most = m > most ? m : most;
        }
      fill = (int)wave_op_desc((uint32_t)most, OpIMax{});
    }
    fill = uniform(fill < size ? fill : size);

    // ---- the tokens: eight values of one in a lane --------------------------------------
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = INFINITY;
      hi[e] = -INFINITY;
    }
    const uint16_t* k = p.k + (int64_t)page * p.pg.stride_page + (int64_t)g * p.pg.stride_head + lane % kLanes * 8;
    auto take = [&](const u32x4& v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
        lo[e] = fminf(lo[e], f);
        hi[e] = fmaxf(hi[e], f);
      }
    };
    const int part = SHARED ? wave : 0;
    for (int t0 = part * kRows * kAhead; t0 < fill; t0 += kStep * kRows * kAhead) {
      u32x4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        // Past the last token: the first of the batch again.
        int token = t0 + j * kRows + lane / kLanes;
        token = token < fill ? token : t0;
        v[j] = *reinterpret_cast<const u32x4*>(k + (int64_t)token * p.pg.stride_tok);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) take(v[j]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kLanes <= 8) {
        lo[e] = -xor_fmaxf<8>(-lo[e]);
        hi[e] = xor_fmaxf<8>(hi[e]);
      }
      if constexpr (kLanes <= 16) {
        lo[e] = -rows16_fmaxf(-lo[e]);
        hi[e] = rows16_fmaxf(hi[e]);
      }
      lo[e] = -halves_fmaxf(-lo[e]);
      hi[e] = halves_fmaxf(hi[e]);
    }
    uint16_t* out = p.bounds + ((int64_t)page * p.kv_heads + g) * 2 * D;
    if constexpr (SHARED) {
      __syncthreads();
      if (lane < kLanes) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          joined[(wave * 2) * D + lane * 8 + e] = lo[e];
          joined[(wave * 2 + 1) * D + lane * 8 + e] = hi[e];
        }
      }
      __syncthreads();
      for (int d = threadIdx.x; d < 2 * D; d += kBoundWaves * 64) {
        float x = joined[d];
#pragma unroll
        for (int i = 1; i < kBoundWaves; ++i) x = d < D ? fminf(x, joined[i * 2 * D + d]) : fmaxf(x, joined[i * 2 * D + d]);
        out[d] = (uint16_t)f32_to_bf16_bits(x);
      }
    } else if (lane < kLanes) {
      u32x4 a, c;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = f32x2_to_bf16x2_bits(lo[2 * e], lo[2 * e + 1]);
        c[e] = f32x2_to_bf16x2_bits(hi[2 * e], hi[2 * e + 1]);
      }
      *reinterpret_cast<u32x4*>(out + lane * 8) = a;
      *reinterpret_cast<u32x4*>(out + D + lane * 8) = c;
    }
  }
}

// ---------------------------------------------------------------------- scores
constexpr int kScoreWaves = 4;
constexpr int kScoreAhead = 4;  // pages whose bounds are on their way, for each group of lanes
// Waves of one page for each group of lanes up to which there is no more than one: what a wave does shows where few
// waves are there to hide it.  kScoreAhead / one, us of the sparse attention: 1,024 waves (4 rows of 127 pages, H = 32, Hkv = 8,
// D = 128) 17.35 / 16.3, 2,052 (one of 2,051, H = 16, Hkv = 2, D = 256) 24.0 / 22.8; 4,096 (32 of 128) 33.0 / 34.4.
constexpr int64_t kFewScoreWaves = 2560;
// Waves from which on each takes four times as many pages, to load the queries less often.  One / four times, us:
// 2,112 work-groups (32 sequences of up to 32,768 tokens, pages of 32, H = 8, Hkv = 2, D = 256) 14.6 / 21.6.
constexpr int64_t kManyScoreWaves = 65536;

// x of lane l ^ MASK.
template <int MASK>
__device__ __forceinline__ double xor_move(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  uint32_t w[2] = {(uint32_t)u, (uint32_t)(u >> 32)};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (MASK == 16) {
      const auto r = __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false);  // the even rows' values, the odd rows'
      w[i] = threadIdx.x & 16 ? r[0] : r[1];
    } else {
      w[i] = xor_partner_bits<MASK>(w[i]);
    }
  }
  return __longlong_as_double((long long)((uint64_t)w[1] << 32 | w[0]));
}

// Sums over the 2 * MASK lanes of a page of N heads each, then the largest of them: with every step half the
// heads go to the other half of the lanes, until a lane has one.  head: this lane's, as it is found.
template <int N, int MASK>
__device__ __forceinline__ double largest_sum(double (&x)[N], int head, int group) {
  if constexpr (MASK == 0) {
    const double y = head < group && x[0] == x[0] ? x[0] : -INFINITY;  // not a number: the least
    return y;
  } else if constexpr (N > 1) {
    const bool upper = threadIdx.x & MASK;
    double y[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const double mine = upper ? x[i + N / 2] : x[i], other = upper ? x[i] : x[i + N / 2];
      y[i] = mine + xor_move<MASK>(other);
    }
    const double best = largest_sum<N / 2, MASK / 2>(y, 2 * head + (upper ? 1 : 0), group);
    const double theirs = xor_move<MASK>(best);
    return best > theirs ? best : theirs;
  } else {
    double y[1] = {x[0] + xor_move<MASK>(x[0])};
    return largest_sum<1, MASK / 2>(y, head, group);
  }
}

// A page's bounds lie in D / 8 lanes, eight channels a lane, whose queries of all heads stay there as 64-bit
// values; a wave takes 64 / (D / 8) pages at once, AHEAD times on their way, `batches` times over.
template <int D, int GMAX, int AHEAD>
__global__ __launch_bounds__(kScoreWaves * 64, 2) void page_score_kernel(SelectParams p, int batches) {
  constexpr int kLanes = D / 8, kPages = 64 / kLanes;
  const int kvh = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int cap = p.pg.pages_per_seq << p.pg.page_shift;
  int n = uniform_load(p.lens, b);
  n = n < 0 ? 0 : (n > cap ? cap : n);
  const int others = ((n + (1 << p.pg.page_shift) - 1) >> p.pg.page_shift) - 1;
  if (others < p.count) return;  // every page is kept
  const int first = ((int)blockIdx.x * kScoreWaves + wave) * batches * AHEAD * kPages;
  if (first >= others) return;
  const int c = lane % kLanes * 8;
  const int32_t* table = p.pg.table + (int64_t)b * p.pg.table_stride;
  const uint16_t* bounds = p.bounds + (int64_t)kvh * 2 * D + c;
  double* out = p.score + ((int64_t)b * p.kv_heads + kvh) * p.pg.pages_per_seq;
  double q[GMAX][8];
#pragma unroll
  for (int h = 0; h < GMAX; ++h) {
    const int64_t at = (int64_t)b * p.q_stride_seq + ((int64_t)kvh * p.group + (h < p.group ? h : 0)) * D + c;
    if (p.q_bf16) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.q) + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) q[h][e] = (double)__uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    } else {
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.q) + at);
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.q) + at + 4);
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) q[h][e] = (double)v[e];
    }
  }
  for (int k = 0; k < batches; ++k) {
    const int e0 = first + k * AHEAD * kPages + lane / kLanes;
    if (first + k * AHEAD * kPages >= others) break;
    int page[AHEAD];
    u32x4 lo[AHEAD], hi[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) page[i] = e0 + i * kPages < others ? table[e0 + i * kPages] : -1;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint16_t* at = bounds + ((uint32_t)page[i] < (uint32_t)p.pg.num_pages ? (int64_t)page[i] : 0) * p.kv_heads * 2 * D;
      lo[i] = *reinterpret_cast<const u32x4*>(at);
      hi[i] = *reinterpret_cast<const u32x4*>(at + D);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      double sum[GMAX];
#pragma unroll
      for (int h = 0; h < GMAX; ++h) sum[h] = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double l = (double)__uint_as_float(e & 1 ? lo[i][e >> 1] & 0xffff0000u : lo[i][e >> 1] << 16);
        const double u = (double)__uint_as_float(e & 1 ? hi[i][e >> 1] & 0xffff0000u : hi[i][e >> 1] << 16);
#pragma unroll
        for (int h = 0; h < GMAX; ++h) sum[h] = fma(q[h][e], q[h][e] > 0.0 ? u : l, sum[h]);
      }
      const double best = largest_sum<GMAX, kLanes / 2>(sum, 0, p.group);
      if (lane % kLanes == 0 && e0 + i * kPages < others)
        out[e0 + i * kPages] = (uint32_t)page[i] < (uint32_t)p.pg.num_pages ? best : -INFINITY;
    }
  }
}

// ---------------------------------------------------------------------- choice
constexpr int kChooseThreads = 1024;

// Scores as integers of the same order.
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // -0 as 0
  return u >> 63 ? ~u : u | (1ull << 63);
}

// Lengths and outputs of a (sequence, kv head) whose choice is made; true where all pages are kept.
struct Choice {
  int used, others, want;  // pages; those besides the last; those of them that are taken
  const int32_t* table;
  int32_t* out;
  const double* score;
  __device__ __forceinline__ bool begin(const SelectParams& p, int b, int kvh, int threads) {
    const int tid = threadIdx.x, cap = p.pg.pages_per_seq << p.pg.page_shift;
    int n = uniform_load(p.lens, b);
    n = n < 0 ? 0 : (n > cap ? cap : n);
    used = (n + (1 << p.pg.page_shift) - 1) >> p.pg.page_shift;
    others = used - 1;
    want = p.count - 1;
    table = p.pg.table + (int64_t)b * p.pg.table_stride;
    out = p.chosen + ((int64_t)b * p.kv_heads + kvh) * p.count;
    score = p.score + ((int64_t)b * p.kv_heads + kvh) * p.pg.pages_per_seq;
    const int have = used < p.count ? used : p.count;
    for (int i = have + tid; i < p.count; i += threads) out[i] = -1;
    if (kvh == 0 && tid == 0)
      p.chosen_len[b] = used <= p.count ? n : ((p.count - 1) << p.pg.page_shift) + n - ((used - 1) << p.pg.page_shift);
    if (used <= p.count) {
      for (int i = tid; i < used; i += threads) out[i] = table[i];
      return true;
    }
    if (tid == 0) out[p.count - 1] = table[used - 1];
    return want == 0;
  }
};

// Bins of equal width between the least and the largest finite score, the outer two for the infinite ones; the
// order of bins is that of the scores, so all above the want-th score's bin are taken, and of that bin, which
// holds a page or a few, those that few others of it exceed.
constexpr int kBins = 2048;
constexpr int kPerThread = 8;  // scores a thread holds
constexpr int kListed = 512;   // of one bin that are ranked by counting (bit by bit: 33 and 71 us for 24.5 and 50.5 of the attention)

template <int T>
__global__ __launch_bounds__(T) void page_choose_kernel(SelectParams p, int per) {
  constexpr int kWaves = T / 64, kEach = kBins / T;
  __shared__ int hist[kBins];
  __shared__ double ends[2 * kWaves];
  __shared__ int sums[kWaves], found[3];  // the bin, its pages to take, its pages
  __shared__ double list[kListed];
  __shared__ int list_at[kListed];
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  // `per` consecutive entries a thread, asked for before the row's length is there.  (Where there are no
  // scores there is no place for them.)
  const int first = tid * per;
  double x[kPerThread] = {};
  int id[kPerThread] = {};
  if (p.score) {
    const double* score = p.score + ((int64_t)b * p.kv_heads + kvh) * p.pg.pages_per_seq;
    const int32_t* table = p.pg.table + (int64_t)b * p.pg.table_stride;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int at = i < per && first + i < p.pg.pages_per_seq ? first + i : 0;
      x[i] = score[at];
      id[i] = table[at];
    }
  }
  Choice ch;
  if (ch.begin(p, b, kvh, T)) return;
  const int mine = first >= ch.others ? 0 : (ch.others - first < per ? ch.others - first : per);
  double least = INFINITY, most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) x[i] = i < mine ? x[i] + 0.0 : -INFINITY;  // -0 as 0
#pragma unroll
  for (int i = 0; i < kPerThread; ++i)
    if (fabs(x[i]) < INFINITY) {
      least = x[i] < least ? x[i] : least;
      most = x[i] > most ? x[i] : most;
    }
  for (int i = tid; i < kBins; i += T) hist[i] = 0;
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const double l = __shfl_xor(least, m), h = __shfl_xor(most, m);
    least = l < least ? l : least;
    most = h > most ? h : most;
  }
  if (lane == 0) {
    ends[wave] = least;
    ends[kWaves + wave] = most;
  }
  if (tid == 0) found[2] = 0;
  __syncthreads();
  least = ends[lane % kWaves];
  most = ends[kWaves + lane % kWaves];
#pragma unroll
  for (int m = kWaves / 2; m; m >>= 1) {
    const double l = __shfl_xor(least, m), h = __shfl_xor(most, m);
    least = l < least ? l : least;
    most = h > most ? h : most;
  }
  // At most 1e300, so that scores nearer to each other than 1e-297 fall into one bin and no product is infinite.
  const double per_bin = most > least ? fmin((kBins - 3) / (most - least), 1e300) : 0.0;
  auto bin_of = [&](double v) -> int {
    if (v == -INFINITY) return 0;
    if (v == INFINITY) return kBins - 1;
    const int at = 1 + (int)((v - least) * per_bin);
    return at < kBins - 2 ? at : kBins - 2;
  };
  int bin[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    bin[i] = bin_of(x[i]);
    if (i < mine) atomicAdd(&hist[bin[i]], 1);
  }
  __syncthreads();
  // Thread t holds kEach bins, the highest from kBins - 1 - kEach t down: pages above them.
  int c[kEach], in = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    c[i] = hist[kBins - 1 - kEach * tid - i];
    in += c[i];
  }
  int above = wave_scan(in);
  if (lane == 63) sums[wave] = above;
  above -= in;
  __syncthreads();
  {
    const int upto = wave_scan(lane < kWaves ? sums[lane] : 0);
    above += wave ? __builtin_amdgcn_readlane(upto, wave - 1) : 0;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (above < ch.want && above + c[i] >= ch.want) {
      found[0] = kBins - 1 - kEach * tid - i;
      found[1] = ch.want - above;
    }
    above += c[i];
  }
  __syncthreads();
  const int edge = found[0], take = found[1], members = hist[edge];
  uint32_t taken = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i)
    if (i < mine && (bin[i] > edge || (bin[i] == edge && members == take))) taken |= 1u << i;
  if (members != take && members <= kListed) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (i < mine && bin[i] == edge) {
        const int at = atomicAdd(&found[2], 1);
        list[at] = x[i];
        list_at[at] = first + i;
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (i < mine && bin[i] == edge) {
        int before = 0;
        for (int j = 0; j < members; ++j) before += list[j] > x[i] || (list[j] == x[i] && list_at[j] < first + i);
        if (before < take) taken |= 1u << i;
      }
  } else if (members != take) {
    // Many in one bin: its want-th largest, bit by bit, and of equal ones the first.
    uint64_t low = 0;
    int need = take;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t mark = low | 1ull << bit;
      int c = 0;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) c += i < mine && bin[i] == edge && order_of(x[i]) >> bit == mark >> bit;
      c = (int)wave_op_desc((uint32_t)c, OpIAdd{});
      __syncthreads();
      if (lane == 0) sums[wave] = c;
      __syncthreads();
      const int s = lane < kWaves ? sums[lane] : 0;
      c = (int)wave_op_desc((uint32_t)s, OpIAdd{});
      if (c >= need) low = mark;
      else need -= c;
    }
    int same = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) same += i < mine && bin[i] == edge && order_of(x[i]) == low;
    int rank = wave_scan(same);
    __syncthreads();
    if (lane == 63) sums[wave] = rank;
    rank -= same;
    __syncthreads();
    const int upto = wave_scan(lane < kWaves ? sums[lane] : 0);
    rank += wave ? __builtin_amdgcn_readlane(upto, wave - 1) : 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (i < mine && bin[i] == edge) {
        const uint64_t o = order_of(x[i]);
        if (o > low || (o == low && rank < need)) taken |= 1u << i;
        rank += o == low;
      }
  }
  // Taken pages in the table's order.
  const int count = __popc(taken);
  int at = wave_scan(count);
  __syncthreads();
  if (lane == 63) sums[wave] = at;
  at -= count;
  __syncthreads();
  const int upto = wave_scan(lane < kWaves ? sums[lane] : 0);
  at += wave ? __builtin_amdgcn_readlane(upto, wave - 1) : 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i)
    if (taken >> i & 1) ch.out[at++] = id[i];
}

// The same for rows of more pages than the threads hold: the want-th largest score byte by byte.
__global__ __launch_bounds__(kChooseThreads) void page_choose_long_kernel(SelectParams p) {
  __shared__ int hist[256];
  __shared__ int picked[2];
  __shared__ int sums[2 * kChooseThreads / 64];
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Choice ch;
  if (ch.begin(p, b, kvh, kChooseThreads)) return;
  const int others = ch.others;
  uint64_t edge = 0;
  int equal = ch.want;  // of the edge's value that are taken
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kChooseThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < others; i += kChooseThreads) {
      const uint64_t x = order_of(ch.score[i]);
      if (shift == 56 || x >> (shift + 8) == edge >> (shift + 8)) atomicAdd(&hist[(int)(x >> shift & 255)], 1);
    }
    __syncthreads();
    if (wave == 0) {
      // Lane l holds bytes 255 - 4 l .. 252 - 4 l, the largest first.
      int c[4], s = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = hist[255 - 4 * lane - i];
        s += c[i];
      }
      int above = wave_scan(s) - s;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < equal && above + c[i] >= equal) {
          picked[0] = 255 - 4 * lane - i;
          picked[1] = equal - above;
        }
        above += c[i];
      }
    }
    __syncthreads();
    edge |= (uint64_t)picked[0] << shift;
    equal = picked[1];
    __syncthreads();
  }
  // Taken entries in the table's order.
  int base = 0, base_equal = 0;
  for (int i0 = 0; i0 < others; i0 += kChooseThreads) {
    const int i = i0 + tid;
    const uint64_t x = i < others ? order_of(ch.score[i]) : 0;
    const bool more = i < others && x > edge, same = i < others && x == edge;
    const uint64_t m = __builtin_amdgcn_ballot_w64(more), e = __builtin_amdgcn_ballot_w64(same);
    const uint64_t below = (1ull << lane) - 1;
    if (lane == 0) {
      sums[wave] = __popcll(m);
      sums[kChooseThreads / 64 + wave] = __popcll(e);
    }
    __syncthreads();
    int at = base + __popcll(m & below), rank = base_equal + __popcll(e & below);
    for (int w = 0; w < kChooseThreads / 64; ++w) {
      if (w < wave) {
        at += sums[w];
        rank += sums[kChooseThreads / 64 + w];
      }
      base += sums[w];
      base_equal += sums[kChooseThreads / 64 + w];
    }
    // Before this one: `at` larger ones, and of `rank` equal ones those that are taken.
    if (more || (same && rank < equal)) ch.out[at + (rank < equal ? rank : equal)] = ch.table[i];
    __syncthreads();
  }
}

template <int D>
hipError_t launch_bounds_dim(const BoundsParams& p, hipStream_t stream) {
  const bool shared = 1 << p.pg.page_shift >= kSharedPage;
  const int64_t most = (int64_t)p.batch * p.pg.pages_per_seq * p.kv_heads;
  const int64_t groups = shared ? most : (most + kBoundWaves - 1) / kBoundWaves;
  const dim3 grid((unsigned)(groups < kBoundGroups ? groups : kBoundGroups)), block(kBoundWaves * 64);
  if (shared) hipLaunchKernelGGL((key_bounds_kernel<D, true>), grid, block, p.batch * 4, stream, p);
  else hipLaunchKernelGGL((key_bounds_kernel<D, false>), grid, block, p.batch * 4, stream, p);
  return hipGetLastError();
}

template <int D, int AHEAD>
hipError_t launch_score_ahead(const SelectParams& p, hipStream_t stream) {
  const int at_once = AHEAD * (64 / (D / 8));
  const int64_t waves = (int64_t)p.batch * p.kv_heads * ((p.pg.pages_per_seq + at_once - 1) / at_once);
  const int batches = waves > kManyScoreWaves ? 4 : 1, per_group = at_once * batches * kScoreWaves;
  const dim3 grid((unsigned)((p.pg.pages_per_seq + per_group - 1) / per_group), p.kv_heads, p.batch);
  // The queries of four heads take half the registers of eight: with eight for a group of four 64.8 us for 50.6.
  if (p.group <= 4) hipLaunchKernelGGL((page_score_kernel<D, 4, AHEAD>), grid, dim3(kScoreWaves * 64), 0, stream, p, batches);
  else hipLaunchKernelGGL((page_score_kernel<D, 8, AHEAD>), grid, dim3(kScoreWaves * 64), 0, stream, p, batches);
  return hipGetLastError();
}

template <int D>
hipError_t launch_score_dim(const SelectParams& p, hipStream_t stream) {
  const int64_t alone = (int64_t)p.batch * p.kv_heads * ((p.pg.pages_per_seq + 64 / (D / 8) - 1) / (64 / (D / 8)));
  return alone <= kFewScoreWaves ? launch_score_ahead<D, 1>(p, stream) : launch_score_ahead<D, kScoreAhead>(p, stream);
}

}  // namespace

hipError_t launch_key_bounds(const BoundsParams& p, hipStream_t stream) {
  switch (p.head_dim) {
    case 64: return launch_bounds_dim<64>(p, stream);
    case 128: return launch_bounds_dim<128>(p, stream);
    case 256: return launch_bounds_dim<256>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_select_pages(const SelectParams& p, hipStream_t stream) {
  if (p.score) {
    hipError_t e;
    switch (p.head_dim) {
      case 64: e = launch_score_dim<64>(p, stream); break;
      case 128: e = launch_score_dim<128>(p, stream); break;
      case 256: e = launch_score_dim<256>(p, stream); break;
      default: return hipErrorInvalidValue;
    }
    if (e != hipSuccess) return e;
  }
  // As many threads as hold a row's scores, eight each; 1,024 throughout: 19.4, 52.7 and 24.7 us of the whole
  // sparse attention in place of 17.4, 51.1 and 23.5 (rows of 127, 1,026 and 2,050 pages).
  const dim3 grid(p.kv_heads, p.batch);
  const int pages = p.pg.pages_per_seq;
  if (pages <= 256 * kPerThread) hipLaunchKernelGGL(page_choose_kernel<256>, grid, dim3(256), 0, stream, p, (pages + 255) / 256);
  else if (pages <= 512 * kPerThread) hipLaunchKernelGGL(page_choose_kernel<512>, grid, dim3(512), 0, stream, p, (pages + 511) / 512);
  else if (pages <= 1024 * kPerThread) hipLaunchKernelGGL(page_choose_kernel<1024>, grid, dim3(1024), 0, stream, p, (pages + 1023) / 1024);
  else hipLaunchKernelGGL(page_choose_long_kernel, grid, dim3(kChooseThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace bt
