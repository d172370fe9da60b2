// Attention of drafted tokens over a paged bf16 KV cache for gfx950: a sequence's
// drafts hang from its cached tokens as a tree, draft i in slot len + i.
//
//   x_ij = q_i . k_j * scale * log2e  over j < len and j - len in {i, its ancestors}
//   out_i = sum_j exp2(x_ij - m_i) v_j / l_i,  zeros for a draft that is not there
//
// A draft is there where its parent is -1 (the cached tokens) or an earlier draft that is
// there.  A table entry outside [0, num_pages) holds no keys.
//
// The rows of a kv head are its drafts times the heads of the group, up to 512, and share
// one read of K and V: bound by that stream for few rows, by the products for many.  Each
// wave takes 16 rows, four waves side by side a tile of 32 keys; row blocks of 64 run on one
// XCD, whose L2 has the tiles for all of them.  (One wave for 32 rows with wider products, or
// for two sets of 16, leaves one wave a SIMD and was slower by half.)  S^T = K Q^T
// leaves the scores of a row in four lanes, which then are, rounded, the operand of
// O^T += V^T P^T as they lie; V is read transposed from LDS.  f32 queries and the
// probabilities enter as sums of three bf16 terms, which hold all 24 bits of them.  The
// next tile's scores are worked out beside this one's softmax.
//
// The tiles of the batch are dealt out by the work-groups themselves, from the lengths, in
// parts of one sequence each, or in equal runs where sequences are many; parts are joined by
// a kernel behind this one.
//
// Measured, both kernels: 32 sequences of 256 to 32,768 tokens, 5 drafts, H = 8, Hkv = 2,
// D = 256, f32: 94 us, this kernel 91, 5.0 TB/s of cache where a large copy reaches 4.93 and
// the decode of one token 6.0.  24 of 1,800 to 3,000 tokens, 16 drafts, H = 32, Hkv = 8, D =
// 128, bf16: 63 and 55 us.  One of 32,768, 64 drafts, H = 16, Hkv = 2, D = 256, f32: 90 us, 1.16
// PFLOP/s of bf16 products (three for each of the formula's; a library's large product reaches
// 1.2 here).  One of 301, 8 drafts: 14 us, a chain of loads (arguments, length, table, tiles,
// parts) and of instructions fetched for the first time.
#include "bt_common.h"
#include "bt_decode.h"
#include "bt_kernels.h"

namespace bt {

namespace {

constexpr int kWaves = 4;
constexpr int kRows = 64;  // of a work-group at most
// A work-group takes a part of one sequence, or an equal run of the batch's tiles, which may hold the end of one
// sequence and the start of the next: its share is exact, but each of the two pays the way to the first product
// (up to 7 us).  Runs are taken where parts would not fit the places there are (fewer than two a sequence) and have
// more than so many tiles.  Part / run, us, H = 8, Hkv = 2, D = 256, 8 drafts: 4 sequences of 1,000 tokens 16.9 / 18.3,
// 32 of 1,000 30 / 34, 32 of 2,000 41 / 52, 32 of 256 to 32,768 102 / 108, 128 of 2,000 (two places each) 121 / 132;
// 300 of 100 to 3,000 (less than one) 196 / 158.
constexpr int kPartTiles = 8;
// Fewest tiles of a part: one while that takes a quarter of the places, then two, four where the tiles are more
// than the places, since parts are written and read again.  One / two, us: one of 301 tokens 14.1 / 15.4, 500 14.1 / 15.2,
// 2,000 15.8 / 16.2, 8,000 25.5 / 20.1.  Two / four: 4 of 1,000 16.9 / 18.5; 32 of 500 25.7 / 22.8, 128 of 100 28.3 / 21.4.
constexpr int kFewTiles = 2, kManyTiles = 4;
constexpr float kLazy = 8.0f;  // log2-domain slack before the reference max moves: probabilities stay below 2^8

// HBM -> LDS copy of 16 bytes per lane (lane l's bytes land at lds + 16 * l).
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, unsigned char* lds, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (BT_LDS void*)lds, 16, (int)voff, (int)soff, 0, 0);
}

// Waits until results of MFMAs can be read, where a branch lies between (hipcc 7.2 puts too few
// wait states behind one).
template <int N>
__device__ __forceinline__ void mfma_settle(floatx4 (&acc)[N]) {
  asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(acc[i]));
}

// Work-groups a CU, which wait for their tiles apart.  More, which D = 64 and 128 have room for, cut the
// sequences into more parts: three take 55.5 us where two take
// 54.1 (32 sequences of 256 to 32,768 tokens, D = 128; in runs across sequences 63 and 56).
constexpr int kGroups = 2;

// bf16 terms of a probability, also where the result is rounded to bf16: with two, 3,101 of the 1,572,864 results of 24
// sequences of 1,800 to 3,000 tokens (16 drafts, H = 32, Hkv = 8, D = 128) fall to the wrong side of that rounding, with
// three 560 (777 in plain f32 torch operations).  us, two / three: that case 52.6 / 53.3, 32 of 500 19.1 / 19.5, and where
// products are what counts, 64 drafts of 16 heads behind 32,768, bf16 queries, 64 / 73.
constexpr int kTerms = 3;

// QT: bf16 terms of a query (3: f32, 1: bf16 as it is).
template <int D, int QT>
__global__ __launch_bounds__(kWaves * 64, kGroups) void gqa_tree_kernel(TreeParams p) {
  constexpr int kSteps = D / 32;
  constexpr int kDT = D / 16;
  constexpr int kSlots = D / 8;
  constexpr int kRowBytes = 2 * D;
  constexpr int kTile = 32 * kRowBytes;
  constexpr int kRpl = 1024 / kRowBytes;         // rows of a 1 KiB wave load
  constexpr int kLoads = kTile / 1024 / kWaves;  // of K, and of V, per wave and tile
  // Two buffers of K tiles and two of V tiles, in turn.  Arrays of their own: the compiler
  // then tells copies into one from reads of another.
  constexpr int kBuf = 64 * D;
  __shared__ __attribute__((aligned(1024))) unsigned char ka[kBuf];
  __shared__ __attribute__((aligned(1024))) unsigned char va[kBuf];
  __shared__ __attribute__((aligned(1024))) unsigned char kb[kBuf];
  __shared__ __attribute__((aligned(1024))) unsigned char vb[kBuf];
  __shared__ int wsum[64];
  __shared__ int spoiled;  // a draft's value that is not finite was taken out of this part
  extern __shared__ int ends[];  // tiles up to and with each sequence

  const int lane = threadIdx.x & 63;
  const int wave = uniform((int)threadIdx.x >> 6);
  const int kg = lane >> 4, i16 = lane & 15;
  const int G = p.group, R = p.drafts * G;
  const int cap = p.pg.pages_per_seq << p.pg.page_shift;
  // Row blocks of one run and kv head lie 8 work-groups apart: on one XCD, whose L2 then has the tiles.
  const int blocks = p.row_blocks;
  const int pair = (int)(blockIdx.x / (8u * blocks)) * 8 + (int)(blockIdx.x & 7u), rb = (int)(blockIdx.x / 8u) % blocks;
  const int work_groups = (p.runs ? p.runs + p.batch : p.batch) * p.kv_heads;
  if (pair >= work_groups) return;
  const int kvh = pair % p.kv_heads, w = pair / p.kv_heads;

  auto tokens_of = [&](int len) {
    len = len < 0 ? 0 : (len > cap ? cap : len);
    return len + p.drafts < cap ? len + p.drafts : cap;
  };
  // ---- this work-group's run of the batch's tiles, or part of a sequence --------------
  const int windows = (p.batch + 63) >> 6;
  // Running sums over the sequences of their tiles, `most` as one, those of up to 64 in a register of their
  // lanes; returns the last.
  int held = 0;
  const int len_held = p.runs && windows == 1 && lane < p.batch ? p.lens[lane] : 0;
  auto sum_up = [&](int most) -> int {
    auto of = [&](int len) { return (uint32_t)(((tokens_of(len) + 31) >> 5) + most - 1) / (uint32_t)most; };
    if (windows == 1) {
      held = wave_scan(lane < p.batch ? (int)of(len_held) : 0);
      return __builtin_amdgcn_readlane(held, 63);
    }
    for (int i = wave; i < windows; i += kWaves) {
      const int b = 64 * i + lane;
      const int e = wave_scan(b < p.batch ? (int)of(p.lens[b]) : 0);
      if (b < p.batch) ends[b] = e;
      if (lane == 63) wsum[i] = e;
    }
    __syncthreads();
    const int wends = wave_scan(lane < windows ? wsum[lane] : 0);
    for (int i = wave; i < windows; i += kWaves) {
      const int before = i ? __builtin_amdgcn_readlane(wends, i - 1) : 0;
      if (64 * i + lane < p.batch) ends[64 * i + lane] += before;
    }
    __syncthreads();
    return __builtin_amdgcn_readlane(wends, 63);
  };
  auto sum_to = [&](int b) -> int {
    if (b < 0) return 0;
    return windows == 1 ? __builtin_amdgcn_readlane(held, b) : uniform(ends[b]);
  };
  // The sequence of number t among those summed up.
  auto find = [&](int t) -> int {
    if (windows == 1) return __popcll(__builtin_amdgcn_ballot_w64(lane < p.batch && held <= t));
    int at = 64 * lane + 63;
    at = at < p.batch ? at : p.batch - 1;
    const int i = __popcll(__builtin_amdgcn_ballot_w64(lane < windows && ends[at] <= t));
    at = 64 * i + lane;
    return uniform(64 * i + __popcll(__builtin_amdgcn_ballot_w64(at < p.batch && ends[at < p.batch ? at : p.batch - 1] <= t)));
  };
  auto len_of = [&](int b) -> int {
    const int x = p.runs && windows == 1 ? __builtin_amdgcn_readlane(len_held, b) : uniform_load(p.lens, b);
    return x < 0 ? 0 : (x > cap ? cap : x);
  };
  int t0 = 0, t1 = 1, share = 0;  // tiles of the run; share 0: not a run, the part [first, end) of sequence b
  int b = w, first = 0, end = 0, slot = w;
  bool whole = true;
  if (p.runs == 0) {
    end = (tokens_of(len_of(w)) + 31) >> 5;
  } else {
    int runs = 0, total = 0, parts = 0, most = 1;
    bool by_run = false;
    const bool fits = p.places >= 2 * p.batch;
#pragma unroll 1
    for (int pass = 0;; ++pass) {
      const int n = sum_up(most);
      if (pass == 0) {
        total = n;
        const int fewest = total >= p.places ? kManyTiles : total > p.places / 4 ? kFewTiles : 1;
        most = (total + p.places - 1) / p.places;
        most = most > fewest ? most : fewest;
        by_run = p.batch == 1 || (most > kPartTiles && !fits);
        if (by_run) {
          runs = (total + fewest - 1) / fewest;
          runs = runs < p.runs ? runs : p.runs;
          share = (total + runs - 1) / runs;
          break;
        }
      } else {
        // Parts of one sequence each, no more than there are places for at once.
        parts = n;
        if (parts <= p.places || !fits || pass == 8) break;
        most += (most >> 4) + 1;
      }
    }
    if (w >= (by_run ? runs : parts)) return;
    if (by_run) {
      t0 = w * share < total ? w * share : total;
      t1 = t0 + share < total ? t0 + share : total;
    } else {
      b = find(w);
      const int s0 = sum_to(b - 1), count = sum_to(b) - s0, tiles = (tokens_of(len_of(b)) + 31) >> 5;
      const int each = tiles / count, more = tiles - each * count, at = w - s0;  // `more` parts have a tile more
      first = at * each + (at < more ? at : more);
      end = first + each + (at < more ? 1 : 0);
      whole = count == 1;
    }
    // Where each sequence's parts are, for the combine: their number (1: the result is written) and first slot.
    if (w == (by_run ? runs : parts) - 1 && kvh == 0 && rb == 0) {
      for (int i = threadIdx.x; i < p.batch; i += kWaves * 64) {
        const int before = __shfl_up(held, 1);
        const int s0 = i == 0 ? 0 : windows == 1 ? before : ends[i - 1], s1 = windows == 1 ? held : ends[i];
        p.part_base[i] = by_run ? s0 / share + i : s0;
        p.part_count[i] = by_run ? (s1 - 1) / share - s0 / share + 1 : s1 - s0;
      }
    }
  }

  // ---- tiles ----------------------------------------------------------------------
  const uint32_t row_bytes = (uint32_t)(p.pg.stride_tok * 2);
  const uint16_t* k_head = p.k + (int64_t)kvh * p.pg.stride_head;
  const uint16_t* v_head = p.v + (int64_t)kvh * p.pg.stride_head;
  uint32_t load_base = (uint32_t)((lane % kSlots) ^ slot_of<D>(lane / kSlots)) * 16;
  const uint32_t lane_row = (uint32_t)(lane / kSlots) * row_bytes;
  struct Tile {
    int id0, id1;  // pages of its halves
    int at;        // first token
  };
  const int32_t* table = p.pg.table;
  int n = 0, len = 0;  // of the sequence at hand: tokens with the drafts, and without
  // Entries are read whether there is such a tile or not (the last one's then), so that they are on their
  // way before the row's length is there.
  auto look_up = [&](int tile, int end) -> Tile {
    Tile x{-1, -1, tile * 32};
    const int last = p.pg.pages_per_seq - 1, e0 = x.at >> p.pg.page_shift, e1 = (x.at + 16) >> p.pg.page_shift;
    const int id0 = uniform_load(table, e0 < last ? e0 : last), id1 = uniform_load(table, e1 < last ? e1 : last);
    x.id0 = tile < end ? id0 : -1;
    x.id1 = tile < end ? id1 : -1;
    return x;
  };
  // Copies a tile of K or V; every wave asks for as many loads whether there is a tile or not (none: no rows,
  // zeros), so that the number of requests behind those waited for is known.
  auto fetch = [&](const Tile& x, const uint16_t* head, unsigned char* dst) {
    asm volatile("" : "+v"(load_base));
    __amdgpu_buffer_rsrc_t rs;
    {
      const int i = wave * 2 >= kWaves, id = i ? x.id1 : x.id0, at = x.at + 16 * i, left = n - at;
      const bool ok = (uint32_t)id < (uint32_t)p.pg.num_pages && left > 0;
      const int rows = ok ? (left < 16 ? left : 16) : 0;
      const int64_t off = ok ? (int64_t)id * p.pg.stride_page + (int64_t)(at & ((1 << p.pg.page_shift) - 1)) * p.pg.stride_tok : 0;
      rs = make_rsrc(head + off, (uint32_t)rows * row_bytes);
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int at = wave * kLoads + j;  // whole eights of rows a wave
      dma16(rs, dst + at * 1024, (load_base ^ (uint32_t)(slot_of<D>(j * kRpl) * 16)) + lane_row, (uint32_t)((at * kRpl) & 15) * row_bytes);
    }
  };
  auto fetch_k = [&](const Tile& x, unsigned char* dst) { fetch(x, k_head, dst); };
  auto fetch_v = [&](const Tile& x, unsigned char* dst) { fetch(x, v_head, dst); };

  const int vrow = 4 * kg + (i16 >> 2);  // V^T read: token row of this lane, and 16 further on
  const uint32_t k_lane = (uint32_t)(i16 * kRowBytes + ((kg ^ slot_of<D>(i16)) * 16));
  const uint32_t v_lane = (uint32_t)(vrow * kRowBytes + ((((i16 & 3) >> 1) ^ slot_of<D>(vrow)) * 16) + (i16 & 1) * 8);

  for (int t = t0; t < t1;) {
    // ---- one sequence's part: its tiles [first, end) --------------------------------
    int next = t1;
    if (share) {
      b = find(t);
      const int seq0 = sum_to(b - 1), seq1 = sum_to(b);
      first = t - seq0;
      next = seq1 < t1 ? seq1 : t1;
      end = next - seq0;
      whole = first == 0 && next == seq1;
      slot = w + b;
    }
    len = len_of(b);
    n = tokens_of(len);
    table = p.pg.table + (int64_t)b * p.pg.table_stride;

    // Tiles of this step, the next and the one after it.
    Tile t0_ = look_up(first, end), t1_ = look_up(first + 1, end), t2_ = look_up(first + 2, end);
    // ---- this lane's row, a draft and a head: its queries, and the drafts' tree -------------
    const int r = rb * kRows + wave * 16 + i16;
    const int draft = r < R ? r / G : 0;
    int up = lane < p.drafts ? p.parents[(int64_t)b * p.drafts + lane] : -2;
    constexpr int kRaw = QT == 1 ? 1 : 2;
    u32x4 qraw[kSteps][kRaw];
    {
      const int64_t at = (int64_t)b * p.q_stride_seq + ((int64_t)draft * p.heads + kvh * G + (r < R ? r - draft * G : 0)) * D + kg * 8;
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
#pragma unroll
        for (int i = 0; i < kRaw; ++i)
          qraw[st][i] = QT == 1 ? *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.q) + at + st * 32)
                                : *reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(p.q) + at + st * 32 + i * 4);
    }
    if (t != t0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the tiles' places are free
    if (threadIdx.x == 0) spoiled = 0;
    asm volatile("" ::: "memory");  // the queries' loads stay ahead of the tiles', behind which they would wait
    fetch_k(t0_, ka);
    fetch_v(t0_, va);
    fetch_k(t1_, kb);

    // ---- ancestors: a draft per lane, paths doubled six times ------------------------
    uint32_t anc0, anc1;
    bool there;
    {
      if (up < -1 || up >= lane) up = -2;
      anc0 = lane < 32 ? 1u << lane : 0u;
      anc1 = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        const int from = up < 0 ? lane : up;
        const uint32_t a0 = (uint32_t)__shfl((int)anc0, from), a1 = (uint32_t)__shfl((int)anc1, from);
        const int u = __shfl(up, from);
        anc0 |= a0;
        anc1 |= a1;
        up = up < 0 ? up : u;
      }
      there = up == -1;
    }
    {
      const uint32_t a0 = (uint32_t)__shfl((int)anc0, draft), a1 = (uint32_t)__shfl((int)anc1, draft);
      there = __shfl((int)there, draft) != 0 && r < R;
      anc0 = a0;
      anc1 = a1;
    }
    const uint64_t anc = there ? ((uint64_t)anc1 << 32) | anc0 : 0;
    u32x4 qop[QT][kSteps];
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      if constexpr (QT == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qop[0][st][e] = (qraw[st][0][e] ^ (p.scale_log2 < 0.f ? 0x80008000u : 0u)) & (p.scale_log2 == 0.f ? 0u : ~0u);
      } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(qraw[st][e >> 2][e & 3]) * p.scale_log2;
#pragma unroll
        for (int term = 0; term < QT; ++term)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t h = f32x2_to_bf16x2_bits(v[2 * e], v[2 * e + 1]);
            qop[term][st][e] = h;
            v[2 * e] -= __uint_as_float(h << 16);
            v[2 * e + 1] -= __uint_as_float(h & 0xffff0000u);
          }
      }
    }

    // QT = 1: of the scores.  A negative one's sign is the queries', and for zero they are: a masked score is -inf.
    const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
    floatx4 oacc[kDT];
#pragma unroll
    for (int i = 0; i < kDT; ++i) oacc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    // Scores of a K tile: this lane's row, keys 16 * i + 4 * kg + j.
    struct Scores {
      floatx4 x[2];
    };
    // Of a tile's keys, those that this lane's row attends: cached tokens, its ancestors and itself.
    auto attended = [&](const Tile& x) -> uint32_t {
      auto half = [&](int id, int at) -> uint32_t {
        const int left = n - at;
        if ((uint32_t)id >= (uint32_t)p.pg.num_pages || left <= 0) return 0;
        return left < 16 ? (1u << left) - 1 : 0xffffu;
      };
      const uint32_t live = half(x.id0, x.at) | half(x.id1, x.at + 16) << 16;
      uint32_t mask = 0xffffffffu;
      const int d0 = len - x.at;  // the first draft's place in the tile
      if (d0 < 32) mask = d0 >= 0 ? ((1u << d0) - 1) | (uint32_t)(anc << d0) : (d0 > -64 ? (uint32_t)(anc >> -d0) : 0u);
      return mask & live;
    };
    float m_use = 0.f;  // m_run, 0 before the first key
    // Before a step's probabilities: keys that a row does not attend, and a row's reference where a score
    // exceeds it by 2^8 (which is rare, so that the scores' maximum is not followed across lanes, and O
    // and l are not rescaled, for nothing).
    auto settle = [&](Scores& s, const Tile& x) {
      if (x.at + 32 > len || (uint32_t)x.id0 >= (uint32_t)p.pg.num_pages || (uint32_t)x.id1 >= (uint32_t)p.pg.num_pages) {
        const uint32_t mask = attended(x) >> (4 * kg);
#pragma unroll
        for (int e = 0; e < 8; ++e) s.x[e >> 2][e & 3] = mask >> (16 * (e >> 2) + (e & 3)) & 1 ? s.x[e >> 2][e & 3] : -INFINITY;
      }
      float top = s.x[0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmax_nc(top, s.x[e >> 2][e & 3]);
      if constexpr (QT == 1) top *= scale;
      if (__builtin_amdgcn_ballot_w64(top > m_run + kLazy)) {
        top = halves_max(rows16_max(top));
        const bool move = top > m_run + kLazy;
        const float m_new = move ? top : m_run;
        const float alpha = move ? fast_exp2(m_run - m_new) : 1.f;  // 0 when m_run is -inf
        m_run = m_new;
        m_use = m_new == -INFINITY ? 0.f : m_new;
        l_run *= alpha;
        mfma_settle(oacc);
#pragma unroll
        for (int i = 0; i < kDT; ++i) oacc[i] *= alpha;
      }
    };
    // One step's work before its products: the probabilities' terms, in stages between the products of
    // the next tile's scores, which the matrix unit works on meanwhile (behind the last tile: of zeros;
    // a branch around them costs more).
    u32x4 pop[kTerms];
    auto advance = [&](const unsigned char* kt, const Scores& s) -> Scores {
      constexpr int kStages = 2 + kTerms;
      float v[8], sum = 0.f;
      auto stage = [&](int i) {
        if (i < 2) {
#pragma unroll
          for (int e = 4 * i; e < 4 * i + 4; ++e) {
            v[e] = fast_exp2(QT == 1 ? fmaf(s.x[e >> 2][e & 3], scale, -m_use) : s.x[e >> 2][e & 3] - m_use);
            sum += v[e];
          }
          if (i == 1) l_run += sum;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w2 = f32x2_to_bf16x2_bits(v[2 * e], v[2 * e + 1]);
            pop[i - 2][e] = w2;
            v[2 * e] -= __uint_as_float(w2 << 16);
            v[2 * e + 1] -= __uint_as_float(w2 & 0xffff0000u);
          }
          asm volatile("" : "+v"(pop[i - 2]));  // made here, not where it is used
        }
      };
      Scores out{{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}};
      {
        // Offsets are made where they are used, a hundred fewer registers through the loop.
        uint32_t base = k_lane;
        asm volatile("" : "+v"(base));
        const BT_LDS unsigned char* tile = (const BT_LDS unsigned char*)kt;
        auto read = [&](int st, int i) { return *reinterpret_cast<const BT_LDS u32x4*>(tile + (base ^ (uint32_t)(st * 64)) + i * 16 * kRowBytes); };
        // Operands are read kAhead steps before their products, no sooner: they would take the registers.
        constexpr int kAhead = 2;
        u32x4 kop[kAhead][2];
#pragma unroll
        for (int st = 0; st < kAhead; ++st)
#pragma unroll
          for (int i = 0; i < 2; ++i) kop[st][i] = read(st, i);
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
#pragma unroll
          for (int term = 0; term < QT; ++term)
#pragma unroll
            for (int i = 0; i < 2; ++i) out.x[i] = mfma16(as_bf16x8(kop[st % kAhead][i]), as_bf16x8(qop[term][st]), out.x[i]);
          if (st + kAhead < kSteps) {
#pragma unroll
            for (int i = 0; i < 2; ++i) kop[st % kAhead][i] = read(st + kAhead, i);
          }
#pragma unroll
          for (int i = 0; i < kStages; ++i)
            if (i * kSteps / kStages == st) stage(i);
#pragma unroll
          for (int i = 0; i < 2 * QT; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // vector work beside it
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      return out;
    };
    // The first tile's scores alone.
    auto scores = [&](const unsigned char* kt) -> Scores {
      Scores out{{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}};
      const BT_LDS unsigned char* tile = (const BT_LDS unsigned char*)kt;
      auto read = [&](int st, int i) { return *reinterpret_cast<const BT_LDS u32x4*>(tile + (k_lane ^ (uint32_t)(st * 64)) + i * 16 * kRowBytes); };
      constexpr int kAhead = 2;
      u32x4 kop[kAhead][2];
#pragma unroll
      for (int st = 0; st < kAhead; ++st)
#pragma unroll
        for (int i = 0; i < 2; ++i) kop[st][i] = read(st, i);
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
#pragma unroll
        for (int term = 0; term < QT; ++term)
#pragma unroll
          for (int i = 0; i < 2; ++i) out.x[i] = mfma16(as_bf16x8(kop[st % kAhead][i]), as_bf16x8(qop[term][st]), out.x[i]);
        if (st + kAhead < kSteps) {
#pragma unroll
          for (int i = 0; i < 2; ++i) kop[st % kAhead][i] = read(st + kAhead, i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      return out;
    };
    // O^T += V^T P^T.
    auto products = [&](const unsigned char* vt) {
      uint32_t base = v_lane;
      asm volatile("" : "+v"(base));
      const BT_LDS unsigned char* tile = (const BT_LDS unsigned char*)vt;
      auto read = [&](int dt) {
        const BT_LDS unsigned char* at = tile + (base ^ (uint32_t)(dt * 32));
        return lds_read_tr_pair(reinterpret_cast<const BT_LDS uint16_t*>(at), reinterpret_cast<const BT_LDS uint16_t*>(at + 16 * kRowBytes));
      };
      constexpr int kAhead = 4;
      bf16x8 vop[kAhead];
#pragma unroll
      for (int dt = 0; dt < kAhead; ++dt) vop[dt] = read(dt);
#pragma unroll
      for (int dt = 0; dt < kDT; dt += 2) {
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int i = 0; i < 2; ++i) oacc[dt + i] = mfma16(vop[(dt + i) % kAhead], as_bf16x8(pop[term]), oacc[dt + i]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (dt + i + kAhead < kDT) vop[(dt + i) % kAhead] = read(dt + i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // A draft's values must not reach rows that do not attend it, and zero times infinity is NaN: in the
    // tiles with drafts their values that are not finite are taken out, and put back where the result is written.
    auto has_drafts = [&](int tile) { return (tile + 1) * 32 > len; };
    auto take_out = [&](unsigned char* vt, const Tile& x) {
      for (int c = threadIdx.x * 16; c < kTile; c += kWaves * 1024) {
        const int token = x.at + c / kRowBytes;
        u32x4 v = *reinterpret_cast<const u32x4*>(vt + c);
        uint32_t odd = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = ((v[e] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((v[e] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
          odd |= bad;
          v[e] &= ~bad;
        }
        if (token >= len && token < n && odd) {
          *reinterpret_cast<u32x4*>(vt + c) = v;
          spoiled = 1;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };

    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool busy = rb * kRows + wave * 16 < R;  // a wave without rows only copies
    Scores s{};
    if (busy) s = scores(ka);
    // The next K and this V tile are there, the ones after them on their way.
    auto step = [&](int tile, unsigned char* k_next, unsigned char* k_free, unsigned char* v_now, unsigned char* v_free) {
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      fetch_k(t2_, k_free);
      fetch_v(t1_, v_free);
      if (has_drafts(tile)) take_out(v_now, t0_);
      if (busy) {
        settle(s, t0_);
        s = advance(k_next, s);
        // Of a SIMD's two waves the one that has nothing but products goes first: 101 us without for 95.5 (one sequence
        // of 32,768 tokens, 64 drafts of 16 heads).
        __builtin_amdgcn_s_setprio(1);
        products(v_now);
        __builtin_amdgcn_s_setprio(0);
      }
      t0_ = t1_;
      t1_ = t2_;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      // Scalar loads and LDS reads share a counter that the former complete out of order: asked for here,
      // where the next wait is for the tiles, and not ahead of LDS reads.
      t2_ = look_up(tile + 3, end);
    };
    for (int tile = first; tile < end; tile += 2) {
      step(tile, kb, ka, va, vb);
      if (tile + 1 >= end) break;
      step(tile + 1, ka, kb, vb, va);
    }

    // ---- rows written ---------------------------------------------------------------------
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy into LDS outlives the work-group
    mfma_settle(oacc);
    l_run = halves_sum(rows16_sum(l_run));
    const float l = there ? l_run : 0.f;  // 0: no keys, or no draft
    if (spoiled) {
      for (uint64_t todo = anc; todo; todo &= todo - 1) {
        const int token = len + __builtin_ctzll(todo);
        if (token < first * 32 || token >= end * 32 || token >= n) continue;
        const int page = table[token >> p.pg.page_shift];
        if ((uint32_t)page >= (uint32_t)p.pg.num_pages) continue;
        const uint16_t* at = v_head + (int64_t)page * p.pg.stride_page + (int64_t)(token & ((1 << p.pg.page_shift) - 1)) * p.pg.stride_tok + kg * 4;
        auto add = [](float a, uint32_t x) { return (x & 0x7f800000u) == 0x7f800000u ? a + __uint_as_float(x) : a; };
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) {
          const u32x2 v = *reinterpret_cast<const u32x2*>(at + dt * 16);
          oacc[dt][0] = add(oacc[dt][0], v[0] << 16);
          oacc[dt][1] = add(oacc[dt][1], v[0] & 0xffff0000u);
          oacc[dt][2] = add(oacc[dt][2], v[1] << 16);
          oacc[dt][3] = add(oacc[dt][3], v[1] & 0xffff0000u);
        }
      }
    }
    // Each lane writes four channels of its row at a time, 64 bytes a row: fewer steps than rows by way of LDS.
    if (r < R) {
      const int head = draft * p.heads + kvh * G + r - draft * G;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (l == 0.f) {
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) oacc[dt] = floatx4{0.f, 0.f, 0.f, 0.f};
      }
      if (!whole) {
        const int64_t at = (int64_t)head * (p.runs + p.batch) + slot;
        if (kg == 0) p.lse[at] = l == 0.f ? -INFINITY : fast_log2(l) + m_run;
        float* to = p.part + at * D + kg * 4;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) *reinterpret_cast<floatx4*>(to + dt * 16) = oacc[dt] * inv;
      } else if (p.out_bf16) {
        uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + (int64_t)b * p.out_stride_seq + (int64_t)head * D + kg * 4;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) {
          const floatx4 x = oacc[dt] * inv;
          *reinterpret_cast<u32x2*>(to + dt * 16) = u32x2{f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3])};
        }
      } else {
        float* to = reinterpret_cast<float*>(p.out) + (int64_t)b * p.out_stride_seq + (int64_t)head * D + kg * 4;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) *reinterpret_cast<floatx4*>(to + dt * 16) = oacc[dt] * inv;
      }
    }
    t = next;
  }
}

// Joins the parts of a row: a lane holds four values of it, S groups of lanes take its parts in turn, four on their
// way each, or eight; a work-group of T threads takes C columns of one row or more.
// Parts a group of lanes from which on eight are on their way.  The number of groups follows from the batch's average,
// and one long sequence may have nearly all parts.  us, four / eight / 16 throughout: one sequence of 60,000 tokens among
// 63 of 100 (H = 8, Hkv = 2, D = 256, 5 drafts) 65.4 / 53.0 / 50.1, among 63 of 1,000 69.0 / 60.4 / 59.4; 24 of 1,800 to
// 3,000 (H = 32, Hkv = 8, D = 128, 16 drafts) 52.6 / 52.5 / 53.6, for 16 take the registers of half the waves.
constexpr int kManyParts = 8;
template <int D, int S, int T, int C>
__global__ __launch_bounds__(T) void tree_join_kernel(TreeParams p) {
  constexpr int kLanes = C / 4, kRowsHere = T / kLanes / S;
  __shared__ float ms[S > 1 ? T / kLanes : 1], ls[S > 1 ? T / kLanes : 1];
  __shared__ float4 os[S > 1 ? T : 1];
  const int per_seq = p.drafts * p.heads, group = threadIdx.x / kLanes, part = group % S;
  const int64_t row = (int64_t)blockIdx.x * kRowsHere + group / S;
  const bool live = row < (int64_t)p.batch * per_seq;
  const int b = live ? (int)(row / per_seq) : 0, head = live ? (int)(row % per_seq) : 0, c = blockIdx.y * C + threadIdx.x % kLanes * 4;
  const int count = live ? p.part_count[b] : 1;
  if (S == 1 && count == 1) return;  // written
  const int64_t slot = (int64_t)head * (p.runs + p.batch) + p.part_base[b];
  float m = -INFINITY, l = 0.f;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  // Also with a weight of zero: a part's values that are not finite stay that in the result.
  auto add = [&](float top, float x, const float4& v) {
    const float wgt = fast_exp2(x - (top == -INFINITY ? 0.f : top));
    l += wgt;
    acc.x += wgt * v.x; acc.y += wgt * v.y; acc.z += wgt * v.z; acc.w += wgt * v.w;
  };
  auto take = [&](auto ahead) {
    constexpr int kAhead = decltype(ahead)::value;
    for (int s = part; s < count; s += kAhead * S) {
      float x[kAhead];
      float4 v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t at = slot + (s + i * S < count ? s + i * S : s);
        x[i] = p.lse[at];
        v[i] = *reinterpret_cast<const float4*>(p.part + at * D + c);
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        x[i] = s + i * S < count ? x[i] : -INFINITY;
        top = fmax_nc(top, x[i]);
      }
      const float old = fast_exp2(m - (top == -INFINITY ? 0.f : top));
      l *= old;
      acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (s + i * S < count) add(top, x[i], v[i]);
      m = top;
    }
  };
  if (count > kManyParts * S) take(IntConst<8>{});
  else if (count > 1) take(IntConst<4>{});
  // The groups' sums, the upper half's into the lower's until one is left.
#pragma unroll
  for (int half = S / 2; half; half >>= 1) {
    if (part >= half && part < 2 * half) {
      os[threadIdx.x] = acc;
      if (threadIdx.x % kLanes == 0) {
        ms[group] = m;
        ls[group] = l;
      }
    }
    __syncthreads();
    if (part < half) {
      const float mo = ms[group + half], lo = ls[group + half], top = fmax_nc(m, mo), use = top == -INFINITY ? 0.f : top;
      const float4 v = os[threadIdx.x + half * kLanes];
      // A sum that is not a number stays one, whatever its weight.
      const float a = l == 0.f ? 0.f : fast_exp2(m - use), o = lo == 0.f ? 0.f : fast_exp2(mo - use);
      l = l * a + lo * o;
      acc.x = acc.x * a + v.x * o; acc.y = acc.y * a + v.y * o; acc.z = acc.z * a + v.z * o; acc.w = acc.w * a + v.w * o;
      m = top;
    }
  }
  if (S > 1 && (part != 0 || count == 1)) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
  const int64_t at = (int64_t)b * p.out_stride_seq + (int64_t)head * D + c;
  if (p.out_bf16) {
    const u32x2 pk = {f32x2_to_bf16x2_bits(acc.x, acc.y), f32x2_to_bf16x2_bits(acc.z, acc.w)};
    *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + at) = pk;
  } else {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = acc;
  }
}

template <int D, int QT>
hipError_t launch_terms(TreeParams p, hipStream_t stream) {
  const int pairs = (p.runs ? p.runs + p.batch : p.batch) * p.kv_heads;
  const dim3 grid((unsigned)((pairs + 7) / 8 * 8 * p.row_blocks));
  const size_t lds = p.runs && p.batch > 64 ? (size_t)p.batch * 4 : 0;
  hipLaunchKernelGGL((gqa_tree_kernel<D, QT>), grid, dim3(kWaves * 64), lds, stream, p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const TreeParams& p, hipStream_t stream) {
  return p.q_bf16 ? launch_terms<D, 1>(p, stream) : launch_terms<D, 3>(p, stream);
}

}  // namespace

int tree_row_blocks(int rows) { return (rows + kRows - 1) / kRows; }

int tree_places(int kv_heads, int rows, int num_cus) {
  const int64_t places = (int64_t)num_cus * kGroups / ((int64_t)kv_heads * tree_row_blocks(rows));
  return places < 1 ? 1 : (int)places;
}

// Whole sequences, without a workspace and a join, where they are short, the longer the more of the chip their
// number fills.  Whole / in parts, us, D = 256, Hkv = 2, 8 drafts: 1 and 4 sequences of 100 tokens 13.8 / 14.9 and
// 14.0 / 15.5, 4 of 250 20.9 / 16.4; 32 of 250 and 500 22.0 / 22.0 and 30 / 23; 128 of 500, 1,000 and 2,000 36 / 46,
// 63 / 74 and 109 / 121 (not taken: one long row among short ones would be waited for).
int tree_runs(int batch, int kv_heads, int rows, int64_t max_tokens, int num_cus) {
  const int64_t groups = (int64_t)batch * kv_heads * tree_row_blocks(rows);
  if (max_tokens <= 128 || (max_tokens <= 320 && 4 * groups >= num_cus) || (max_tokens <= 1024 && groups >= num_cus)) return 0;
  const int64_t most = (int64_t)batch * ((max_tokens + 31) / 32);  // runs of one tile
  const int places = tree_places(kv_heads, rows, num_cus);
  return places < most ? places : (int)most;
}

hipError_t launch_decode_tree(const TreeParams& p, int head_dim, hipStream_t stream) {
  hipError_t e;
  switch (head_dim) {
    case 64: e = launch_dim<64>(p, stream); break;
    case 128: e = launch_dim<128>(p, stream); break;
    case 256: e = launch_dim<256>(p, stream); break;
    default: return hipErrorInvalidValue;
  }
  if (e != hipSuccess || p.runs == 0) return e;
  const int64_t rows = (int64_t)p.batch * p.drafts * p.heads;
  auto join = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    auto launch = [&](auto kernel, int threads, int groups, int columns) {
      const int per = threads / (columns / 4) / groups;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + per - 1) / per), D / columns), dim3(threads), 0, stream, p);
      return hipGetLastError();
    };
    // One, four or 32 groups of lanes a row, the last with a row's columns spread over work-groups.  All three, us of the
    // whole: 2.7 runs a sequence (24 sequences, D = 128) 64.5 / 69 / 171, 8 (32 ragged ones, D = 256) 106 / 101 / 121,
    // 32 (one, 1,024 rows) 100 / 97 / 113, 128 (four, one of them of 39,000 tokens, Hkv = 1, D = 128) 81 / 36 / 24, 256
    // (one of 8,000 tokens) 41 / 25 / 20.
    const int runs = p.runs > p.places / 4 && p.runs < p.places ? (p.runs + 1) / 2 : p.runs;  // of two tiles, not one
    if (runs <= 4 * p.batch) return launch(tree_join_kernel<D, 1, 256, D>, 256, 1, D);
    if (runs <= 32 * p.batch) return launch(tree_join_kernel<D, 4, 256, D>, 256, 4, D);
    return launch(tree_join_kernel<D, 32, 512, 64>, 512, 32, 64);
  };
  switch (head_dim) {
    case 64: return join(IntConst<64>{});
    case 128: return join(IntConst<128>{});
    default: return join(IntConst<256>{});
  }
}

}  // namespace bt
