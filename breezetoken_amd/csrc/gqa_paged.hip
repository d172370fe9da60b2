// Decode attention over a paged bf16 KV cache for gfx950: one new token per
// sequence, keys 0 .. lens[b] - 1 found through the page table.
//
//   x_j = q . k_j * scale * log2e,  m = max_j x_j,  l = sum_j exp2(x_j - m)
//   out = sum_j exp2(x_j - m) v_j / l,  zeros for a sequence without keys
//
// A table entry outside [0, num_pages) holds no keys.
//
// Bound by the stream of K and V: 32 sequences of 256 to 32,768 tokens, H = 8, Hkv = 2,
// D = 256 (454 MB), take 71 us, 6.35 TB/s, and the combine 4.7; one of 131,072, H = 16, 44
// and 4.6; 24 of 1,800 to 3,000, H = 32, Hkv = 8, D = 128, 40 and 4.7.
//
// The batch's tiles (16 tokens each, never across a page) are numbered through, sequence
// after sequence, and every work-group of a kv head takes an equal run of them, whatever sequences it
// falls into: all CUs stream the same number of bytes for any mix of lengths,
// with no plan, no host lengths and no rounds of work-groups.  A run that covers
// a sequence writes its result; the parts of a sequence cut by a run's end go to
// the workspace as (lse, normalised partial) and the combine joins them.  The
// part of work-group w in sequence b has slot w + b: runs and sequences both
// advance in order, so slots are unique and a sequence's are consecutive.  Where the
// tables are short (paged_runs) a work-group takes a sequence, and nothing is joined.
//
// Within a work-group the waves take a run's tiles in turn, each with an online
// softmax of its own, merged through LDS where a sequence ends.  A wave's next
// tile -- K, V, and the page id of the one after -- is on its way while it works
// on the current one, also across the end of a sequence, so the merge and the
// next sequence's queries hide behind the stream.
//
// The MFMA takes K as it is and the query heads of the group as columns.  Scaled
// queries and probabilities enter as sums of three bf16 terms, which hold all 24 bits
// of them, in further columns (and, for 5 to 8 heads, a second MFMA).  Two terms, for 5
// to 8 heads where the output is rounded to bf16 (2^-8), leave 2^-16 (launch_mode).
#include "bt_common.h"
#include "bt_decode.h"
#include "bt_kernels.h"

namespace bt {

namespace {

constexpr int kWaves = 8;
constexpr float kLazy = 8.0f;  // log2-domain slack before the reference max moves: probabilities stay below 2^8

// Sum over the column groups of 16 / GMAX that hold the terms of one head: every
// column gets its head's sum.
template <int GMAX>
__device__ __forceinline__ float term_sum(float v) {
  v += dpp_f32<0x128>(v);  // row_ror:8
  if constexpr (GMAX == 4) v += dpp_f32<0x124>(v);  // row_ror:4
  return v;
}

// The 16-byte slot of a tile's row that holds chunk c is c ^ slot_of(row): linear in the
// row's bits, and without bank conflicts (measured) both for the operand reads of K, whose
// 16 bytes a lane the LDS serves in groups of lanes 0-3, 12-15, 20-23, 24-27 (and so on),
// and for the transposed reads of V (8 rows, a pair of chunks).
template <int D>
__device__ __forceinline__ constexpr int slot_of(int r) {
  return D == 64 ? r & 6 : (r & 7) * 2;
}

__device__ __forceinline__ int bcast(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// 64 sequences' lengths and the batch-wide number of their last tile + 1.
struct Window {
  int first;  // sequence of lane 0
  int start;  // tiles before it
  int len, ends;
  __device__ __forceinline__ void load(const PagedDecodeParams& p, int f, int s, int cap, int count = 64) {
    first = f;
    start = s;
    const int lane = threadIdx.x & 63;
    len = f + lane < p.batch && lane < count ? p.lens[f + lane] : 0;
    len = len < 0 ? 0 : (len > cap ? cap : len);
    ends = s + wave_scan((len + 15) >> 4);
  }
  // The lane whose sequence holds tile t (64: a later window).
  __device__ __forceinline__ int find(int t) const { return __popcll(__builtin_amdgcn_ballot_w64(ends <= t)); }
  __device__ __forceinline__ int begin(int lane) const { return lane ? bcast(ends, lane - 1) : start; }
};
constexpr int kKeptWindows = 8;  // in LDS: 512 sequences; further windows load their lengths again

// WHOLE: work-group w takes sequence w, numbered alone; two of them fit a CU below D =
// 256 (128 registers).  Runs have a CU each (paged_runs) and take 130 to 195.
template <int GMAX, int D, bool QBF16, int TERMS, bool WHOLE>
__global__ __launch_bounds__(kWaves * 64, WHOLE && D < 256 ? 4 : 2) void gqa_paged_kernel(PagedDecodeParams p) {
  constexpr int kThreads = kWaves * 64;
  constexpr int kSteps = D / 32;
  constexpr int kDTiles = D / 16;
  constexpr int kSlots = D / 8;
  constexpr int kRowBytes = D * 2;
  constexpr int kTileBytes = 16 * kRowBytes;
  constexpr int kLoads = kTileBytes / 1024;  // 1 KiB wave loads per K or V tile
  constexpr int kRowsPerLoad = 1024 / kRowBytes;
  constexpr int kGroups = 16 / GMAX;                  // column groups
  constexpr bool kSecond = TERMS > kGroups;           // the third term in an MFMA of its own
  constexpr int kMoStride = D + 4;
  static_assert(kSteps == kLoads && kSteps <= kWaves, "one wave per d-step builds Q^T");

  __shared__ __attribute__((aligned(1024))) unsigned char tiles_lds[kWaves * kTileBytes];
  __shared__ __attribute__((aligned(16))) float mlds[kWaves * GMAX * kMoStride];
  __shared__ __attribute__((aligned(16))) u32x4 qlds[(kSecond ? 2 : 1) * kSteps * 64];
  __shared__ float mstat[2 * kWaves * GMAX];
  __shared__ int wsum[64];
  __shared__ int2 kept[kKeptWindows * 64];  // len and ends, from the window's own start

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = (int)blockIdx.x % p.kv_heads, w = (int)blockIdx.x / p.kv_heads;
  const int G = p.group, head0 = kvh * G;
  const int cap = p.pg.pages_per_seq << p.pg.page_shift;

  // ---- the batch's tiles and this work-group's run ---------------------------
  const int windows = WHOLE ? 1 : (p.batch + 63) >> 6;  // at most 64
  Window win;  // of the tile looked at last
  int wends = 0, total;
  if (windows == 1) {
    win.load(p, WHOLE ? w : 0, 0, cap, WHOLE ? 1 : 64);
    total = bcast(win.ends, 63);
  } else {
    for (int i = wave; i < windows; i += kWaves) {
      win.load(p, 64 * i, 0, cap);
      if (lane == 63) wsum[i] = win.ends;
      if (i < kKeptWindows) kept[64 * i + lane] = int2{win.len, win.ends};
    }
    __syncthreads();
    wends = wave_scan(lane < windows ? wsum[lane] : 0);
    total = bcast(wends, 63);
    win.first = -1;
  }
  auto window = [&](int i) {
    const int start = i ? bcast(wends, i - 1) : 0;
    if (i < kKeptWindows) {
      const int2 x = kept[64 * i + lane];
      win.first = 64 * i;
      win.start = start;
      win.len = x.x;
      win.ends = start + x.y;
    } else {
      win.load(p, 64 * i, start, cap);
    }
  };
  // To the window that holds tile t < total.
  auto seek = [&](int t) {
    if (windows == 1) return;
    const int i = __popcll(__builtin_amdgcn_ballot_w64(wends <= t));
    if (win.first != 64 * i) window(i);
  };
  int runs = (total + kPagedTilesPerRun - 1) / kPagedTilesPerRun;
  runs = runs < 1 ? 1 : (runs < p.runs ? runs : p.runs);
  const int share = total ? (total + runs - 1) / runs : 1;
  const int t0 = WHOLE ? 0 : (w * share < total ? w * share : total);
  const int t1 = WHOLE || t0 + share > total ? total : t0 + share;

  // The last work-group of the first head, often an idle one, says where each
  // sequence's parts are: their number (1: the result is written) and first slot.
  if (!WHOLE && w == p.runs - 1 && kvh == 0) {
    for (int i = wave; i < windows; i += kWaves) {
      if (windows > 1) window(i);
      const int b = 64 * i + lane, n = (win.len + 15) >> 4;
      if (b < p.batch) {
        const int w0 = (win.ends - n) / share;
        p.part_base[b] = w0 + b;
        p.part_count[b] = n ? (win.ends - 1) / share - w0 + 1 : 0;
      }
    }
  }

  auto store_out = [&](int b, int h, int d, const float4& a) {
    const int64_t row = (int64_t)b * p.out_stride_seq + (int64_t)(head0 + h) * D + d;
    if (p.out_bf16) {
      const u32x2 pk = {f32x2_to_bf16x2_bits(a.x, a.y), f32x2_to_bf16x2_bits(a.z, a.w)};
      *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + row) = pk;
    } else {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + row) = a;
    }
  };
  if (WHOLE && total == 0) {  // no combine follows
    for (int item = threadIdx.x; item < G * (D / 4); item += kThreads)
      store_out(w, item / (D / 4), item % (D / 4) * 4, float4{0.f, 0.f, 0.f, 0.f});
  }
  if (t0 >= t1) return;

  // ---- columns: head col % GMAX, term col / GMAX -------------------------------
  const int col = lane & 15, kg = lane >> 4;
  const int col_head = col & (GMAX - 1), term = col / GMAX;
  // A value's terms as packed bf16: this lane's, and (second) the third one for the first columns.
  const uint32_t keep0 = term == 0 && col_head < G ? 0xffffffffu : 0u;
  const uint32_t keep1 = term == 1 && col_head < G ? 0xffffffffu : 0u;
  const uint32_t keep2 = !kSecond && TERMS == 3 && term == 2 && col_head < G ? 0xffffffffu : 0u;
  auto terms2 = [&](float a, float b, uint32_t& second) -> uint32_t {
    const uint32_t h = f32x2_to_bf16x2_bits(a, b);
    a -= __uint_as_float(h << 16);
    b -= __uint_as_float(h & 0xffff0000u);
    const uint32_t m = f32x2_to_bf16x2_bits(a, b);
    uint32_t r = (h & keep0) | (m & keep1);
    if constexpr (TERMS == 3) {
      const uint32_t l = f32x2_to_bf16x2_bits(a - __uint_as_float(m << 16), b - __uint_as_float(m & 0xffff0000u));
      if constexpr (kSecond) second = l & keep0;
      else r |= l & keep2;
    }
    return r;
  };

  // ---- K/V tiles --------------------------------------------------------------
  const uint32_t row_bytes = (uint32_t)(p.pg.stride_tok * 2);
  unsigned char* tile_lds = tiles_lds + wave * kTileBytes;
  // Load j of a tile fetches whole rows j * kRowsPerLoad + lane / kSlots; chunk c of row
  // r goes to slot c ^ slot_of(r).  The part of the slot that depends on j is a constant,
  // so an offset is one exclusive-or with it and one addition.
  constexpr int kHiRows = kRowsPerLoad;  // rows of one load: a power of two
  const uint32_t lane_slot = (uint32_t)((lane % kSlots) ^ slot_of<D>(lane / kSlots)) * 16;
  const uint32_t lane_row = (uint32_t)(lane / kSlots) * row_bytes;
  uint32_t load_base = lane_slot;
  auto offset = [&](int j) -> uint32_t { return (load_base ^ (uint32_t)(slot_of<D>(j * kHiRows) * 16)) + lane_row; };
  u32x4 kr[kSteps], vr[kLoads];
  __amdgpu_buffer_rsrc_t krs, vrs;
  auto issue_k = [&]() {
    asm volatile("" : "+v"(load_base));  // offsets are made where they are used: sixteen fewer registers through the loop
#pragma unroll
    for (int j = 0; j < kLoads; ++j) kr[j] = buf_load16(krs, offset(j), (uint32_t)(j * kRowsPerLoad) * row_bytes);
  };
  auto issue_v = [&]() {
    asm volatile("" : "+v"(load_base));
#pragma unroll
    for (int j = 0; j < kLoads; ++j) vr[j] = buf_load16(vrs, offset(j), (uint32_t)(j * kRowsPerLoad) * row_bytes);
  };
  // A tile to come: its page id (on its way), rows with keys, and first token in the page.
  struct Tile {
    int id, rows, token;
  };
  int seq_tile = 0, seq_end_tile = 0, seq_len = 0;  // of the sequence looked at last: tiles [seq_tile, seq_end_tile)
  const int32_t* seq_table = p.pg.table;
  auto look_up = [&](int t) -> Tile {
    Tile x{-1, 0, 0};
    if (t < t1) {
      if (t >= seq_end_tile) {
        seek(t);
        const int i = win.find(t);
        seq_tile = win.begin(i);
        seq_end_tile = bcast(win.ends, i);
        seq_len = bcast(win.len, i);
        seq_table = p.pg.table + (int64_t)(win.first + i) * p.pg.table_stride;
      }
      const int at = (t - seq_tile) * 16, left = seq_len - at;
      x.rows = left < 16 ? left : 16;
      x.token = at & ((1 << p.pg.page_shift) - 1);
      x.id = uniform_load(seq_table, at >> p.pg.page_shift);
    }
    return x;
  };
  // Points the tile's buffers at its page; returns the rows with keys.
  const uint16_t* k_head = p.k + (int64_t)kvh * p.pg.stride_head;
  const uint16_t* v_head = p.v + (int64_t)kvh * p.pg.stride_head;
  auto open = [&](const Tile& x) -> int {
    const bool ok = (uint32_t)x.id < (uint32_t)p.pg.num_pages;
    const int rows = ok ? x.rows : 0;
    const int64_t off = (int64_t)(ok ? x.id : 0) * p.pg.stride_page + (uint32_t)x.token * (row_bytes / 2);
    krs = make_rsrc(k_head + off, (uint32_t)rows * row_bytes);
    vrs = make_rsrc(v_head + off, (uint32_t)rows * row_bytes);
    return rows;
  };

  // ---- queries of a sequence: raw values, then the Q^T operand ------------------
  u32x4 qraw[2];
  auto load_q = [&](int b) {
    if (wave < kSteps) {
      const int64_t row = (int64_t)b * p.q_stride_seq + (int64_t)(head0 + (col_head < G ? col_head : 0)) * D + (wave * 4 + kg) * 8;
      if constexpr (QBF16) {
        qraw[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.q) + row);
      } else {
        qraw[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(p.q) + row);
        qraw[1] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(p.q) + row + 4);
      }
    }
  };
  auto build_q = [&]() {
    if (wave < kSteps) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (QBF16) {
          v[2 * i] = bf16_bits_to_f32(qraw[0][i] & 0xffffu);
          v[2 * i + 1] = bf16_bits_to_f32(qraw[0][i] >> 16);
        } else {
          v[i] = __uint_as_float(qraw[0][i]);
          v[4 + i] = __uint_as_float(qraw[1][i]);
        }
      }
      u32x4 a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t second = 0;
        a[i] = terms2(v[2 * i] * p.scale_log2, v[2 * i + 1] * p.scale_log2, second);
        b[i] = second;
      }
      qlds[wave * 64 + lane] = a;
      if constexpr (kSecond) qlds[(kSteps + wave) * 64 + lane] = b;
    }
  };

  // ---- first tile of this wave, and the id of its second -------------------------
  int t = t0 + wave;
  seek(t0);
  load_q(win.first + win.find(t0));
  Tile cur = look_up(t), next = look_up(t + kWaves);
  int rows = open(cur);
  issue_k();
  issue_v();

  const int i16 = lane & 15;
  const int row1 = 4 * kg + (i16 >> 2);  // V^T read: token row of this lane
  // LDS addresses of the operand reads of step / d-tile 0; those of the others differ in
  // bits of their own (rows are powers of two, slots are exclusive-ors), so they are made
  // by an exclusive-or where they are used and take no registers through the loop.
  const uint32_t tile_at = (uint32_t)(uintptr_t)(BT_LDS unsigned char*)tile_lds;
  uint32_t k_at = tile_at + col * kRowBytes + ((kg ^ slot_of<D>(col)) * 16);
  uint32_t v_at = tile_at + row1 * kRowBytes + ((((i16 & 3) >> 1) ^ slot_of<D>(row1)) * 16) + (i16 & 1) * 8;
  for (int s0 = t0; s0 < t1;) {
    // ---- one sequence's part: tiles [s0, s1) -------------------------------------
    seek(s0);
    const int lane_b = win.find(s0), b = win.first + lane_b;
    const int seq_begin = win.begin(lane_b), seq_end = bcast(win.ends, lane_b);
    const int s1 = seq_end < t1 ? seq_end : t1;
    build_q();
    // Also: every thread is done with the merge of the part before.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // The next sequence's queries, ahead of further tiles: loads complete in order, and asked for at
    // this one's end they would be there only when its first tile is, with nothing else on its way.
    if (!WHOLE && s1 < t1) {
      seek(s1);
      load_q(win.first + win.find(s1));
    }
    floatx4 oacc[kDTiles];
#pragma unroll
    for (int i = 0; i < kDTiles; ++i) oacc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;
    for (; t < s1; t += kWaves) {
      // The next tile's requests go out whether there is one or not (none: no rows, nothing is
      // read), so no branch parts the loads from their waits, which then are for K alone, or the
      // score MFMAs from the first use of their result: behind a branch hipcc 7.2 puts too few
      // wait states on the path that takes it, and scores were read before they were there.
      // S^T = K . Q^T, K through the wave's tile into the operand layout.
      floatx4 sacc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        *reinterpret_cast<BT_LDS u32x4*>((BT_LDS unsigned char*)tile_lds + j * 1024 + lane * 16) = kr[j];
      const int next_rows = open(next);
      next = look_up(t + 2 * kWaves);
      issue_k();
      u32x4 kop[kSteps];
      asm volatile("" : "+v"(k_at), "+v"(v_at));
#pragma unroll
      for (int st = 0; st < kSteps; ++st) kop[st] = *reinterpret_cast<const BT_LDS u32x4*>(k_at ^ (uint32_t)(st * 64));
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const u32x4 q = qlds[st * 64 + lane];
        sacc = mfma16(as_bf16x8(kop[st]), as_bf16x8(q), sacc);
        if constexpr (kSecond) sacc = mfma16(as_bf16x8(kop[st]), as_bf16x8(qlds[(kSteps + st) * 64 + lane]), sacc);
      }
      // V into the wave's tile behind K's reads (one wave's LDS operations stay in order).
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        *reinterpret_cast<BT_LDS u32x4*>((BT_LDS unsigned char*)tile_lds + j * 1024 + lane * 16) = vr[j];
      issue_v();
      // Terms summed, rows without a key masked, online softmax.
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = term_sum<GMAX>(sacc[j]);
        x[j] = kg * 4 + j < rows ? v : -INFINITY;
      }
      float tmax = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      tmax = rows16_fmaxf(tmax);
      tmax = halves_fmaxf(tmax);
      // The reference max moves only when a score exceeds it by 2^8, so O and l are
      // rescaled almost never; lse = log2(l) + m is exact for any reference.
      const bool move = tmax > m_run + kLazy;
      const float m_new = move ? tmax : m_run;
      const float alpha = move ? fast_exp2(m_run - m_new) : 1.f;  // 0 when m_run is -inf
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      float pr[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) pr[j] = fast_exp2(x[j] - m_use);
      m_run = m_new;
      l_run = l_run * alpha + ((pr[0] + pr[1]) + (pr[2] + pr[3]));
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
        for (int i = 0; i < kDTiles; ++i) oacc[i] *= alpha;
      }
      u32x2 pop, pop2 = {0u, 0u};
      {
        uint32_t s0_ = 0, s1_ = 0;
        pop = u32x2{terms2(pr[0], pr[1], s0_), terms2(pr[2], pr[3], s1_)};
        if constexpr (kSecond) pop2 = u32x2{s0_, s1_};
      }
      // O^T += V^T . P^T, V^T read transposed.
      u32x2 vop[kDTiles];
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) vop[dt] = lds_read_tr4(reinterpret_cast<const BT_LDS uint16_t*>(v_at ^ (uint32_t)(dt * 32)));
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) {
        oacc[dt] = mfma16k16(vop[dt], pop, oacc[dt]);
        if constexpr (kSecond) oacc[dt] = mfma16k16(vop[dt], pop2, oacc[dt]);
      }
      rows = next_rows;
    }

    // The last MFMAs' results, wherever the loop was left.
    asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) asm volatile("" : "+v"(oacc[dt]));
    // ---- the waves' parts, merged ------------------------------------------------
    l_run = halves_sum(rows16_sum(l_run));
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) oacc[dt][j] = term_sum<GMAX>(oacc[dt][j]);
      asm volatile("" : "+v"(oacc[dt]));  // the lane moves stay here, where every lane is active
    }
    float* mm = mstat;
    float* ml = mstat + kWaves * GMAX;
    if (col_head < G) {
      // Every column group holds the sums: group `term` stores d-tiles term, term + kGroups, ...
      float* dst = mlds + (wave * GMAX + col_head) * kMoStride + term * 16 + kg * 4;
#pragma unroll
      for (int i = 0; i < kDTiles / kGroups; ++i) {
        float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kGroups; ++c) {
          const floatx4 a = oacc[i * kGroups + c];
          if (c == 0 || term == c) v = float4{a[0], a[1], a[2], a[3]};
        }
        *reinterpret_cast<float4*>(dst + i * kGroups * 16) = v;
      }
      if (kg == 0 && term == 0) {
        mm[wave * GMAX + col_head] = m_run;
        ml[wave * GMAX + col_head] = l_run;
      }
    }
    // Orders LDS only: the next tiles' loads stay on their way.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // The waves dealt a tile: (s0 - t0) % 8 and the following ones, as many as tiles.
    auto merge = [&](auto nw) {
      constexpr int NW = decltype(nw)::value;
      const int w0 = s0 - t0;
      for (int item = threadIdx.x; item < G * (D / 4); item += kThreads) {
        const int h = item / (D / 4), d = item % (D / 4) * 4;
        float mw[NW], lw[NW];
        float4 ow[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const int at = ((w0 + i) & (kWaves - 1)) * GMAX + h;
          mw[i] = mm[at];
          lw[i] = ml[at];
          ow[i] = *reinterpret_cast<const float4*>(mlds + at * kMoStride + d);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NW; ++i) mx = fmaxf(mx, mw[i]);
        float lsum = 0.f;
        float4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const float e = fast_exp2(mw[i] - mx);
          const float sc = lw[i] == 0.f ? 0.f : e;  // no keys; a NaN sum stays one
          lsum += lw[i] * sc;
          acc.x += ow[i].x * sc; acc.y += ow[i].y * sc; acc.z += ow[i].z * sc; acc.w += ow[i].w * sc;
        }
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
        acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
        if (s0 == seq_begin && s1 == seq_end) {
          store_out(b, h, d, acc);
        } else {
          const int64_t row = (int64_t)(head0 + h) * (p.runs + p.batch) + w + b;
          *reinterpret_cast<float4*>(p.part + row * D + d) = acc;
          if (d == 0) p.lse[row] = lsum == 0.f ? -INFINITY : fast_log2(lsum) + mx;
        }
      }
    };
    if (s1 - s0 <= 2) merge(IntConst<2>{});
    else if (s1 - s0 <= 4) merge(IntConst<4>{});
    else merge(IntConst<kWaves>{});
    s0 = s1;
  }
}

template <int GMAX, int D, int TERMS, bool WHOLE>
hipError_t launch_terms(const PagedDecodeParams& p, hipStream_t stream) {
  const dim3 grid((WHOLE ? p.batch : p.runs) * p.kv_heads), block(kWaves * 64);
  if (p.q_bf16) hipLaunchKernelGGL((gqa_paged_kernel<GMAX, D, true, TERMS, WHOLE>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((gqa_paged_kernel<GMAX, D, false, TERMS, WHOLE>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// Two terms only where a third would take an MFMA of its own and the result is rounded to
// bf16: 300 of 100,000 results then round to the other side, 50 with three (and 60 in plain
// f32 torch operations).  us, two / three terms, bf16 out, 8 heads a kv head: one sequence
// of 131,072, D = 256 47.2 / 48.3; 16 of 4,000 28.3 / 29.5; one of 500, D = 128, whole 7.4 /
// 8.2; 512 of 500, D = 64 11.4 / 11.8.  Up to 4 heads (24 of 2,400, D = 128 42.2 / 42.5; 512
// of 500, D = 64 22.0 / 22.1) the columns are there.
template <int GMAX, int D, bool WHOLE>
hipError_t launch_mode(const PagedDecodeParams& p, hipStream_t stream) {
  if constexpr (GMAX > 4) {
    if (p.out_bf16) return launch_terms<GMAX, D, 2, WHOLE>(p, stream);
  }
  return launch_terms<GMAX, D, 3, WHOLE>(p, stream);
}

template <int GMAX, int D>
hipError_t launch_dim(const PagedDecodeParams& p, hipStream_t stream) {
  return p.runs ? launch_mode<GMAX, D, false>(p, stream) : launch_mode<GMAX, D, true>(p, stream);
}

}  // namespace

int paged_runs(int batch, int kv_heads, int head_dim, int64_t max_tokens, int num_cus) {
  const int64_t most = (int64_t)batch * ((max_tokens + 15) / 16);  // tiles of the largest call
  // Short tables: a work-group per sequence, which writes its result, and no combine.
  // us a graph node (issued one by one), whole sequences / runs, D = 256, Hkv = 2: one
  // sequence of 128 tokens 6.4 (9.6) / 8.8 (13.2), 256 7.6 (9.6) / 8.8 (13.3), 512 10.7
  // (10.6) / 8.8 (13.3); D = 128, Hkv = 8: one of 512 7.4 (9.7) / 7.7 (13.1), 1,024 10.9
  // (11.0) / 7.7 (13.2); D = 64, Hkv = 4: one of 512 5.8 (9.8) / 7.1 (13.1).
  if (max_tokens <= 512 && max_tokens * head_dim <= 65536) return 0;
  // Where sequences fill the chip, longer ones too: every run would end some of them.  us,
  // all full / lengths uniform / their logarithms uniform, whole sequences and then runs:
  // 128 of up to 1,024, D = 256, Hkv = 2 42 / 30 / 23, 48 / 36 / 28; 300 of up to 1,024, D =
  // 128, Hkv = 8 201 / 112 / 45, 215 / 120 / 59; 128 of up to 512, D = 64 13 / 10 / 8, 16 /
  // 18 / 18; 128 of up to 2,048, D = 256 82 / 52 / 43, 89 / 52 / 34 (the longest one counts).
  if (max_tokens <= 1024 && (int64_t)batch * kv_heads >= num_cus) return 0;
  // One work-group a CU: two (D = 128, 64) keep more requests on their way, and the HBM
  // serves them less well.  us, one / two: H = 32, Hkv = 8, D = 128, 32 x 8,000 tokens
  // 166 / 172, 24 x 3,000 53 / 55, one of 131,072 89 / 91; H = 16, Hkv = 2 26 / 34; D =
  // 64, Hkv = 4, 128 x 2,045 45.5 / 46.8.  (D = 256: two rounds 91, one 84.)
  int64_t runs = num_cus / kv_heads;
  const int64_t enough = (most + kPagedTilesPerRun - 1) / kPagedTilesPerRun;
  if (runs > enough) runs = enough;
  return runs < 1 ? 1 : (int)runs;
}

hipError_t launch_decode_paged(const PagedDecodeParams& p, int head_dim, hipStream_t stream) {
  const bool small = p.group <= 4;
  hipError_t e;
  switch (head_dim) {
    case 64: e = small ? launch_dim<4, 64>(p, stream) : launch_dim<8, 64>(p, stream); break;
    case 128: e = small ? launch_dim<4, 128>(p, stream) : launch_dim<8, 128>(p, stream); break;
    case 256: e = small ? launch_dim<4, 256>(p, stream) : launch_dim<8, 256>(p, stream); break;
    default: return hipErrorInvalidValue;
  }
  if (e != hipSuccess || p.runs == 0) return e;
  CombineParams c{};
  c.lse = p.lse;
  c.part = p.part;
  c.total_splits = p.runs + p.batch;
  c.split_base = p.part_base;
  c.split_count = p.part_count;
  c.skip_single = 1;
  c.out = p.out;
  c.out_bf16 = p.out_bf16;
  c.out_stride_seq = p.out_stride_seq;
  return launch_decode_combine(c, head_dim, p.heads, p.batch, stream);
}

}  // namespace bt
