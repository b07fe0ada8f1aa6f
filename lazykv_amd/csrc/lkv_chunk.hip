// A chunk of new tokens of each sequence of a batch over its rows, which lie in pages or one after the other (lkv_chunk_attend).
//
// Token t of a sequence's n new ones, of len rows in all, attends rows 0 .. len - n + t:
//   s_i = scale * q . k_i,  m = max s_i,  out = sum exp(s_i - m) v_i / sum exp(s_i - m),  lse = m + ln sum exp(s_i - m),
// in one pass over the rows, base 2, as in the batch decode (lkv_shared.hip), whose rounding of weights and lift in float16 it has too. Scores, exponents, sums and partial
// results are float32; the weights' rounding to the model dtype shows beside the output's own: against 64 bits 0.0022 for 0.0017 where many rows have weight (bfloat16,
// 2,048 tokens behind 32,768), 0.00024 for 0.00021 (float16, 4,099 from nothing).
//
// The query rows of a KV head are its g heads of every token, x = t * g + j, so that a tile of them spans few tokens: the rows
// that some of them attend and others do not are few.
#include "lkv_attend.h"
#include "lkv_pages.h"

namespace {

using namespace lkv;

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;

struct ChunkArgs {
  const uint16_t* q;
  PagedRows rows;
  const int32_t* lengths;
  const int32_t* counts;
  void* out;
  float* lse;
  float2* part_ml;  // [parts][query rows of a sequence]: a part's maximum (base 2) and sum
  float* part_o;    // [parts][query rows of a sequence][d]
  int64_t q_stride[3];
  float scale2;  // scale * log2(e)
  int32_t n_seqs, n_q, n_kv, g, new_tokens, tokens, max_tokens, out_dtype;
  int32_t tiles;   // of a KV head's query rows
  int32_t unit;    // log2 of the rows that they are divided by
  int32_t share;   // parts that the sequences' rows would make, were they one sequence's; 0: each sequence in one, which writes the output
  int32_t most;    // parts that they make at most
};

// What a sequence has: rows in all, and the call's own among them.
struct Extent {
  int len, n;
};
__device__ __forceinline__ Extent extent_of(const ChunkArgs& a, int b) {
  const int64_t len = (int64_t)a.tokens + (a.lengths ? a.lengths[b] : 0);
  const int n = a.counts ? a.counts[b] : a.new_tokens;
  return {(int)(len < 0 ? 0 : (len > a.max_tokens ? a.max_tokens : len)), n < 0 ? 0 : (n > a.new_tokens ? a.new_tokens : n)};
}

// A lane's query row.
struct QueryRow {
  int64_t row;  // of out and lse; -1 for none
  int limit;    // rows that it attends
  const uint16_t* q;
};
__device__ __forceinline__ QueryRow query_row(const ChunkArgs& a, const Extent& e, int b, int h, int x) {
  const int t = x / a.g, j = h * a.g + (x - t * a.g);
  if (t >= a.new_tokens) return {-1, 0, nullptr};
  const int64_t row = ((int64_t)b * a.n_q + j) * a.new_tokens + t;
  const int limit = t < e.n ? max(e.len - e.n + t + 1, 0) : 0;
  return {row, limit, a.q + b * a.q_stride[0] + j * a.q_stride[1] + t * a.q_stride[2]};
}

// The division of the sequences' rows: by what there is of them on the device, so that all parts are about as long, however the sequences' lengths differ. Rows are counted in
// units; a part has as many as make `share` parts of all at the most, and each sequence at least one part, which writes the output where it is the only one.
// (Each sequence in as many parts as the next, four sequences of 1,643 to 16,475 rows under 64 tokens each took 82 us and now 66, a step of sixteen of up to
// 8,192 71 and now 57.)
__device__ __forceinline__ uint32_t units_of(const ChunkArgs& a, int b) { return b < a.n_seqs ? (uint32_t)(extent_of(a, b).len + (1 << a.unit) - 1) >> a.unit : 0; }
__device__ __forceinline__ uint32_t wave_total(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_inclusive_sum(x), 63); }
__device__ __forceinline__ uint32_t parts_of(const ChunkArgs& a, int b, uint32_t units) { return b < a.n_seqs ? max((units_of(a, b) + units - 1) / units, 1u) : 0; }
// Units of a part: at least those that make `share` parts of all, and so many that the sequences' parts, whose last ones are not whole, are no more than `most`.
// That ends: n_seqs is no more, and parts as long as the longest sequence are as many. The sum stays below 2^32 (plan_of).
__device__ __forceinline__ uint32_t part_units(const ChunkArgs& a) {
  uint32_t all = 0;
  for (int i = threadIdx.x & 63; i < a.n_seqs; i += 64) all += units_of(a, i);
  uint32_t units = max((wave_total(all) + a.share - 1) / a.share, 1u);
  if (a.most >= a.n_seqs + a.share - 1) return units;  // only the sequences' last parts are not whole
  for (;;) {
    uint32_t parts = 0;
    for (int i = 0; i < a.n_seqs; i += 64) parts += parts_of(a, i + (int)(threadIdx.x & 63), units);
    if (wave_total(parts) <= (uint32_t)a.most) return units;
    units += max(units >> 4, 1u);
  }
}
// Parts have places for their partial results where a sequence has several.
__device__ __forceinline__ uint32_t several(uint32_t parts) { return parts > 1 ? parts : 0; }

// What a workgroup does: rows begin .. begin + chunk of sequence b for a tile of KV head h's query rows.
struct Item {
  int b, h, tile, slot, begin, chunk;  // slot: the place of its partial results; -1: the only part of its sequence. b < 0: nothing
};
__device__ __forceinline__ Item item_of(const ChunkArgs& a) {
  int id = blockIdx.x;
  if (a.share == 0) {
    const int heads = a.n_seqs * a.n_kv, bh = id % heads;
    // The longest tiles first: the last ones of a sequence attend the most rows.
    return {bh / a.n_kv, bh % a.n_kv, a.tiles - 1 - id / heads, -1, 0, 1 << 30};
  }
  const int h = id % a.n_kv;
  id /= a.n_kv;
  const int tile = a.tiles - 1 - id % a.tiles;
  const uint32_t number = (uint32_t)(id / a.tiles), units = part_units(a);
  uint32_t before = 0, slots = 0;
  for (int i = 0; i < a.n_seqs; i += 64) {
    const uint32_t mine = parts_of(a, i + (int)(threadIdx.x & 63), units), up_to = before + wave_inclusive_sum(mine), slot = slots + wave_inclusive_sum(several(mine));
    const uint64_t behind = __ballot(up_to > number);
    if (behind) {
      const int lane = __builtin_ctzll(behind);
      const uint32_t parts = (uint32_t)__builtin_amdgcn_readlane((int)mine, lane), part = number + parts - (uint32_t)__builtin_amdgcn_readlane((int)up_to, lane);
      const int at = parts > 1 ? (int)((uint32_t)__builtin_amdgcn_readlane((int)slot, lane) - parts + part) : -1;
      const int chunk = (int)min((uint64_t)units << a.unit, (uint64_t)(1 << 30));
      return {i + lane, h, tile, at, (int)min((uint64_t)part * units << a.unit, (uint64_t)(1 << 30)), chunk};
    }
    before = (uint32_t)__builtin_amdgcn_readlane((int)up_to, 63);
    slots = (uint32_t)__builtin_amdgcn_readlane((int)slot, 63);
  }
  return {-1, h, tile, -1, 0, 0};
}

// Where a query row's partial result is.
__device__ __forceinline__ int64_t part_row(const ChunkArgs& a, int slot, int b, int64_t row) {
  const int64_t rows = (int64_t)a.n_q * a.new_tokens;
  return slot * rows + row - b * rows;
}

// Four channels of a row: a part's, or, where it is the only part, the output's.
template <int D>
__device__ __forceinline__ void store_part(const ChunkArgs& a, const Item& item, int64_t row, int channel, float l, f32x4 x) {
  if (item.slot >= 0) {
    if (l != 0.0f) *(f32x4*)(a.part_o + part_row(a, item.slot, item.b, row) * D + channel) = x;  // a part without weight is not read
    return;
  }
  x = l == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : x * (1.0f / l);
  if (a.out_dtype == LKV_F32) {
    store_four<LKV_F32>(a.out, row * D + channel, x);
  } else if (a.out_dtype == LKV_BF16) {
    store_four<LKV_BF16>(a.out, row * D + channel, x);
  } else {
    store_four<LKV_F16>(a.out, row * D + channel, x);
  }
}
__device__ __forceinline__ void store_sums(const ChunkArgs& a, const Item& item, int64_t row, float m, float l) {
  if (item.slot >= 0) {
    a.part_ml[part_row(a, item.slot, item.b, row)] = make_float2(m, l);
  } else {
    a.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

// Values that are not finite, in a tile whose rows not all attend: a weight of 0 would make NaN of them in rows that do not attend them. They are
// taken out of the product, and what they are is added by products of their own, with 1 for a row that attends and 0 for one that does not.
template <int DT> constexpr uint32_t kInfBits = DT == LKV_BF16 ? 0x7f80u : 0x7c00u;
template <int DT> constexpr uint32_t kOneBits = DT == LKV_BF16 ? 0x3f80u : 0x3c00u;
// For each half of a word: all ones where it satisfies.
template <int DT> __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t I = kInfBits<DT>;
  return ((w & I) == I ? 0xffffu : 0u) | ((w >> 16 & I) == I ? 0xffff0000u : 0u);
}
template <int DT> __device__ __forceinline__ uint32_t ones_where(uint32_t w, uint32_t value) {
  return ((w & 0xffffu) == value ? kOneBits<DT> : 0u) | (w >> 16 == value ? kOneBits<DT> << 16 : 0u);
}
template <int DT> __device__ __forceinline__ uint32_t ones_where_nan(uint32_t w) {
  constexpr uint32_t I = kInfBits<DT>;
  return ((w & 0x7fffu) > I ? kOneBits<DT> : 0u) | ((w >> 16 & 0x7fffu) > I ? kOneBits<DT> << 16 : 0u);
}
template <int DT> __device__ __forceinline__ bool any_not_finite(uint4 x) { return (not_finite<DT>(x.x) | not_finite<DT>(x.y) | not_finite<DT>(x.z) | not_finite<DT>(x.w)) != 0; }

template <int DT, class ACC, class MMA>
__device__ __forceinline__ void add_not_finite(uint4 v, uint4 attended, ACC& o, MMA mma) {
  const auto add = [&](uint4 ones, float what) {
    ACC zero;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(ACC) / 4); ++i) zero[i] = 0.0f;
    const ACC n = mma(ones, attended, zero);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(ACC) / 4); ++i) o[i] += n[i] > 0.0f ? what : 0.0f;
  };
  constexpr uint32_t I = kInfBits<DT>;
  add(make_uint4(ones_where<DT>(v.x, I), ones_where<DT>(v.y, I), ones_where<DT>(v.z, I), ones_where<DT>(v.w, I)), INFINITY);
  add(make_uint4(ones_where<DT>(v.x, I | 0x8000u), ones_where<DT>(v.y, I | 0x8000u), ones_where<DT>(v.z, I | 0x8000u), ones_where<DT>(v.w, I | 0x8000u)), -INFINITY);
  add(make_uint4(ones_where_nan<DT>(v.x), ones_where_nan<DT>(v.y), ones_where_nan<DT>(v.z), ones_where_nan<DT>(v.w)), NAN);
}

// ---- few rows: every wave on its own stream of tokens, straight from memory to registers -----------------
// Bound by memory, where there are enough rows: a token of each of sixteen sequences, 54,810 rows in all (8 heads, d 128, 224 MB), takes 40 us, 5.6 TB/s, and 6 more to join
// the parts, 76,414 61 with the join; one token over 131,072 rows 104 us, in 8 bits 75.

// The two halves of a wave's tile of 32 rows, each in one page; a half that is not there reads the other's rows, or the pool's first.
template <int D, bool MX> struct Halves {
  Stream s[2];
  bool there[2];
  // Rows 16 group .. of which `last` (0 .. 31) is the last one there is.
  __device__ __forceinline__ void find(const PagedRows& p, int b, int h, int group, int last) {
    Sixteen x[2];
    x[0] = sixteen_of<D>(p, b, h, group);
    x[1] = last >= 16 ? sixteen_of<D>(p, b, h, group + 1) : Sixteen{x[0].at + 16 * D, x[0].there};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t at = x[u].at - u * 16 * D;  // as if the tile lay together
      s[u] = {(const uint8_t*)p.rows.k + (MX ? at : 2 * at), (const uint8_t*)p.rows.v + (MX ? at : 2 * at), MX ? p.rows.k_scale + at / kMxGroup : nullptr,
              MX ? p.rows.v_scale + at / kMxGroup : nullptr};
      there[u] = x[u].there;
    }
  }
};

// A tile's scores made ready for the exponential (settle's work), where rows attend to different limits: left[n], tokens of the tile that this lane's
// row attends.
template <int DT, int D, int NR>
__device__ __forceinline__ void mask_scores(f32x4 (&sc)[NR][2], const int (&left)[NR], bool there0, bool there1) {
  const int quarter = (threadIdx.x & 48) / 4;
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x = (j < 4 ? 0 : 16) + (j & 3) + quarter < left[n] && (j < 4 ? there0 : there1) ? sc[n][j / 4][j & 3] : -INFINITY;
      keep_here(x);
      sc[n][j / 4][j & 3] = x;
    }
}

// Whether this lane's row attends its eight tokens of a tile, as the second product's operand.
template <int DT>
__device__ __forceinline__ uint4 attended(int left, bool there0, bool there1) {
  const int quarter = (threadIdx.x & 48) / 4;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = (i < 2 ? 0 : 16) + 2 * (i & 1) + quarter;
    const bool there = i < 2 ? there0 : there1;
    w[i] = (there && at < left ? kOneBits<DT> : 0u) | (there && at + 1 < left ? kOneBits<DT> << 16 : 0u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT, int D, bool MX, int NR>
__device__ __forceinline__ void attend_few(const ChunkArgs& a, int b, int h, const QueryRow (&row)[NR], int first, int step, int end, int whole,
                                           Result<D, NR>& r) {
  const int quarter = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    r.m[n] = -INFINITY;
    r.l[n] = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) r.o[n][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  if (first >= end) return;
  Reference ref[NR];
  uint4 qf[NR][D / 32];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    ref[n].reset();
#pragma unroll
    for (int i = 0; i < D / 32; ++i) qf[n][i] = row[n].row >= 0 ? *(const uint4*)(row[n].q + KeyRegs<D, MX>::channel(quarter, i)) : make_uint4(0, 0, 0, 0);
  }
  KeyRegs<D, MX> k;
  ValueRegs<D, MX> v;
  LaneOffsets<D, MX> at;
  Halves<D, MX> now, next_;
  at.set(min(kTile, end - first) - 1);
  now.find(a.rows, b, h, first >> 4, min(kTile, end - first) - 1);
  k.load(now.s, at);
  v.load(now.s, at);
  load_fence();
  for (int t = first; t < end; t += step) {
    const int next = t + step < end ? t + step : t;
    next_.find(a.rows, b, h, next >> 4, min(kTile, end - next) - 1);
    f32x4 sc[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) sc[n][0] = sc[n][1] = ref[n].negative;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 x = k.template operand<DT>(u, i);
#pragma unroll
        for (int n = 0; n < NR; ++n) sc[n][u] = Mat<DT>::mma(x, qf[n][i], sc[n][u]);
      }
    if (next + kTile > end) at.set(end - next - 1);
    k.load(next_.s, at);
    load_fence();
    const bool there0 = now.there[0], there1 = now.there[1], cut = t + kTile > whole || !there0 || !there1;
    int left[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) left[n] = row[n].limit - t;
    if (cut) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v.keep(j, t + (j < 4 ? 0 : 16) + 4 * quarter + (j & 3) < end && (j < 4 ? there0 : there1));
      mask_scores<DT, D, NR>(sc, left, there0, there1);
    }
    settle<DT, D, NR>(sc, kTile, a.scale2, ref, r);
    uint4 p[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) p[n] = weights<DT, NR>(sc[n], a.scale2, r.l[n]);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint32_t x[8];
      v.template widen<DT>(c, x);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const uint32_t pick = odd ? 0x07060302u : 0x05040100u;
        uint4 w = make_uint4(__builtin_amdgcn_perm(x[1], x[0], pick), __builtin_amdgcn_perm(x[3], x[2], pick), __builtin_amdgcn_perm(x[5], x[4], pick),
                             __builtin_amdgcn_perm(x[7], x[6], pick));
        if (cut && __any(any_not_finite<DT>(w))) {
#pragma unroll
          for (int n = 0; n < NR; ++n)
            add_not_finite<DT>(w, attended<DT>(left[n], there0, there1), r.o[n][2 * c + odd], [](uint4 m, uint4 q, f32x4 z) { return Mat<DT>::mma(m, q, z); });
          w = make_uint4(w.x & ~not_finite<DT>(w.x), w.y & ~not_finite<DT>(w.y), w.z & ~not_finite<DT>(w.z), w.w & ~not_finite<DT>(w.w));
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) r.o[n][2 * c + odd] = Mat<DT>::mma(w, p[n], r.o[n][2 * c + odd]);
      }
    }
    v.load(next_.s, at);
    load_fence();
    now = next_;
  }
  conclude<DT, D, NR>(a.scale2, ref, r);
}

// The results that the workgroup's waves have for the same rows, each from its own tokens, joined and stored: all write theirs to LDS, then
// each takes its share of the channels.
template <int D, int NR>
__device__ __forceinline__ void finish_few(const ChunkArgs& a, const Result<D, NR>& r, const QueryRow (&row)[NR], const Item& item, int wave, f32x4* lds) {
  constexpr int FOURS = D / 16;
  static_assert(FOURS % kWaves == 0, "every wave takes as many channels");
  const int lane = threadIdx.x & 63, quarter = lane >> 4;
  float2* const ml = (float2*)(lds + kWaves * NR * FOURS * 64);
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    ml[(wave * NR + n) * 64 + lane] = make_float2(r.m[n], r.l[n]);
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      int c;
      lds[((wave * NR + n) * FOURS + k) * 64 + lane] = four_of<D, false>(r.o[n], k, c);
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    float2 x[kWaves];
    float top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      x[i] = ml[(i * NR + n) * 64 + lane];
      top = fmaxf(top, x[i].x);
    }
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      x[i].x = join_factor(x[i].x, x[i].y, top);
      total += x[i].x * x[i].y;
    }
    if (row[n].row < 0) continue;
    if (row[n].limit == 0) total = 0.0f;
    if (wave == 0 && quarter == 0) store_sums(a, item, row[n].row, top, total);
#pragma unroll
    for (int j = 0; j < FOURS / kWaves; ++j) {
      const int k = j * kWaves + wave;
      f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kWaves; ++i) o += lds[((i * NR + n) * FOURS + k) * 64 + lane] * x[i].x;
      store_part<D>(a, item, row[n].row, channel_of<D, false>(k), total, o);
    }
  }
}

template <int DT, int D, bool MX, int NR>
__global__ __launch_bounds__(64 * kWaves, NR == 2 && D == 128 ? 1 : 2) void chunk_few_kernel(ChunkArgs a) {
  __shared__ f32x4 lds[kWaves * NR * 64 * (D + 8) / 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item item = item_of(a);
  const int b = item.b, h = item.h, tile = item.tile;
  if (b < 0) return;
  const Extent e = extent_of(a, b);
  QueryRow row[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) row[n] = query_row(a, e, b, h, (tile * NR + n) * 16 + (lane & 15));
  // Rows that the tile's first token attends, and its last one.
  const int t0 = tile * NR * 16 / a.g, t1 = min((tile * NR * 16 + NR * 16 - 1) / a.g, e.n - 1);
  const int whole = max(e.len - e.n + t0 + 1, 0), all = t1 < t0 ? 0 : max(e.len - e.n + t1 + 1, 0);
  const int begin = item.begin, end = (int)min((int64_t)begin + item.chunk, (int64_t)all);
  Result<D, NR> r;
  attend_few<DT, D, MX, NR>(a, b, h, row, begin + wave * kTile, kWaves * kTile, end, whole, r);
  finish_few<D, NR>(a, r, row, item, wave, lds);
}

// ---- many rows: keys and values through LDS --------------------------------------------------------
// A workgroup stages 64 tokens' keys and values in LDS, in the model dtype (8-bit rows are widened on the way), for four waves of 32 query rows
// each, on v_mfma_f32_32x32x16: S^T [32 tokens x 32 rows] = K Q^T, O^T [d x 32] += V^T P^T. A lane holds column lane % 32, of tokens
// 8 (i / 4) + 4 (lane / 32) + i % 4 in register i; the second product's k-th step of 16 tokens takes registers 8 k .. 8 k + 7 as they are. Pieces of 16
// bytes are swizzled by the row, so that both the keys' 32 rows and the values' transposed reads of four rows spread over all banks.
// Bound by issue: a product of 32 x 32 x 16 holds the matrix unit for 32 cycles, and the scores behind it cost, at 128 channels, some five vector operations and an exponential,
// 35 cycles, which two waves of a SIMD hide for two thirds (44.5 for both). 2,048 tokens behind 32,768 (32 heads on 8, d 128) take 1,110 to 1,170 us,
// 1.0 PFLOP/s, the matrix units busy for 47% of the cycles; at 64 channels the vector operations are as long as the products twice over: 4,099 tokens 100 us, 0.69 PFLOP/s.
template <int DT> struct Wide;
template <> struct Wide<LKV_BF16> {
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Wide<LKV_F16> {
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

constexpr int kStage = 64;  // tokens
template <int D> __device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? ((row & 3) << 2 | ((row >> 2) & 3)) : ((row & 2) << 1 | ((row >> 2) & 3));
}

// Where tokens are: a lane looks up sixteen of them, a wave 1,024 at once, and a stage's four are read from their lanes.
template <int D> struct Places {
  uint32_t lo, hi;  // of the lane's sixteen, in elements
  uint64_t there;   // a bit a lane
  // Sixteens first, first + 1, ...; in the place of those behind `last`, that one.
  __device__ __forceinline__ void find(const PagedRows& p, int b, int h, int first, int last) {
    const Sixteen x = sixteen_of<D, false>(p, b, h, min(first + (int)(threadIdx.x & 63), last));
    lo = (uint32_t)x.at;
    hi = (uint32_t)(x.at >> 32);
    there = __ballot(x.there);
  }
  __device__ __forceinline__ int64_t at(int lane) const {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, lane) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, lane));
  }
};

// A stage on its way to LDS. Behind the end, and in the place of rows that are not there, some other row lies: no weight goes to them, and what is not finite
// among their values is taken out where a tile is cut.
//
// Model dtype: straight from memory, a wave 1,024 bytes a load to as many of LDS, so that the swizzle is the loads': a lane takes the piece of its row that
// belongs where it writes.
template <int DT, int D, bool MX> struct StageLoad {
  static constexpr int BYTES = kStage * 2 * D;  // of keys, and of values, in LDS
  static constexpr int ROWS = 512 / D;          // of a load
  static constexpr int LOADS = kStage / ROWS / kWaves;
  uint32_t in;  // where a lane's piece is, from its sixteen's first row
  int row;      // its row in a sixteen
  __device__ __forceinline__ void begin() {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    row = (wave * ROWS + lane / (D / 8)) & 15;
    in = (uint32_t)(row * 2 * D + ((lane % (D / 8)) ^ swizzle<D>(row)) * 16);
  }
  // The stage whose four sixteens lanes first .. of `places` have looked up. CUT: `left` of its tokens are there, 64 or less.
  template <bool CUT> __device__ __forceinline__ void load(const PagedRows& p, const Places<D>& places, int first, int left, uint8_t* lds) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int top = (i * kWaves + wave) * ROWS, sixteen = top / 16;
      uint32_t from = in;
      if (CUT) from -= (uint32_t)(max(row - (left - 1 - min(sixteen, (left - 1) / 16) * 16), 0) * 2 * D);
      const int64_t at = 2 * places.at(first + sixteen);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)((const uint8_t*)p.rows.k + at + from),
                                       (__attribute__((address_space(3))) uint32_t*)(lds + top * 2 * D), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)((const uint8_t*)p.rows.v + at + from),
                                       (__attribute__((address_space(3))) uint32_t*)(lds + BYTES + top * 2 * D), 16, 0, 0);
    }
  }
  __device__ __forceinline__ void store(uint8_t*) const { __builtin_amdgcn_s_waitcnt(0xf70); }  // the loads have arrived: vmcnt(0)
};
// 8 bits: through registers, widened on the way.
template <int DT, int D> struct StageLoad<DT, D, true> {
  static constexpr int PIECES = D / 16;  // 16-byte pieces of a row
  static constexpr int LOADS = kStage * PIECES / (64 * kWaves);
  static constexpr int BYTES = kStage * 2 * D;
  u32x4 k[LOADS], v[LOADS];
  uint32_t ks[LOADS], vs[LOADS];
  __device__ __forceinline__ void begin() {}
  template <bool CUT> __device__ __forceinline__ void load(const PagedRows& p, const Places<D>& places, int first, int left, uint8_t*) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * 64 * kWaves + threadIdx.x, wave_x = i * 64 * kWaves + (threadIdx.x & ~63);
      const int sixteen = __builtin_amdgcn_readfirstlane(wave_x / PIECES / 16);  // a wave's rows of a load lie in one
      int row = x / PIECES & 15;
      if (CUT) row = min(row, left - 1 - min(sixteen, (left - 1) / 16) * 16);
      const int64_t at = places.at(first + sixteen);
      const uint32_t in = (uint32_t)(row * D + x % PIECES * 16);
      k[i] = *(const u32x4*)((const uint8_t*)p.rows.k + at + in);
      v[i] = *(const u32x4*)((const uint8_t*)p.rows.v + at + in);
      ks[i] = (p.rows.k_scale + at / kMxGroup)[in / kMxGroup];
      vs[i] = (p.rows.v_scale + at / kMxGroup)[in / kMxGroup];
    }
  }
  static __device__ __forceinline__ uint4 widen(uint32_t lo, uint32_t hi, uint32_t scale) {
    const float f = bits_to_float(scale << 23);
    return make_uint4(Mat<DT>::template widen<false>(lo, f), Mat<DT>::template widen<true>(lo, f), Mat<DT>::template widen<false>(hi, f),
                      Mat<DT>::template widen<true>(hi, f));
  }
  __device__ __forceinline__ void store(uint8_t* lds) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * 64 * kWaves + threadIdx.x, row = x / PIECES, piece = x % PIECES * 2, sw = swizzle<D>(row);
      uint8_t* to = lds + row * (2 * D);
      *(uint4*)(to + (piece ^ sw) * 16) = widen(k[i].x, k[i].y, ks[i]);
      *(uint4*)(to + ((piece + 1) ^ sw) * 16) = widen(k[i].z, k[i].w, ks[i]);
      to += BYTES;
      *(uint4*)(to + (piece ^ sw) * 16) = widen(v[i].x, v[i].y, vs[i]);
      *(uint4*)(to + ((piece + 1) ^ sw) * 16) = widen(v[i].z, v[i].w, vs[i]);
    }
  }
};

// A row's reference (see Reference in lkv_attend.h), here as the exponent's addend.
struct Level {
  float less;   // -reference in base 2 (+ the lift); 0 at first
  float limit;  // raw scores up to here stay; -inf until there is a reference
};

// The levels of rows whose largest score of some tokens is `top`; their sums follow.
template <int DT, int D>
__device__ __forceinline__ void settle_level(float top, float scale2, Level& level, float& l, f32x16 (&o)[D / 32]) {
  constexpr float lift = lift_of(DT, 2), slack = slack_of(DT, 2);
  if (!__any(top > level.limit)) return;
  const float up = pair_max<32>(top);
  const bool move = up > level.limit && up < INFINITY;
  const float less = lift - up * scale2;
  const float keep = !move ? 1.0f : level.limit == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(less - level.less);
  level.less = move ? less : level.less;
  level.limit = move ? up + slack / scale2 : level.limit;
  l *= keep;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) o[c] *= keep;
}
__device__ __forceinline__ float largest(const f32x16& s) {
  float top = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
  return top;
}
// Scores to weights: the second product's two operands, rounded as `weights` does it.
template <int DT>
__device__ __forceinline__ void wide_weights(const f32x16& s, float scale2, float less, float& l, uint4 (&p)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * k + i], scale2, less));
    l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    p[k] = make_uint4(Mat<DT>::pack(w[0], w[1]), Mat<DT>::pack(w[2], w[3]), Mat<DT>::pack(w[4], w[5]), Mat<DT>::pack(w[6], w[7]));
  }
}
template <int D>
__device__ __forceinline__ uint4 wide_value(const LdsPointer (&value_at)[2][D / 32], int c, int at) {
  const uint2 lo = read_transposed(value_at[0][c] + at), hi = read_transposed(value_at[1][c] + at);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// A stage that all the wave's rows attend: no branch but the level's, so that reads, products and exponentials of its two tiles mix.
// 64 channels: as long in exponentials as in products, and three waves a SIMD. A wave that has come to its exponentials goes before the others' products,
// which the matrix unit holds anyway: 4,099 tokens, 32 query heads on 8, 105.2 -> 98.9 us. 128 channels: twice the products, two waves; there the
// same costs 1130 -> 1140 us (2,048 tokens behind 32,768, 32 heads on 8), and products first gain 0.4%: left to the hardware.
template <int DT, int D>
__device__ __forceinline__ void whole_stage(const LdsPointer (&key_at)[D / 16], const LdsPointer (&value_at)[2][D / 32], int at, const uint4 (&qf)[D / 16], float scale2,
                                            Level& level, float& l, f32x16 (&o)[D / 32]) {
  constexpr bool FIRST = D == 64;
  if constexpr (FIRST) __builtin_amdgcn_s_setprio(0);
  f32x16 s[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s[u] = Wide<DT>::mma(read_piece(key_at[i] + at + u * 32 * 2 * D), qf[i], s[u]);
  if constexpr (FIRST) __builtin_amdgcn_s_setprio(1);
  settle_level<DT, D>(fmaxf(largest(s[0]), largest(s[1])), scale2, level, l, o);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint4 p[2];
    wide_weights<DT>(s[u], scale2, level.less, l, p);
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) o[c] = Wide<DT>::mma(wide_value<D>(value_at, c, at + (32 * u + 16 * k) * 2 * D), p[k], o[c]);
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(1);
  }
}

// 32 staged tokens that not all rows attend. left: those that this lane's row attends; there: of the two sixteens.
template <int DT, int D>
__device__ __forceinline__ void cut_tile(const LdsPointer (&key_at)[D / 16], const LdsPointer (&value_at)[2][D / 32], int at, const uint4 (&qf)[D / 16], int left, bool there0,
                                         bool there1, float scale2, Level& level, float& l, f32x16 (&o)[D / 32]) {
  const int half = (threadIdx.x & 32) >> 3;  // 4 (lane / 32)
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) s = Wide<DT>::mma(read_piece(key_at[i] + at), qf[i], s);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float x = 8 * (i / 4) + i % 4 + half < left && (i < 8 ? there0 : there1) ? s[i] : -INFINITY;
    keep_here(x);
    s[i] = x;
  }
  settle_level<DT, D>(largest(s), scale2, level, l, o);
  uint4 p[2];
  wide_weights<DT>(s, scale2, level.less, l, p);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint4 w[D / 32];
    bool odd = false;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      w[c] = wide_value<D>(value_at, c, at + 16 * k * 2 * D);
      odd |= any_not_finite<DT>(w[c]);
    }
    if (__any(odd)) {
      uint32_t ones[4];
      const bool there = k == 0 ? there0 : there1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int first = 16 * k + 8 * (i / 2) + 2 * (i & 1) + half;
        ones[i] = (there && first < left ? kOneBits<DT> : 0u) | (there && first + 1 < left ? kOneBits<DT> << 16 : 0u);
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        add_not_finite<DT>(w[c], make_uint4(ones[0], ones[1], ones[2], ones[3]), o[c], [](uint4 m, uint4 q, f32x16 z) { return Wide<DT>::mma(m, q, z); });
        w[c] = make_uint4(w[c].x & ~not_finite<DT>(w[c].x), w[c].y & ~not_finite<DT>(w[c].y), w[c].z & ~not_finite<DT>(w[c].z), w[c].w & ~not_finite<DT>(w[c].w));
      }
    }
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = Wide<DT>::mma(w[c], p[k], o[c]);
  }
}

template <int DT, int D, bool MX>
// Three waves a SIMD where the registers allow it without spills: 4,099 tokens, 32 query heads on 8, d 64, 118 us a launch and by two 131; 512 behind 8,192 78 and 76.
__global__ __launch_bounds__(64 * kWaves, D == 64 && !MX ? 3 : 2) void chunk_wide_kernel(ChunkArgs a) {
  using S = StageLoad<DT, D, MX>;
  constexpr int ROWS = 32 * kWaves;
  __shared__ f32x4 lds4[2 * 2 * S::BYTES / 16];
  uint8_t* const lds = (uint8_t*)lds4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item item = item_of(a);
  const int b = item.b, h = item.h, tile = item.tile;
  if (b < 0) return;
  const Extent e = extent_of(a, b);
  const int x0 = tile * ROWS + wave * 32;
  const QueryRow query = query_row(a, e, b, h, x0 + (lane & 31));
  const int limit = query.limit;
  const int past = e.len - e.n, begin = item.begin;
  const int last = min((tile * ROWS + ROWS - 1) / a.g, e.n - 1), wave_first = x0 / a.g, wave_last = min((x0 + 31) / a.g, e.n - 1);
  const int end = last < tile * ROWS / a.g ? 0 : (int)min((int64_t)begin + item.chunk, (int64_t)max(past + last + 1, 0));
  const int wave_end = wave_last < wave_first ? 0 : min(end, max(past + wave_last + 1, 0));
  Level level = {0.0f, -INFINITY};
  float l = 0.0f;
  f32x16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
  if (begin < end) {
    S stage;
    Places<D> places;
    const int last16 = (end - 1) >> 4;
    places.find(a.rows, b, h, begin >> 4, last16);
    stage.begin();
    stage.template load<true>(a.rows, places, 0, min(kStage, end - begin), lds);
    uint4 qf[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qf[i] = query.row >= 0 ? *(const uint4*)(query.q + 16 * i + (lane >> 5) * 8) : make_uint4(0, 0, 0, 0);
    LdsPointer key_at[D / 16], value_at[2][D / 32];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int r = lane & 31;
      key_at[i] = (LdsPointer)lds + r * (2 * D) + ((2 * i + (lane >> 5)) ^ swizzle<D>(r)) * 16;
      keep_here(key_at[i]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const int r = 8 * j + 4 * (lane >> 5) + ((lane & 15) >> 2);
        value_at[j][c] = (LdsPointer)lds + S::BYTES + r * (2 * D) + ((4 * c + ((lane & 16) >> 3) + ((lane & 2) >> 1)) ^ swizzle<D>(r)) * 16 + (lane & 1) * 8;
        keep_here(value_at[j][c]);
      }
    // Stages that all the workgroup's rows attend; then those that some do not, or that have rows which are not there.
    const int full = min(end, max(past + tile * ROWS / a.g + 1, 0));
    int t = begin, buffer = 0;
    uint64_t there = places.there;
    for (; t + kStage <= full && (there & 15) == 15; t += kStage) {
      stage.store(lds + buffer);
      __syncthreads();
      // The other buffer's readers came to this barrier after their last read of it.
      const int next = t + kStage;
      if (next < end) {
        const int at = (next - begin) >> 4 & 63;
        there >>= 4;
        if (at == 0) {
          places.find(a.rows, b, h, next >> 4, last16);
          there = places.there;
        }
        if (next + kStage <= end) {
          stage.template load<false>(a.rows, places, at, kStage, lds + (buffer ^ 2 * S::BYTES));
        } else {
          stage.template load<true>(a.rows, places, at, end - next, lds + (buffer ^ 2 * S::BYTES));
        }
      }
      load_fence();
      whole_stage<DT, D>(key_at, value_at, buffer, qf, a.scale2, level, l, o);
      buffer ^= 2 * S::BYTES;
    }
    for (; t < end; t += kStage) {
      stage.store(lds + buffer);
      __syncthreads();
      const int next = t + kStage;
      const uint32_t here = (uint32_t)there;
      if (next < end) {
        const int at = (next - begin) >> 4 & 63;
        there >>= 4;
        if (at == 0) {
          places.find(a.rows, b, h, next >> 4, last16);
          there = places.there;
        }
        stage.template load<true>(a.rows, places, at, min(kStage, end - next), lds + (buffer ^ 2 * S::BYTES));
      }
      load_fence();
      for (int sub = 0; sub < 2; ++sub) {
        const int now = t + 32 * sub;
        if (now >= wave_end) break;
        cut_tile<DT, D>(key_at, value_at, buffer + sub * 32 * 2 * D, qf, limit - now, here >> (2 * sub) & 1, here >> (2 * sub + 1) & 1, a.scale2, level, l, o);
      }
      buffer ^= 2 * S::BYTES;
    }
  }
  int x = x0 + (lane & 31);
  keep_here(x);  // worked out anew: held from the start it would cost registers
  const QueryRow row = query_row(a, e, b, h, x);
  constexpr float down = 1.0f / (float)(1 << (int)lift_of(DT, 2));
  l = row.limit == 0 ? 0.0f : pair_sum<32>(l) * down;
  if (row.row >= 0 && lane < 32) store_sums(a, item, row.row, level.limit == -INFINITY ? -INFINITY : lift_of(DT, 2) - level.less, l);
  // Through LDS to rows that lie together: a wave's own 32 rows, 16-byte pieces swizzled by the row. (Stored from where they are, 16 bytes a lane, a row's neighbours in
  // the other half of the lanes: 2,048 workgroups' parts took 45 us more than 512's.)
  constexpr int PIECES = D / 4;
  f32x4* const mine = lds4 + wave * 32 * PIECES;
  __syncthreads();  // what LDS held before is read no more
  const float f = item.slot >= 0 ? down : l == 0.0f ? 0.0f : down / l;
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 x = f32x4{o[c][4 * i], o[c][4 * i + 1], o[c][4 * i + 2], o[c][4 * i + 3]} * f;
      mine[(lane & 31) * PIECES + ((8 * c + 2 * i + (lane >> 5)) ^ (lane & (PIECES - 1) & 31))] = l == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : x;
    }
  const int lo = (int)(uint32_t)row.row, hi = (int)(row.row >> 32);
  __builtin_amdgcn_wave_barrier();
#pragma unroll 4
  for (int i = 0; i < 32 * PIECES / 64; ++i) {
    const int r = (i * 64 + lane) / PIECES, piece = lane % PIECES;
    const int64_t to = (int64_t)((uint64_t)(uint32_t)__shfl(hi, r) << 32 | (uint32_t)__shfl(lo, r));
    const float sum = __shfl(l, r);
    const f32x4 x = mine[r * PIECES + (piece ^ (r & (PIECES - 1)))];
    if (to < 0) continue;
    if (item.slot >= 0) {
      if (sum != 0.0f) *(f32x4*)(a.part_o + part_row(a, item.slot, b, to) * D + piece * 4) = x;  // a part without weight is not read
    } else if (a.out_dtype == LKV_F32) {
      store_four<LKV_F32>(a.out, to * D + piece * 4, x);
    } else if (a.out_dtype == LKV_BF16) {
      store_four<LKV_BF16>(a.out, to * D + piece * 4, x);
    } else {
      store_four<LKV_F16>(a.out, to * D + piece * 4, x);
    }
  }
}

// A query row's parts into one, a wave a row: d / 4 lanes take a part's channels, four each, and the others the next part's.
template <int D>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkArgs a, int64_t rows) {
  constexpr int C = D / 4, EACH = 64 / C;
  const int lane = threadIdx.x & 63, c = lane % C;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  // The sequence's parts, as the workgroups above divided its rows.
  const int64_t seq_rows = (int64_t)a.n_q * a.new_tokens;
  const int b = (int)(row / seq_rows);
  const uint32_t units = part_units(a);
  uint32_t first = 0, parts = 0;
  for (int i = 0; i <= b; i += 64) {
    const uint32_t mine = several(parts_of(a, i + lane, units)), before = wave_inclusive_sum(mine) - mine;
    if (b - i < 64) {
      first += (uint32_t)__builtin_amdgcn_readlane((int)before, b - i);
      parts = (uint32_t)__builtin_amdgcn_readlane((int)mine, b - i);
    } else {
      first += (uint32_t)__builtin_amdgcn_readlane((int)(before + mine), 63);
    }
  }
  const int n_parts = (int)parts;
  if (n_parts == 0) return;  // one part, which wrote the output
  const int64_t at = first * seq_rows + (row - b * seq_rows);
  const float2* ml = a.part_ml + at;
  const float* from = a.part_o + at * D + c * 4;
  float top = -INFINITY, total = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int p0 = 0; p0 < n_parts; p0 += 64) {
    const float2 mine = p0 + lane < n_parts ? ml[(p0 + lane) * seq_rows] : make_float2(-INFINITY, 0.0f);
    const float up = fmaxf(top, wave_max_f32(mine.x));
    const float keep = p0 == 0 ? 0.0f : join_factor(top, total, up), f = join_factor(mine.x, mine.y, up);
    top = up;
    total = total * keep + wave_sum_f32(mine.y == 0.0f ? 0.0f : f * mine.y);
    o *= keep;
    const int n = min(64, n_parts - p0);
    for (int p = 0; p < n; p += EACH) {
      const int mine_p = p + lane / C;
      const float w = __shfl(f, mine_p), s = __shfl(mine.y, mine_p);
      if (mine_p < n && s != 0.0f) o += *(const f32x4*)(from + (p0 + mine_p) * seq_rows * D) * w;
    }
  }
  if constexpr (EACH == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pair_sum<16>(o[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pair_sum<32>(o[i]);
  if (lane >= C) return;
  o = total == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * (1.0f / total);
  if (a.out_dtype == LKV_F32) {
    store_four<LKV_F32>(a.out, row * D + c * 4, o);
  } else if (a.out_dtype == LKV_BF16) {
    store_four<LKV_BF16>(a.out, row * D + c * 4, o);
  } else {
    store_four<LKV_F16>(a.out, row * D + c * 4, o);
  }
  if (lane == 0) a.lse[row] = total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a call is divided: see ChunkArgs. nr: tiles of 16 rows of a wave on its own stream, 0: through LDS.
struct Plan {
  int nr, tiles, unit, share, most;
  int slots;  // for partial results: a sequence of several parts has fewer than twice as many as its rows make whole ones
  int64_t blocks;
};

Plan plan_of(const lkv_chunk_desc* d) {
  Plan p = {};
  const int64_t rows = (int64_t)d->new_tokens * (d->n_q / d->n_kv);
  // Few rows from memory, more through LDS (8 heads, d 128): 16 over 32,768 rows 34.4 us, as a wave's two tiles 36.2, through LDS 44.2; 32 over 32,768 36.4 and
  // 44.8, over 4,096 18.2 and 20.4.
  p.nr = rows <= 16 ? 1 : rows <= 32 ? 2 : 0;
  p.tiles = ceil_div(rows, p.nr ? 16 * p.nr : 32 * kWaves);
  // Workgroups for about as many parts as run at once, two a CU, one where its registers or an even division allow no more; none shorter than 128 rows on average (one token over
  // 1,000: 11.4 us, by 256 12.5) or 256 through LDS (40 over 2,040: 22.5, by 128 23.7), and 512 rows are not divided (one token over 300: 9.4 and 11.0, sixteen sequences of 500 12.3 and
  // 15.5; over 700 divided 11.3 and 13.8).
  // One token over 131,072 rows (d 128): 104 us by 256, 116 by 512; 8 tokens (two tiles of 16 rows a wave, one workgroup a CU) over 16,419 26 and 33;
  // sixteen sequences of up to 8,192 71 and 57; 203 tokens over 32,971 199 and 152, by 768 164.
  // Of many parts a sequence, no more than that; of few, those that are not whole come on top. On top, sixteen sequences' steps cost 60.8 us for 57.3 and four questions
  // of 64 tokens 75.2 for 61.6; not on top, sixteen of 64 tokens (two parts each) 135.4 for 121.8. Undivided, a step of 64 sequences of 1,024 rows and one of
  // 65,536 among them cost 1,029 us for 105, 32 chunks of 128 tokens of the same kind 1,916 for 275; 64 and 100 of equal lengths 184.4 for 186.9 and 308.7 for 312.1.
  // More than 256 sequences are not divided: every workgroup goes through their lengths for its part, and a part more than a sequence each is looked for again. 257 and 300 of 1,024 rows a token
  // each 219 and 253 us, divided 227 and 259; 300 under 32 tokens each 300, divided 410. What that leaves: with one of 65,536 rows among them, a workgroup a head has it, 1,140 and
  // 1,157 us for 272 and 307, under 32 tokens 1,727 for 457.
  const int64_t units = (int64_t)d->n_kv * p.tiles, room = p.nr && (d->n_seqs == 1 || (p.nr == 2 && d->head_dim == 128)) ? 256 : 512;
  int64_t share = units > 0 ? room / units : 1;
  const int64_t longest = d->n_seqs * (int64_t)ceil_div(d->max_tokens, p.nr ? 128 : 256);
  share = share > longest ? longest : share;
  int64_t most = share >= (p.nr ? 2 : 4) * (int64_t)d->n_seqs ? share : d->n_seqs + share - 1;
  most = most > longest ? longest : most;
  const bool divided = share > 1 && d->max_tokens > 512 && most > d->n_seqs && d->n_seqs <= 256;
  p.unit = p.nr ? 7 : 6;  // a round of the workgroup
  if (d->n_seqs * (((int64_t)d->max_tokens >> p.unit) + 1) >= 1LL << 31) p.unit = 12;
  p.share = divided ? (int)share : 0;
  p.most = divided ? (int)most : 0;
  p.slots = divided ? (int)(most < 2 * share ? most : 2 * share) : 0;
  p.blocks = units * (divided ? most : d->n_seqs);
  return p;
}

size_t scratch_of(const lkv_chunk_desc* d, const Plan& p) {
  const size_t rows = (size_t)p.slots * d->n_q * d->new_tokens;
  return lkv_align_up(rows * sizeof(float2), 16) + rows * d->head_dim * sizeof(float);
}

template <int DT, int D, bool MX>
void launch(const Plan& p, dim3 grid, hipStream_t s, const ChunkArgs& a) {
  auto kernel = p.nr == 1 ? chunk_few_kernel<DT, D, MX, 1> : p.nr == 2 ? chunk_few_kernel<DT, D, MX, 2> : chunk_wide_kernel<DT, D, MX>;
  hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, s, a);
}

}  // namespace

int lkv_check_chunk(const lkv_chunk_desc* d) {
  LKV_CHECK_ARG(d, "NULL pointer");
  LKV_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "head_dim %d unsupported (64 or 128)", d->head_dim);
  LKV_CHECK_ARG(d->n_seqs >= 0 && d->n_kv > 0 && d->n_q > 0 && d->n_q % d->n_kv == 0 && d->new_tokens >= 0, "bad shape: %d sequences, %d query heads over %d, %d tokens",
                d->n_seqs, d->n_q, d->n_kv, d->new_tokens);
  LKV_CHECK_ARG((__int128)d->n_seqs * d->n_q * (d->new_tokens > 0 ? d->new_tokens : 1) <= (1 << 26), "%d x %d x %d query rows in one call", d->n_seqs, d->n_q, d->new_tokens);
  LKV_CHECK_ARG(d->scale > 0.0f && d->scale * lkv::kLog2e < INFINITY, "scale %g: positive and finite", (double)d->scale);
  LKV_CHECK_ARG(d->tokens >= 0 && d->max_tokens >= 0 && d->max_tokens <= (1 << 30), "bad extent: %d rows of at most %d", d->tokens, d->max_tokens);
  LKV_CHECK_ARG(((d->q_stride[0] | d->q_stride[1] | d->q_stride[2]) & 7) == 0, "strides must be multiples of 8 elements");
  return LKV_OK;
}

extern "C" size_t lkv_chunk_attend_workspace_bytes(const lkv_chunk_desc* desc) {
  if (lkv_check_chunk(desc)) return 0;
  return scratch_of(desc, plan_of(desc));
}

extern "C" int lkv_chunk_attend(uintptr_t stream, const lkv_chunk_desc* desc, const void* q, int q_dtype, const lkv_kv_rows* rows, const lkv_pages* pages,
                                const int32_t* lengths, const int32_t* counts, void* out, int out_dtype, float* lse, void* ws, size_t ws_bytes) {
  if (int rc = lkv_check_chunk(desc)) return rc;
  LKV_CHECK_ARG(q && out && lse, "NULL pointer");
  LKV_CHECK_ARG(q_dtype == LKV_F16 || q_dtype == LKV_BF16, "queries are float16 or bfloat16, got dtype %d", q_dtype);
  LKV_CHECK_ARG(lkv_is_model_dtype(out_dtype), "unsupported output dtype %d", out_dtype);
  LKV_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0, "queries and outputs must start on 16 bytes");
  ChunkArgs a = {};
  if (int rc = lkv_paged_rows(rows, pages, desc->n_seqs, q_dtype, desc->head_dim, a.rows)) return rc;
  LKV_CHECK_ARG(desc->max_tokens <= a.rows.capacity, "%d rows of a sequence over %d", desc->max_tokens, a.rows.capacity);
  const size_t need = lkv_chunk_attend_workspace_bytes(desc);
  LKV_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), "workspace of %zu bytes: %zu are needed", ws_bytes, need);
  LKV_CHECK_ARG(need == 0 || ((uintptr_t)ws & 15) == 0, "the workspace must start on 16 bytes");
  const int64_t n = (int64_t)desc->n_seqs * desc->n_q * desc->new_tokens;
  if (n == 0) return LKV_OK;
  const Plan p = plan_of(desc);
  LKV_CHECK_ARG(p.blocks < (1 << 24), "%lld workgroups in one call", (long long)p.blocks);
  a.q = (const uint16_t*)q;
  a.lengths = lengths;
  a.counts = counts;
  a.out = out;
  a.lse = lse;
  a.part_ml = (float2*)ws;
  a.part_o = (float*)((uint8_t*)ws + lkv_align_up((size_t)p.slots * desc->n_q * desc->new_tokens * sizeof(float2), 16));
  for (int i = 0; i < 3; ++i) a.q_stride[i] = desc->q_stride[i];
  a.scale2 = desc->scale * kLog2e;
  a.n_seqs = desc->n_seqs;
  a.n_q = desc->n_q;
  a.n_kv = desc->n_kv;
  a.g = desc->n_q / desc->n_kv;
  a.new_tokens = desc->new_tokens;
  a.tokens = desc->tokens;
  a.max_tokens = desc->max_tokens;
  a.out_dtype = out_dtype;
  a.tiles = p.tiles;
  a.unit = p.unit;
  a.share = p.share;
  a.most = p.most;
  const hipStream_t s = (hipStream_t)stream;
  const bool half = q_dtype == LKV_F16, wide = desc->head_dim == 128, mx = rows->dtype == LKV_MXFP8;
  const dim3 grid((unsigned)p.blocks);
  if (half) {
    wide ? (mx ? launch<LKV_F16, 128, true>(p, grid, s, a) : launch<LKV_F16, 128, false>(p, grid, s, a))
         : (mx ? launch<LKV_F16, 64, true>(p, grid, s, a) : launch<LKV_F16, 64, false>(p, grid, s, a));
  } else {
    wide ? (mx ? launch<LKV_BF16, 128, true>(p, grid, s, a) : launch<LKV_BF16, 128, false>(p, grid, s, a))
         : (mx ? launch<LKV_BF16, 64, true>(p, grid, s, a) : launch<LKV_BF16, 64, false>(p, grid, s, a));
  }
  LKV_CHECK_LAUNCH("chunk_attend");
  if (p.share) {
    hipLaunchKernelGGL((wide ? chunk_join_kernel<128> : chunk_join_kernel<64>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, s, a, n);
    LKV_CHECK_LAUNCH("chunk_attend (join)");
  }
  return LKV_OK;
}
