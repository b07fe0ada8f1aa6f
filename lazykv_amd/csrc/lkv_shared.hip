// One decode token of each sequence of a batch: attention over a prefix that all sequences share and
// over each sequence's own rows (lkv_shared_decode). Rows are the model dtype's or 8-bit codes.
//
// Of query row r over keys k_t and values v_t, t in r's set:
//   s_t = scale * r . k_t,  m = max s_t,  out = sum exp(s_t - m) v_t / sum exp(s_t - m),
//   lse = m + ln sum exp(s_t - m),
// taken in one pass over the tokens, the sums so far scaled down whenever the maximum rises; in base 2,
// with log2(e) in the scale. Partial results of token ranges join by the same rule.
//
// The prefix's keys and values are read once for all sequences: the query rows of a KV head, g of each
// sequence, are the columns of the matrix products. A wave takes 32 tokens and 16 * NR rows at a time,
//   S^T [32 x rows] = K [32 x d] Q^T,   O^T [d x rows] += V^T [d x 32] P^T,
// on v_mfma_f32_16x16x32: the transposed forms leave a row's scores and its sums in the lanes of one
// column (lane % 16), so that the maximum, the weights and the rescaling are each lane's own, and a lane's
// weights are the second product's operand as they are. V^T takes its operand's order of tokens from
// there: a lane holds tokens 4q .. 4q+3 and 16+4q .. 16+4q+3 (q = lane / 16), loads d/16 neighbouring
// channels of each of these eight rows, 16 lanes a whole row, and pairs them by byte permutes.
//
// Weights are rounded to the model dtype for the second product (the matrix units' 16-bit form, 16 times
// float32's rate): with h = 2^-8 (bfloat16) or 2^-11 (float16) an output is off by at most h sum p_t |v_t| for it and, in float16, whose
// small numbers have fewer bits, by 2^-38 max |v| more for each token that is 2^-27 of the largest or less (2^-40 and 2^-29 with up to 16
// rows; `lift_of`). Where values cancel, that is more than the output's own rounding. Scores, maxima, sums of
// weights (unrounded) and outputs are float32.
//
// Three forms, by the rows that share a KV head's prefix (sequences times group):
//  - up to 16 or 32: a wave reads its own tokens from memory to registers; the workgroup's four waves, then the parts,
//    join. Bound by memory: one sequence over 131,072 tokens of 8 KV heads, d 128, takes 52.4 us in 8 bits (277 MB, 5.3 TB/s) and
//    93.5 in bfloat16 (537 MB, 5.7 TB/s), of which the join is 5. (64 rows a wave, one wave a SIMD: 16 sequences over
//    32,768 bfloat16 tokens 32.4 us where the next form takes 29.7, launches left out.)
//  - up to 64: through LDS, eight waves; 16 sequences over 32,768 bfloat16 tokens 35 us (134 MB; 6.1 TB/s in the loop, 5 us
//    before it, 3 after it and 5 for the join).
//  - more: through LDS, four waves, two workgroups a CU; 64 sequences over 32,768 tokens 60 us, over 131,072 180 (0.76
//    PFLOP/s; a library product of 8192^3 reaches 1.2).
// Own rows are read as in the first form, an item for each sequence and KV head, in the same launch.
#include "lkv_mx.h"

namespace {

constexpr int kWaves = 4;       // of a workgroup whose waves read streams of their own
constexpr int kTile = 32;       // tokens
// How far (in base 2) a score may lie above the reference that weights are taken from. A weight is then at most 2^slack:
// nothing to a 16-bit weight's precision or a float32 sum's. With more than 16 rows a reference that moves seldom is 2 to 8%
// of a call's time (8 sequences over 16,411 8-bit tokens, d 64: 12.6 -> 11.6 us); with fewer it costs nothing to hold it at the
// maximum, whose weight of 1 no rounding touches. Float16 pays for slack with the range of its weights (`lift_of`): 2 for 4 more powers of two
// than 6 leaves, at no time up to 32 rows, 64 sequences over 32,768 tokens, d 128, 71.9 -> 73.4 us, 32 over 65,536 8-bit tokens, d 64, 37.1 -> 39.5.
constexpr float slack_of(int dt, int row_tiles) { return row_tiles == 1 ? 0.0f : (dt == LKV_F16 ? 2.0f : 6.0f); }
// Float16 weights are held 2^lift larger than they are, the largest at 2^15, and the sums scaled back at the end (exactly): of float16's
// 30 powers of two above its subnormal numbers all but one then lie below the largest weight. Held as they are, weights below 2^-14 of it would
// lose bits and those below 2^-25 be lost from the products though not from the sum: one token 17.4 above the others in score, as the
// first of a prompt often is, would leave nothing of them. The lift is the exponential's addend, a multiplication's cost.
constexpr float lift_of(int dt, int row_tiles) { return dt == LKV_F16 ? 15.0f - slack_of(dt, row_tiles) : 0.0f; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT> struct Mat;
template <> struct Mat<LKV_BF16> {
  using V8 = bf16x8;
  static __device__ __forceinline__ f32x4 mma(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {  // round to nearest even
    bf16x2 v = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, v);
  }
  // Two codes of a word (the low or the high half) times their scale: exact.
  template <bool HI> static __device__ __forceinline__ uint32_t widen(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
  }
};
template <> struct Mat<LKV_F16> {
  using V8 = f16x8;
  static __device__ __forceinline__ f32x4 mma(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    f16x2 v = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(uint32_t, v);
  }
  template <bool HI> static __device__ __forceinline__ uint32_t widen(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI));
  }
};

struct SharedArgs {
  const uint16_t* q;
  lkv_kv_rows prefix, own;
  const int32_t* lengths;
  void* out;
  float* lse;
  float2* part_ml;  // [rows][parts]: a part's maximum (base 2) and sum
  float* part_o;    // [rows][parts][d]
  float scale2;     // scale * log2(e)
  int32_t n_seqs, n_q, n_kv, g, prefix_tokens, own_tokens, max_own, out_dtype;
  // The division of the work: the prefix in p_parts ranges of p_chunk tokens by row_tiles tiles of 16 * NR
  // rows, every sequence's own rows in o_parts ranges of o_chunk by g_tiles tiles of 16 heads.
  int32_t row_tiles, p_parts, p_chunk, p_groups, g_tiles, o_parts, o_chunk;
};

// Rows of sequence b: the lengths' sum, inside what was planned for.
__device__ __forceinline__ int own_length(const SharedArgs& a, int b) {
  const int64_t n = (int64_t)a.own_tokens + (a.lengths ? a.lengths[b] : 0);
  return (int)(n < 0 ? 0 : (n > a.max_own ? a.max_own : n));
}

// One source's rows of one head, as a wave reads them.
struct Stream {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
};

template <int D, bool MX>
__device__ __forceinline__ Stream stream_of(const lkv_kv_rows& r, int64_t seq, int64_t head) {
  const int64_t e = seq * r.seq_stride + head * r.head_stride;
  return {(const uint8_t*)r.k + (MX ? e : 2 * e), (const uint8_t*)r.v + (MX ? e : 2 * e), MX ? r.k_scale + e / kMxGroup : nullptr,
          MX ? r.v_scale + e / kMxGroup : nullptr};
}

// Keeps what a rarely taken branch computes in the branch: as selects it would be in every tile's way.
template <class T> __device__ __forceinline__ void keep_here(T& x) { asm volatile("" : "+v"(x)); }

// Where a lane's rows of a tile lie, in bytes from the tile's first: fixed but for a tile that the end cuts, whose
// tokens behind the end read the last one instead.
template <int D, bool MX> struct LaneOffsets {
  static constexpr int ROW = MX ? D : 2 * D;  // bytes
  uint32_t key[2];
  uint32_t value[8];
  bool cut;
  __device__ __forceinline__ void set(int last) {  // last: the last token of the tile that there is, 31 or less
    const int lane = threadIdx.x & 63, quarter = lane >> 4;
    cut = last < kTile - 1;
#pragma unroll
    for (int u = 0; u < 2; ++u) key[u] = (uint32_t)(min(16 * u + (lane & 15), last) * ROW + quarter * (MX ? D / 4 : 16));
#pragma unroll
    for (int j = 0; j < 8; ++j) value[j] = (uint32_t)(min((j < 4 ? 0 : 16) + 4 * quarter + (j & 3), last) * ROW + (lane & 15) * (ROW / 16));
  }
};

// Keys of a tile: two halves of 16 tokens, a lane token lane % 16 of each. Raw as loaded.
// Model dtype: channels 32 i + 8 q .. + 8 for the i-th product. 8 bits: channels (d/4) q .. + d/4, so that a
// lane's codes lie together under one scale; the i-th product takes the i-th eight of them.
template <int D, bool MX> struct KeyRegs;
template <int D> struct KeyRegs<D, false> {
  uint4 w[2][D / 32];
  __device__ __forceinline__ void load(const Stream& s, int64_t t, const LaneOffsets<D, false>& at) {
    const uint8_t* base = s.k + t * (2 * D);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) w[u][i] = *(const uint4*)(base + at.key[u] + i * 64);
  }
  template <int DT> __device__ __forceinline__ uint4 operand(int u, int i) const { return w[u][i]; }
  static __device__ __forceinline__ int channel(int q, int i) { return 32 * i + 8 * q; }
};
template <int D> struct KeyRegs<D, true> {
  uint4 w[2][D / 64];
  uint32_t scale[2];
  __device__ __forceinline__ void load(const Stream& s, int64_t t, const LaneOffsets<D, true>& at) {
    const uint8_t *base = s.k + t * D, *scales = s.ks + t * (D / kMxGroup);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) w[u][i] = *(const uint4*)(base + at.key[u] + i * 16);
      scale[u] = scales[at.key[u] / kMxGroup];
    }
  }
  template <int DT> __device__ __forceinline__ uint4 operand(int u, int i) const {
    const uint4& x = w[u][i / 2];
    const uint32_t lo = i & 1 ? x.z : x.x, hi = i & 1 ? x.w : x.y;
    const float f = lkv::bits_to_float(scale[u] << 23);  // the conversion takes a scale's exponent field alone
    return make_uint4(Mat<DT>::template widen<false>(lo, f), Mat<DT>::template widen<true>(lo, f), Mat<DT>::template widen<false>(hi, f),
                      Mat<DT>::template widen<true>(hi, f));
  }
  static __device__ __forceinline__ int channel(int q, int i) { return (D / 4) * q + 8 * i; }
};

// Values of a tile: eight tokens a lane, d/16 neighbouring channels of each.
template <int D, bool MX> struct ValueRegs;
template <int D> struct ValueRegs<D, false> {
  uint32_t w[8][D / 32];
  __device__ __forceinline__ void load(const Stream& s, int64_t t, const LaneOffsets<D, false>& at) {
    const uint8_t* base = s.v + t * (2 * D);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (D == 128) {
        const uint4 x = *(const uint4*)(base + at.value[j]);
        w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
      } else {
        const uint2 x = *(const uint2*)(base + at.value[j]);
        w[j][0] = x.x, w[j][1] = x.y;
      }
    }
  }
  __device__ __forceinline__ void keep(int j, bool live) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      w[j][c] = live ? w[j][c] : 0;
      keep_here(w[j][c]);
    }
  }
  template <int DT> __device__ __forceinline__ void widen(int c, uint32_t (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = w[j][c];
  }
};
// 8 bits: the scales of four tokens in a row come with one load.
template <int D> struct ValueRegs<D, true> {
  static constexpr int WORDS = D / 64;  // a token's scales: 4 or 2 bytes
  uint32_t w[8][WORDS];
  uint32_t scale[2][2 * WORDS];  // of tokens 4q.. and 16+4q..
  __device__ __forceinline__ void load(const Stream& s, int64_t t, const LaneOffsets<D, true>& at) {
    const uint8_t *base = s.v + t * D, *scales = s.vs + t * (D / kMxGroup);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (D == 128) {
        const uint2 x = *(const uint2*)(base + at.value[j]);
        w[j][0] = x.x, w[j][1] = x.y;
      } else {
        w[j][0] = *(const uint32_t*)(base + at.value[j]);
      }
    }
    if (!at.cut) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        __builtin_memcpy(scale[u], scales + (uint32_t)(((threadIdx.x & 48) / 4 + 16 * u) * (D / kMxGroup)), sizeof(scale[u]));
    } else {  // token by token: the four may not all be there
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t row = at.value[4 * u + j] / D * (D / kMxGroup);
          if constexpr (D == 128) {
            __builtin_memcpy(&scale[u][j], scales + row, 4);
          } else {
            uint16_t x;
            __builtin_memcpy(&x, scales + row, 2);
            scale[u][j / 2] = j & 1 ? scale[u][j / 2] | (uint32_t)x << 16 : x;
          }
        }
    }
  }
  __device__ __forceinline__ void keep(int j, bool live) {  // the scales are the last token's there
#pragma unroll
    for (int c = 0; c < WORDS; ++c) {
      w[j][c] = live ? w[j][c] : 0;
      keep_here(w[j][c]);
    }
  }
  template <int DT> __device__ __forceinline__ void widen(int c, uint32_t (&x)[8]) const {
    const int mine = (threadIdx.x & 15) * (D / 16) / kMxGroup * 8;  // this lane's scale in a token's
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t word = D == 128 ? scale[j / 4][j & 3] : scale[j / 4][(j & 3) / 2] >> (16 * (j & 1));
      const float f = lkv::bits_to_float((word >> mine) << 23 & 0x7f800000u);
      x[j] = c & 1 ? Mat<DT>::template widen<true>(w[j][c / 2], f) : Mat<DT>::template widen<false>(w[j][c / 2], f);
    }
  }
};

// A wave's running result for 16 * NR rows: lane l has rows l % 16 (+ 16 n) and channels (d/4)(l / 16) .. + d/4,
// channel (d/4) q + (d/16) i + e in o[n][e][i].
template <int D, int NR> struct Result {
  f32x4 o[NR][D / 16];
  float m[NR];  // the rows' reference, in base 2: the maximum of some tile, at most the slack below any score
  float l[NR];  // this lane's tokens' part of the sum
};

// Rows' reference: what their scores are taken from before the exponential. It need not be a row's maximum, only
// near it: it moves when a score is more than the slack above it, so that most tiles pass without a look at
// the other lanes. The products start from its negative, so that scores come out relative to it.
struct Reference {
  f32x4 negative;  // four times -reference, the products' first addend; 0 at first
  float limit;     // the slack in scores; -inf until there is a reference
  __device__ __forceinline__ void reset() {
    negative = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    limit = -INFINITY;
  }
  // The reference in base 2, as partial results carry it.
  __device__ __forceinline__ float level(float scale2) const { return limit == -INFINITY ? -INFINITY : -negative[0] * scale2; }
};

// A tile's scores, relative to the references, made ready for the exponential: tokens behind the end without weight
// (`left`: tokens that the tile has, if fewer than 32), a reference moved where it must be; l and o follow it.
template <int DT, int D, int NR>
__device__ __forceinline__ void settle(f32x4 (&sc)[NR][2], int left, float scale2, Reference (&ref)[NR], Result<D, NR>& r) {
  if (left < kTile) {
    int mine = left - (int)(threadIdx.x & 48) / 4;
    keep_here(mine);
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float x = (j < 4 ? 0 : 16) + (j & 3) < mine ? sc[n][j / 4][j & 3] : -INFINITY;
        keep_here(x);
        sc[n][j / 4][j & 3] = x;
      }
  }
  float top[NR];
  bool any = false;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const f32x4 x = sc[n][0], y = sc[n][1];
    top[n] = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
    any |= top[n] > ref[n].limit;
  }
  if (__any(any)) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if (!__any(top[n] > ref[n].limit)) continue;
      const float up = lkv::pair_max<32>(lkv::pair_max<16>(top[n]));
      const bool move = up > ref[n].limit && up < INFINITY;
      const float by = move ? up : 0.0f, keep = ref[n].limit == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-by * scale2);
      ref[n].negative -= by;
      ref[n].limit = move ? slack_of(DT, NR) / scale2 : ref[n].limit;
      r.l[n] *= keep;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) r.o[n][e] *= keep;
      sc[n][0] -= by;
      sc[n][1] -= by;
    }
  }
}

// Settled scores to weights, the second product's operand.
template <int DT, int NR>
__device__ __forceinline__ uint4 weights(const f32x4 (&sc)[2], float scale2, float& l) {
  float w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = sc[j / 4][j & 3];
    w[j] = __builtin_amdgcn_exp2f(lift_of(DT, NR) != 0.0f ? __builtin_fmaf(x, scale2, lift_of(DT, NR)) : x * scale2);
  }
  l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  return make_uint4(Mat<DT>::pack(w[0], w[1]), Mat<DT>::pack(w[2], w[3]), Mat<DT>::pack(w[4], w[5]), Mat<DT>::pack(w[6], w[7]));
}

// A range's sums and references as partial results carry them.
template <int DT, int D, int NR>
__device__ __forceinline__ void conclude(float scale2, const Reference (&ref)[NR], Result<D, NR>& r) {
  constexpr float down = 1.0f / (float)(1 << (int)lift_of(DT, NR));
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    r.l[n] = lkv::pair_sum<32>(lkv::pair_sum<16>(r.l[n])) * down;
    r.m[n] = ref[n].level(scale2);
    if constexpr (down != 1.0f) {
#pragma unroll
      for (int e = 0; e < D / 16; ++e) r.o[n][e] *= down;
    }
  }
}

// Loads stay on their side: moved down to where the next tile uses them, they would be waited for.
__device__ __forceinline__ void load_fence() { asm volatile("" ::: "memory"); }

// Tokens first, first + step, ... (tiles of 32) below end, for rows q[n].
template <int DT, int D, bool MX, int NR>
__device__ __forceinline__ void attend_range(const Stream& s, const uint16_t* const (&q)[NR], int first, int step, int end, float scale2,
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
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      qf[n][i] = q[n] ? *(const uint4*)(q[n] + KeyRegs<D, MX>::channel(quarter, i)) : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int n = 0; n < NR; ++n) ref[n].reset();
  KeyRegs<D, MX> k;
  ValueRegs<D, MX> v;
  LaneOffsets<D, MX> at;
  at.set(min(kTile, end - first) - 1);
  k.load(s, first, at);
  v.load(s, first, at);
  load_fence();
  for (int t = first; t < end; t += step) {
    f32x4 sc[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) sc[n][0] = sc[n][1] = ref[n].negative;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 a = k.template operand<DT>(u, i);
#pragma unroll
        for (int n = 0; n < NR; ++n) sc[n][u] = Mat<DT>::mma(a, qf[n][i], sc[n][u]);
      }
    // The next tile's keys are under way while this one's weights are computed, its values from the end of
    // this tile's products on. Behind the last tile that tile's own rows are read again.
    const int next = t + step < end ? t + step : t;
    if (next + kTile > end) at.set(end - next - 1);
    k.load(s, next, at);
    load_fence();
    if (t + kTile > end) {  // tokens behind the end: no value that a weight of 0 could turn to NaN
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v.keep(j, t + (j < 4 ? 0 : 16) + 4 * quarter + (j & 3) < end);
    }
    settle<DT, D, NR>(sc, end - t, scale2, ref, r);
    uint4 p[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) p[n] = weights<DT, NR>(sc[n], scale2, r.l[n]);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint32_t x[8];
      v.template widen<DT>(c, x);
      uint4 even, odd;
      even = make_uint4(__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
                        __builtin_amdgcn_perm(x[5], x[4], 0x05040100u), __builtin_amdgcn_perm(x[7], x[6], 0x05040100u));
      odd = make_uint4(__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u),
                       __builtin_amdgcn_perm(x[5], x[4], 0x07060302u), __builtin_amdgcn_perm(x[7], x[6], 0x07060302u));
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        r.o[n][2 * c] = Mat<DT>::mma(even, p[n], r.o[n][2 * c]);
        r.o[n][2 * c + 1] = Mat<DT>::mma(odd, p[n], r.o[n][2 * c + 1]);
      }
    }
    v.load(s, next, at);
    load_fence();
  }
  conclude<DT, D, NR>(scale2, ref, r);
}

__device__ __forceinline__ float join_factor(float m, float l, float top) {
  return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - top);
}

// Four neighbouring outputs.
template <int ODT>
__device__ __forceinline__ void store_four(void* out, int64_t at, f32x4 x) {
  if constexpr (ODT == LKV_F32) {
    *(f32x4*)((float*)out + at) = x;
  } else {
    *(uint2*)((uint16_t*)out + at) = make_uint2(Mat<ODT>::pack(x[0], x[1]), Mat<ODT>::pack(x[2], x[3]));
  }
}

// Where the k-th four channels of a lane's lie. TILED: channels 16 e + 4 q + i in o[e][i], else (d/4) q + (d/16) i + e.
template <int D, bool TILED>
__device__ __forceinline__ int channel_of(int k) {
  const int quarter = (threadIdx.x & 63) >> 4;
  return TILED ? 16 * k + 4 * quarter : (D / 4) * quarter + (D / 16) * (k / (D / 64)) + k % (D / 64) * 4;
}
template <int D, bool TILED>
__device__ __forceinline__ f32x4 four_of(const f32x4 (&o)[D / 16], int k, int& channel) {
  channel = channel_of<D, TILED>(k);
  if constexpr (TILED) {
    return o[k];
  } else {
    const int i = k / (D / 64), e = k % (D / 64) * 4;
    return f32x4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
  }
}

// Four channels of a row: a part's, or, where it is the only part, the output's.
template <int D>
__device__ __forceinline__ void store_part(const SharedArgs& a, int64_t row, int part, int channel, float l, f32x4 x) {
  const int parts = a.p_parts + a.o_parts;
  if (parts > 1) {
    *(f32x4*)(a.part_o + (row * parts + part) * D + channel) = x;
    return;
  }
  x *= l == 0.0f ? 0.0f : 1.0f / l;
  if (a.out_dtype == LKV_F32) {
    store_four<LKV_F32>(a.out, row * D + channel, x);
  } else if (a.out_dtype == LKV_BF16) {
    store_four<LKV_BF16>(a.out, row * D + channel, x);
  } else {
    store_four<LKV_F16>(a.out, row * D + channel, x);
  }
}
__device__ __forceinline__ void store_sums(const SharedArgs& a, int64_t row, int part, float m, float l) {
  const int parts = a.p_parts + a.o_parts;
  if (parts > 1) {
    a.part_ml[row * parts + part] = make_float2(m, l);
  } else {
    a.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * lkv::kLn2;
  }
}

// The end of a part: the results that GROUPS waves have for the same rows, each from its own tokens, joined and
// stored. All waves write theirs to LDS, then each takes its share of the channels. `group` and `slot`: which of
// the waves this is, and whose rows of `width` sets it has. row[n]: this lane's rows, -1 for none.
template <int D, int NR, int GROUPS, bool TILED>
__device__ __forceinline__ void finish(const SharedArgs& a, const Result<D, NR>& r, const int64_t (&row)[NR], int part, int group, int slot, int width,
                                       f32x4* lds) {
  constexpr int FOURS = D / 16;
  const int lane = threadIdx.x & 63, quarter = lane >> 4;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if (row[n] < 0) continue;
      if (quarter == 0) store_sums(a, row[n], part, r.m[n], r.l[n]);
#pragma unroll
      for (int k = 0; k < FOURS; ++k) {
        int c;
        const f32x4 x = four_of<D, TILED>(r.o[n], k, c);
        store_part<D>(a, row[n], part, c, r.l[n], x);
      }
    }
    return;
  } else {
    static_assert(FOURS % GROUPS == 0, "every wave takes as many channels");
    float2* const ml = (float2*)(lds + GROUPS * width * NR * FOURS * 64);
    __syncthreads();  // what LDS held before is read no more
    const int mine = (group * width + slot) * NR;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      ml[(mine + n) * 64 + lane] = make_float2(r.m[n], r.l[n]);
#pragma unroll
      for (int k = 0; k < FOURS; ++k) {
        int c;
        lds[((mine + n) * FOURS + k) * 64 + lane] = four_of<D, TILED>(r.o[n], k, c);
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float2 x[GROUPS];
      float top = -INFINITY, total = 0.0f;
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        x[i] = ml[((i * width + slot) * NR + n) * 64 + lane];
        top = fmaxf(top, x[i].x);
      }
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        x[i].x = join_factor(x[i].x, x[i].y, top);
        total += x[i].x * x[i].y;
      }
      if (group == 0 && quarter == 0 && row[n] >= 0) store_sums(a, row[n], part, top, total);
#pragma unroll
      for (int j = 0; j < FOURS / GROUPS; ++j) {
        const int k = j * GROUPS + group;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) o += lds[(((i * width + slot) * NR + n) * FOURS + k) * 64 + lane] * x[i].x;
        if (row[n] >= 0) store_part<D>(a, row[n], part, channel_of<D, TILED>(k), total, o);
      }
    }
  }
}
constexpr int finish_bytes(int d, int nr, int groups, int width) { return groups == 1 ? 0 : groups * width * nr * 64 * (d + 8); }

// A KV head's query row x of the prefix's: row x of all sequences', g a sequence; -1 behind the last.
__device__ __forceinline__ int64_t prefix_row(const SharedArgs& a, int h, int x) {
  const int b = x / a.g;
  return b < a.n_seqs ? (int64_t)b * a.n_q + h * a.g + (x - b * a.g) : -1;
}

// The `item`-th piece of own rows, by W waves; `lds`: the item's own. Every wave of the workgroup takes part in the
// barriers at the end.
template <int DT, int D, bool OMX, int W>
__device__ __forceinline__ void own_item(const SharedArgs& a, int64_t item, int wave, f32x4* lds) {
  const bool live = item < (int64_t)a.n_seqs * a.n_kv * a.g_tiles * a.o_parts;
  int id = live ? (int)item : 0;
  const int part = id % a.o_parts;
  id /= a.o_parts;
  const int tile = id % a.g_tiles;
  id /= a.g_tiles;
  const int h = id % a.n_kv, b = id / a.n_kv;
  const int j = tile * 16 + (threadIdx.x & 15);
  const int64_t row[1] = {live && j < a.g ? (int64_t)b * a.n_q + h * a.g + j : -1};
  const int t0 = part * a.o_chunk, end = live ? min(t0 + a.o_chunk, own_length(a, b)) : 0;
  const uint16_t* q[1] = {row[0] >= 0 ? a.q + row[0] * D : nullptr};
  Result<D, 1> r;
  attend_range<DT, D, OMX, 1>(stream_of<D, OMX>(a.own, b, h), q, t0 + wave * kTile, W * kTile, end, a.scale2, r);
  finish<D, 1, W, false>(a, r, row, a.p_parts + part, wave, 0, 1, lds);
}

// Few rows: every wave on its own stream of tokens, straight from memory to registers.
template <int DT, int D, bool PMX, bool OMX, int NR>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_decode_kernel(SharedArgs a) {
  __shared__ f32x4 lds[finish_bytes(D, NR, kWaves, 1) / 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = blockIdx.x, p_blocks = a.p_groups * 8 * a.row_tiles;
  if (id >= p_blocks) return own_item<DT, D, OMX, kWaves>(a, id - p_blocks, wave, lds);
  // Workgroups go round the 8 XCDs by their number: the row tiles of one head and token range sit on
  // one of them, one after the other, and find its keys and values in that L2.
  const int unit = (id / (8 * a.row_tiles)) * 8 + id % 8, tile = id / 8 % a.row_tiles;
  if (unit >= a.p_parts * a.n_kv) return;
  const int part = unit / a.n_kv, h = unit % a.n_kv;
  const uint16_t* q[NR];
  int64_t row[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    row[n] = prefix_row(a, h, (tile * NR + n) * 16 + (lane & 15));
    q[n] = row[n] >= 0 ? a.q + row[n] * D : nullptr;
  }
  const int t0 = part * a.p_chunk, end = min(t0 + a.p_chunk, a.prefix_tokens);
  Result<D, NR> r;
  attend_range<DT, D, PMX, NR>(stream_of<D, PMX>(a.prefix, 0, h), q, t0 + wave * kTile, kWaves * kTile, end, a.scale2, r);
  finish<D, NR, kWaves, false>(a, r, row, part, wave, 0, 1, lds);
}

// ---- many rows: the prefix through LDS --------------------------------------------------------------
// Each wave on its own stream of tokens reads all keys and values for its 32 rows alone: with many rows of
// a head, the reads from L2 bound that (10 TB/s over all row tiles). Here a workgroup stages its tokens' keys and
// values in LDS once, in the model dtype (8-bit rows are widened on the way, once for all rows), for WR waves
// across rows and WT across tokens. 16-byte pieces are swizzled by the row, so that the 16 tokens of an
// operand lie in different banks; the values' operands are read transposed.
//
// Up to 64 rows the reads from memory bound it: eight waves, two across the rows, each on its own tokens of a stage of
// 128. From there on the products and the exponentials do, and the card's power: under 256 rows of random values it
// runs at 1.75 GHz, 2.3 with zeros. There four waves take 32 rows each of the same tokens, one on each SIMD, and a
// second workgroup keeps each SIMD at work while the first one's waves meet at a barrier. (One workgroup of eight waves, two
// on a SIMD, came to each barrier one wave after the other: 87,000 cycles for 32,768 tokens under 256 rows, 50,000 with
// the barriers left out.)
template <int D, int WR, int W> struct Stage {
  static constexpr int THREADS = 64 * W, WT = W / WR, NR = 2;
  static constexpr int TOKENS = W == 8 ? 128 : 64;
  static constexpr int TILES = TOKENS / (kTile * WT);      // of a wave in a stage
  static constexpr int PIECES = D / 8;                     // 16-byte pieces of a row
  static constexpr int BYTES = TOKENS * 2 * D;             // of keys, and of values
  static __device__ __forceinline__ int swizzle(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
};

// What a thread holds of a stage on its way to LDS.
template <int DT, int D, bool MX, class S> struct StageRegs;
template <int DT, int D, class S> struct StageRegs<DT, D, false, S> {
  static constexpr int LOADS = S::TOKENS * S::PIECES / S::THREADS;  // 16-byte pieces of keys, and of values
  u32x4 k[LOADS], v[LOADS];
  // Tokens t0 .. of the stream; behind `end`, its last token.
  __device__ __forceinline__ void load(const Stream& s, int t0, int end) {
    const int last = min(S::TOKENS, end - t0) - 1;
    const uint8_t *kb = s.k + (int64_t)t0 * (2 * D), *vb = s.v + (int64_t)t0 * (2 * D);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * S::THREADS + threadIdx.x;
      const uint32_t at = (uint32_t)(min(x / S::PIECES, last) * (2 * D) + x % S::PIECES * 16);
      k[i] = *(const u32x4*)(kb + at);
      v[i] = *(const u32x4*)(vb + at);
    }
  }
  // Into LDS; values of tokens behind the end as zeros, which a weight of 0 leaves.
  __device__ __forceinline__ void store(uint8_t* lds, int live) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * S::THREADS + threadIdx.x, row = x / S::PIECES;
      uint8_t* to = lds + row * (2 * D) + (x % S::PIECES ^ S::swizzle(row)) * 16;
      const uint32_t keep = row < live ? ~0u : 0u;
      *(u32x4*)to = k[i];
      *(u32x4*)(to + S::BYTES) = v[i] & keep;
    }
  }
};
// 8 bits: 16 codes under one scale become two pieces.
template <int DT, int D, class S> struct StageRegs<DT, D, true, S> {
  static constexpr int LOADS = S::TOKENS * D / 16 / S::THREADS;
  static_assert(LOADS * S::THREADS * 16 == S::TOKENS * D, "whole loads of every thread");
  uint4 k[LOADS], v[LOADS];
  uint32_t ks[LOADS], vs[LOADS];
  __device__ __forceinline__ void load(const Stream& s, int t0, int end) {
    const int last = min(S::TOKENS, end - t0) - 1;
    const uint8_t *kb = s.k + (int64_t)t0 * D, *vb = s.v + (int64_t)t0 * D;
    const uint8_t *ksb = s.ks + (int64_t)t0 * (D / kMxGroup), *vsb = s.vs + (int64_t)t0 * (D / kMxGroup);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * S::THREADS + threadIdx.x;
      const uint32_t at = (uint32_t)(min(x / (D / 16), last) * D + x % (D / 16) * 16);
      k[i] = *(const uint4*)(kb + at);
      v[i] = *(const uint4*)(vb + at);
      ks[i] = ksb[at / kMxGroup];
      vs[i] = vsb[at / kMxGroup];
    }
  }
  static __device__ __forceinline__ uint4 widen(uint32_t lo, uint32_t hi, uint32_t scale) {
    const float f = lkv::bits_to_float(scale << 23);
    return make_uint4(Mat<DT>::template widen<false>(lo, f), Mat<DT>::template widen<true>(lo, f), Mat<DT>::template widen<false>(hi, f),
                      Mat<DT>::template widen<true>(hi, f));
  }
  __device__ __forceinline__ void store(uint8_t* lds, int live) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * S::THREADS + threadIdx.x, row = x / (D / 16), piece = x % (D / 16) * 2, sw = S::swizzle(row);
      uint8_t* to = lds + row * (2 * D);
      const uint32_t keep = row < live ? ~0u : 0u;  // a code of zero is zero under any scale that is written
      *(uint4*)(to + (piece ^ sw) * 16) = widen(k[i].x, k[i].y, ks[i]);
      *(uint4*)(to + ((piece + 1) ^ sw) * 16) = widen(k[i].z, k[i].w, ks[i]);
      to += S::BYTES;
      *(uint4*)(to + (piece ^ sw) * 16) = widen(v[i].x & keep, v[i].y & keep, vs[i]);
      *(uint4*)(to + ((piece + 1) ^ sw) * 16) = widen(v[i].z & keep, v[i].w & keep, vs[i]);
    }
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) const uint8_t* LdsPointer;

// Four tokens of one channel a lane, of a 4 x 16 piece whose rows the 16 lanes name eight bytes of.
__device__ __forceinline__ uint2 read_transposed(LdsPointer p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}
__device__ __forceinline__ uint4 read_piece(LdsPointer p) {
  const u32x4 x = *(__attribute__((address_space(3))) const u32x4*)p;
  return make_uint4(x.x, x.y, x.z, x.w);
}

// The scores of a tile of 32 staged tokens, relative to the references.
template <int DT, int D, int NR>
__device__ __forceinline__ void wide_scores(const uint4 (&k)[2][D / 32], const uint4 (&qf)[NR][D / 32], const Reference (&ref)[NR], f32x4 (&sc)[NR][2]) {
#pragma unroll
  for (int n = 0; n < NR; ++n) sc[n][0] = sc[n][1] = ref[n].negative;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < NR; ++n) sc[n][u] = Mat<DT>::mma(k[u][i], qf[n][i], sc[n][u]);
}
// A tile's keys and values at offset `at` from the lane's places: all reads at once, for one by one before their
// products each would be waited for.
template <int D>
__device__ __forceinline__ void wide_keys(const LdsPointer (&key_at)[D / 32], int at, uint4 (&k)[2][D / 32]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) k[u][i] = read_piece(key_at[i] + at + u * 16 * (2 * D));
}
template <int D>
__device__ __forceinline__ void wide_values(const LdsPointer (&value_at)[D / 16], int at, uint2 (&v)[D / 16][2]) {
#pragma unroll
  for (int e = 0; e < D / 16; ++e)
#pragma unroll
    for (int u = 0; u < 2; ++u) v[e][u] = read_transposed(value_at[e] + at + u * 16 * (2 * D));
}
// One tile of 32 staged tokens.
template <int DT, int D, int NR>
__device__ __forceinline__ void wide_tile(const LdsPointer (&key_at)[D / 32], const LdsPointer (&value_at)[D / 16], int at, const uint4 (&qf)[NR][D / 32],
                                          int left, float scale2, Reference (&ref)[NR], Result<D, NR>& r) {
  uint4 k[2][D / 32];
  uint2 v[D / 16][2];
  wide_keys<D>(key_at, at, k);
  wide_values<D>(value_at, at, v);
  __builtin_amdgcn_sched_barrier(0);
  f32x4 sc[NR][2];
  wide_scores<DT, D, NR>(k, qf, ref, sc);
  settle<DT, D, NR>(sc, left, scale2, ref, r);
  uint4 p[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) p[n] = weights<DT, NR>(sc[n], scale2, r.l[n]);
#pragma unroll
  for (int e = 0; e < D / 16; ++e)
#pragma unroll
    for (int n = 0; n < NR; ++n) r.o[n][e] = Mat<DT>::mma(make_uint4(v[e][0].x, v[e][0].y, v[e][1].x, v[e][1].y), p[n], r.o[n][e]);
}

template <int DT, int D, bool MX, class S>
__device__ __forceinline__ void attend_wide(const Stream& s, const uint16_t* const (&q)[S::NR], int t0, int end, int wt, float scale2, Result<D, S::NR>& r,
                                            uint8_t* lds) {
  constexpr int NR = S::NR;
  const int lane = threadIdx.x & 63, quarter = lane >> 4;
  Reference ref[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    ref[n].reset();
    r.l[n] = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) r.o[n][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  StageRegs<DT, D, MX, S> regs;
  regs.load(s, t0, end);
  uint4 qf[NR][D / 32];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) qf[n][i] = q[n] ? *(const uint4*)(q[n] + 32 * i + 8 * quarter) : make_uint4(0, 0, 0, 0);
  // A lane's places in its wave's first tile: keys of token lane % 16 (and 16 on), values of token 4 q + (lane % 16) / 4.
  LdsPointer key_at[D / 32], value_at[D / 16];
  const int tile0 = wt * S::TILES * kTile;  // a wave's tiles of a stage lie together
#pragma unroll
  for (int i = 0; i < D / 32; ++i) key_at[i] = (LdsPointer)lds + (tile0 + (lane & 15)) * (2 * D) + ((4 * i + quarter) ^ S::swizzle(lane & 15)) * 16;
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    const int row = 4 * quarter + ((lane & 15) >> 2);
    value_at[e] = (LdsPointer)lds + S::BYTES + (tile0 + row) * (2 * D) + ((2 * e + ((lane & 2) >> 1)) ^ S::swizzle(row)) * 16 + (lane & 1) * 8;
  }
  // As they stand: worked out anew for each tile, from what they have in common, they would cost more than registers.
#pragma unroll
  for (int i = 0; i < D / 32; ++i) keep_here(key_at[i]);
#pragma unroll
  for (int e = 0; e < D / 16; ++e) keep_here(value_at[e]);
  // Two stages a round, one in each buffer. A stage's barrier also ends the reads of the other buffer: its readers
  // came to this one after them.
  for (int t = t0; t < end; t += 2 * S::TOKENS) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int now = t + half * S::TOKENS, left = end - now - tile0;
      if (half && now >= end) break;
      regs.store(lds + half * 2 * S::BYTES, end - now);
      __syncthreads();
      if (now + S::TOKENS < end) regs.load(s, now + S::TOKENS, end);
      load_fence();
#pragma unroll
      for (int tile = 0; tile < S::TILES; ++tile)
        if (left > tile * kTile)
          wide_tile<DT, D, NR>(key_at, value_at, half * 2 * S::BYTES + tile * kTile * 2 * D, qf, left - tile * kTile, scale2, ref, r);
    }
  }
  conclude<DT, D, NR>(scale2, ref, r);
}

template <int DT, int D, bool PMX, bool OMX, int WR, int W>
__global__ __launch_bounds__(64 * W, 2) void shared_wide_kernel(SharedArgs a) {
  using S = Stage<D, WR, W>;
  constexpr int OWN_WAVES = W / 2;  // two items a workgroup
  constexpr int STAGES = 2 * 2 * S::BYTES, JOIN = finish_bytes(D, S::NR, S::WT, WR), OWN = finish_bytes(D, 1, OWN_WAVES, 1);
  constexpr int BYTES = STAGES > JOIN ? (STAGES > 2 * OWN ? STAGES : 2 * OWN) : (JOIN > 2 * OWN ? JOIN : 2 * OWN);
  __shared__ f32x4 lds[BYTES / 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = blockIdx.x, p_blocks = a.p_groups * 8 * a.row_tiles;
  if (id >= p_blocks)
    return own_item<DT, D, OMX, OWN_WAVES>(a, (int64_t)(id - p_blocks) * 2 + wave / OWN_WAVES, wave % OWN_WAVES, lds + wave / OWN_WAVES * (OWN / 16));
  const int unit = (id / (8 * a.row_tiles)) * 8 + id % 8, tile = id / 8 % a.row_tiles;
  if (unit >= a.p_parts * a.n_kv) return;
  const int part = unit / a.n_kv, h = unit % a.n_kv, wr = wave % WR, wt = wave / WR;
  const uint16_t* q[S::NR];
  int64_t row[S::NR];
#pragma unroll
  for (int n = 0; n < S::NR; ++n) {
    row[n] = prefix_row(a, h, ((tile * WR + wr) * S::NR + n) * 16 + (lane & 15));
    q[n] = row[n] >= 0 ? a.q + row[n] * D : nullptr;
  }
  const int t0 = part * a.p_chunk, end = min(t0 + a.p_chunk, a.prefix_tokens);
  Result<D, S::NR> r;
  attend_wide<DT, D, PMX, S>(stream_of<D, PMX>(a.prefix, 0, h), q, t0, end, wt, a.scale2, r, (uint8_t*)lds);
  finish<D, S::NR, S::WT, true>(a, r, row, part, wt, wr, WR, lds);
}

// A workgroup a query row: its parts' results into one. d/4 threads take a part's channels, four each, and
// the threads' groups the parts in turn. The sums of 64 parts are under way before their weights are known: an empty
// part has written zeros.
template <int D>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a) {
  constexpr int C = D / 4, GROUPS = 256 / C, EACH = 64 / GROUPS;
  __shared__ f32x4 red[GROUPS][C];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, parts = a.p_parts + a.o_parts, group = threadIdx.x / C, c = threadIdx.x % C;
  const float2* ml = a.part_ml + row * parts;
  const float* from = a.part_o + row * parts * D + c * 4;
  float top = -INFINITY, total = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int p0 = 0; p0 < parts; p0 += 64) {
    f32x4 x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int p = p0 + i * GROUPS + group;
      x[i] = p < parts ? *(const f32x4*)(from + (int64_t)p * D) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float2 mine = p0 + lane < parts ? ml[p0 + lane] : make_float2(-INFINITY, 0.0f);
    const float up = fmaxf(top, lkv::wave_max_f32(mine.x));
    const float keep = p0 == 0 ? 0.0f : join_factor(top, total, up), f = join_factor(mine.x, mine.y, up);
    top = up;
    total = total * keep + lkv::wave_sum_f32(mine.y == 0.0f ? 0.0f : f * mine.y);
    o *= keep;
#pragma unroll
    for (int i = 0; i < EACH; ++i) o += x[i] * __shfl(f, i * GROUPS + group);
  }
  red[group][c] = o;
  __syncthreads();
  if (threadIdx.x >= C) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) o += red[i][c];
  o *= total == 0.0f ? 0.0f : 1.0f / total;
  if (a.out_dtype == LKV_F32) {
    store_four<LKV_F32>(a.out, row * D + c * 4, o);
  } else if (a.out_dtype == LKV_BF16) {
    store_four<LKV_BF16>(a.out, row * D + c * 4, o);
  } else {
    store_four<LKV_F16>(a.out, row * D + c * 4, o);
  }
  if (threadIdx.x == 0) a.lse[row] = total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * lkv::kLn2;
}

int check_desc(const lkv_shared_desc* d) {
  LKV_CHECK_ARG(d, "NULL pointer");
  LKV_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "head_dim %d unsupported (64 or 128)", d->head_dim);
  LKV_CHECK_ARG(d->n_seqs >= 0 && d->n_kv > 0 && d->n_q > 0 && d->n_q % d->n_kv == 0, "bad shape: %d sequences, %d query heads over %d",
                d->n_seqs, d->n_q, d->n_kv);
  LKV_CHECK_ARG((int64_t)d->n_seqs * d->n_q <= (1 << 24), "%lld query rows in one call", (long long)d->n_seqs * d->n_q);
  LKV_CHECK_ARG(d->scale > 0.0f && d->scale * lkv::kLog2e < INFINITY, "scale %g: positive and finite", (double)d->scale);
  LKV_CHECK_ARG(d->prefix_tokens >= 0 && d->max_own >= 0 && d->own_tokens >= 0, "bad extent: prefix %d, own %d of at most %d",
                d->prefix_tokens, d->own_tokens, d->max_own);
  LKV_CHECK_ARG(d->prefix_tokens <= (1 << 30) && d->max_own <= (1 << 30), "at most %d tokens: prefix %d, own %d", 1 << 30, d->prefix_tokens,
                d->max_own);
  return LKV_OK;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a call is divided: see SharedArgs.
struct Plan {
  int nr;  // tiles of 16 rows of a wave, on its own stream; 0: through LDS
  int wr;  // there, waves across rows
  int waves;
  int row_tiles, p_parts, p_chunk, p_groups, g_tiles, o_parts, o_chunk;
};

Plan plan_of(const lkv_shared_desc* d) {
  Plan p = {};
  const int g = d->n_q / d->n_kv;
  const int64_t rows = (int64_t)d->n_seqs * g;
  // Rows of a KV head to a form. Up to 32 on streams of the waves' own: 32 rows over 131,072 tokens (d 128, 8 bits / 16; 8 KV heads here
  // and below) take 54 / 96 us, in LDS by eight waves 67 / 97; 40 rows 79 / 110 against 67 / 97. Up to 64 by eight waves: 64 rows take 75 / 107,
  // by four 86 / 105; 80 rows 106 / 133 against 88 / 107. Over 32,768 tokens the order is the same but for 64 rows of 8 bits (26.8 in LDS, 24.6 as
  // streams); up to 4,099 all are within 1 us.
  p.nr = d->prefix_tokens == 0 || rows <= 16 ? 1 : (rows <= 32 ? 2 : 0);
  p.waves = p.nr || rows > 64 ? 4 : 8;
  p.wr = p.waves == 8 ? 2 : 4;
  p.row_tiles = ceil_div(rows, p.nr ? 16 * p.nr : 32 * p.wr);
  p.g_tiles = ceil_div(g, 16);
  // Tokens that a workgroup takes, in steps of 128: so many that all workgroups run at once, one on each CU, and no
  // fewer than fill it for longer than it takes to begin and end.
  const int64_t cus = 256, items = (int64_t)d->n_seqs * d->n_kv * p.g_tiles;
  int64_t tokens = (int64_t)p.row_tiles * d->n_kv * d->prefix_tokens, room = cus, least = 128;
  if (p.nr) {
    tokens += items * d->max_own;
  } else {
    // Own rows, two items a workgroup, beside the prefix's where that is bound by memory and not by the products (32 sequences over 128K
    // tokens: 102 us behind them, 149 beside). 12 sequences over 32,768 tokens with room for 50, 384, 1,024 and 3,000 of their own: 31.8,
    // 41.1, 56.3 and 61.1 behind, 29.6, 32.5, 37.8 and 62.6 beside; over 131,072: 99, 107, 120 and 124 against 102, 103, 104 and 113.
    const int64_t beside = (items + 1) / 2;
    if (d->max_own > 0 && d->max_own <= 1024 && p.waves == 8 && beside <= cus / 4) room -= beside;
    // Two workgroups of four waves a CU, where their parts stay long beside what a part costs to store and join: of 512 tokens, or of 1,024
    // for one tile of 128 rows of d 128, whose 16-bit form is bound by memory. One workgroup / two, us, at parts of 256 (with two), 512 and 1,024:
    // two tiles, d 128, 16 bits 26.6/28.7, 37.6/36.5, 64.0/56.2, 8 bits 29.4/31.6, 38.7/36.8, 62.8/54.3; one tile, d 64, 8 bits 22.2/24.0, 28.6/28.0,
    // 44.9/40.0; one tile, d 128, 16 bits 25.9/29.6, 39.8/42.3, 64.1/68.5, 8 bits 26.5/29.4, 37.9/36.9, 64.2/56.6 (the call does not tell
    // the two apart here: scratch is asked for without the rows).
    const int64_t enough = p.row_tiles == 1 && d->head_dim == 128 ? 1024 : 512;
    if (p.waves == 4 && tokens >= enough * 2 * cus) room = 2 * cus;
    least = 256;
  }
  int64_t chunk = (tokens + room - 1) / room;
  // Few tokens and no prefix: one part, whose workgroup stores the output itself. 200 tokens (d 128, 16 bits) 8.0 -> 5.9 us, 500
  // (d 64, 8 bits) 6.5 -> 5.4; 1,000 of those 6.5 -> 7.4.
  if (d->prefix_tokens == 0 && (int64_t)d->max_own * d->head_dim <= 32768 && d->max_own > least) least = d->max_own;
  chunk = ((chunk < least ? least : chunk) + 127) / 128 * 128;
  p.p_chunk = p.o_chunk = (int)(chunk > (1 << 30) ? (1 << 30) : chunk);
  if (!p.nr) {
    // Own rows in about as many pieces as the card takes at once, four a CU, however many rows there is room for: each stores its
    // partial result, rows or none. Pieces of the prefix's size gave 398 MiB of scratch for 64 sequences with room for 100,000 tokens. 64
    // sequences of 32,768 tokens behind 1,021, d 128, 8 bits: 905 us in pieces of 256 tokens, 740, 729 and 727 in 16, 8 and 4 pieces a CU; 16 of
    // up to 16,384 behind 32,768: 118, 118, 118 and 109.
    const int64_t piece = (items * d->max_own + 4 * cus - 1) / (4 * cus);
    p.o_chunk = p.o_chunk > 1024 ? 1024 : p.o_chunk;
    if (piece > p.o_chunk) p.o_chunk = (int)((piece > (1 << 30) ? (1 << 30) : piece) + 127) / 128 * 128;
  }
  p.p_parts = ceil_div(d->prefix_tokens, p.p_chunk);
  p.o_parts = ceil_div(d->max_own, p.o_chunk);
  p.p_groups = ceil_div((int64_t)p.p_parts * d->n_kv, 8);
  return p;
}

template <int DT, int D, bool PMX, bool OMX>
void launch(const Plan& p, dim3 grid, hipStream_t s, const SharedArgs& a) {
  auto kernel = p.nr == 1      ? shared_decode_kernel<DT, D, PMX, OMX, 1>
                : p.nr == 2    ? shared_decode_kernel<DT, D, PMX, OMX, 2>
                : p.waves == 8 ? shared_wide_kernel<DT, D, PMX, OMX, 2, 8>
                               : shared_wide_kernel<DT, D, PMX, OMX, 4, 4>;
  hipLaunchKernelGGL(kernel, grid, dim3(64 * p.waves), 0, s, a);
}

template <int DT, int D>
void launch(bool pmx, bool omx, const Plan& p, dim3 grid, hipStream_t s, const SharedArgs& a) {
  if (pmx) {
    omx ? launch<DT, D, true, true>(p, grid, s, a) : launch<DT, D, true, false>(p, grid, s, a);
  } else {
    omx ? launch<DT, D, false, true>(p, grid, s, a) : launch<DT, D, false, false>(p, grid, s, a);
  }
}

}  // namespace

extern "C" size_t lkv_shared_decode_workspace_bytes(const lkv_shared_desc* desc) {
  if (check_desc(desc)) return 0;
  const Plan p = plan_of(desc);
  const size_t parts = p.p_parts + p.o_parts, rows = (size_t)desc->n_seqs * desc->n_q;
  return parts < 2 ? 0 : lkv_align_up(rows * parts * sizeof(float2), 16) + rows * parts * desc->head_dim * sizeof(float);
}

extern "C" int lkv_shared_decode(uintptr_t stream, const lkv_shared_desc* desc, const void* q, int q_dtype, const lkv_kv_rows* prefix,
                                 const lkv_kv_rows* own, const int32_t* lengths, void* out, int out_dtype, float* lse, void* ws,
                                 size_t ws_bytes) {
  if (int rc = check_desc(desc)) return rc;
  LKV_CHECK_ARG(q && out && lse, "NULL pointer");
  LKV_CHECK_ARG(q_dtype == LKV_F16 || q_dtype == LKV_BF16, "queries are float16 or bfloat16, got dtype %d", q_dtype);
  LKV_CHECK_ARG(lkv_is_model_dtype(out_dtype), "unsupported output dtype %d", out_dtype);
  LKV_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0, "queries and outputs must start on 16 bytes");
  const size_t need = lkv_shared_decode_workspace_bytes(desc);
  LKV_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), "workspace of %zu bytes: %zu are needed", ws_bytes, need);
  LKV_CHECK_ARG(need == 0 || ((uintptr_t)ws & 15) == 0, "the workspace must start on 16 bytes");
  SharedArgs a = {};
  if (desc->prefix_tokens > 0) {
    LKV_CHECK_ARG(prefix, "a prefix of %d tokens without rows", desc->prefix_tokens);
    if (int rc = lkv_check_rows(prefix, "prefix", 1, q_dtype, desc->head_dim)) return rc;
    LKV_CHECK_ARG(desc->prefix_tokens <= prefix->tokens, "a prefix of %d tokens over %lld rows", desc->prefix_tokens, (long long)prefix->tokens);
    a.prefix = *prefix;
  }
  if (desc->max_own > 0) {
    LKV_CHECK_ARG(own, "%d own tokens without rows", desc->max_own);
    if (int rc = lkv_check_rows(own, "own", desc->n_seqs, q_dtype, desc->head_dim)) return rc;
    LKV_CHECK_ARG(desc->max_own <= own->tokens, "%d own tokens over %lld rows", desc->max_own, (long long)own->tokens);
    a.own = *own;
  }
  if (desc->n_seqs == 0) return LKV_OK;
  const Plan p = plan_of(desc);
  const int64_t rows = (int64_t)desc->n_seqs * desc->n_q, parts = p.p_parts + p.o_parts;
  const int64_t items = (int64_t)desc->n_seqs * desc->n_kv * p.g_tiles * p.o_parts;
  const int64_t blocks = (int64_t)p.p_groups * 8 * p.row_tiles + (p.nr ? items : (items + 1) / 2);
  LKV_CHECK_ARG(blocks < (1LL << 31) && items < (1LL << 31) && rows * parts < (1LL << 31), "%lld workgroups in one call", (long long)blocks);
  a.q = (const uint16_t*)q;
  a.lengths = lengths;
  a.out = out;
  a.lse = lse;
  a.part_ml = (float2*)ws;
  a.part_o = (float*)((uint8_t*)ws + lkv_align_up(rows * parts * sizeof(float2), 16));
  a.scale2 = desc->scale * lkv::kLog2e;
  a.n_seqs = desc->n_seqs;
  a.n_q = desc->n_q;
  a.n_kv = desc->n_kv;
  a.g = desc->n_q / desc->n_kv;
  a.prefix_tokens = desc->prefix_tokens;
  a.own_tokens = desc->own_tokens;
  a.max_own = desc->max_own;
  a.out_dtype = out_dtype;
  a.row_tiles = p.row_tiles;
  a.p_parts = p.p_parts;
  a.p_chunk = p.p_chunk;
  a.p_groups = p.p_groups;
  a.g_tiles = p.g_tiles;
  a.o_parts = p.o_parts;
  a.o_chunk = p.o_chunk;
  const hipStream_t s = (hipStream_t)stream;
  const bool half = q_dtype == LKV_F16, wide = desc->head_dim == 128;
  if (blocks > 0) {
    const bool omx = p.o_parts ? own->dtype == LKV_MXFP8 : prefix->dtype == LKV_MXFP8, pmx = p.p_parts ? prefix->dtype == LKV_MXFP8 : omx;
    const dim3 grid((unsigned)blocks);
    if (half) {
      wide ? launch<LKV_F16, 128>(pmx, omx, p, grid, s, a) : launch<LKV_F16, 64>(pmx, omx, p, grid, s, a);
    } else {
      wide ? launch<LKV_BF16, 128>(pmx, omx, p, grid, s, a) : launch<LKV_BF16, 64>(pmx, omx, p, grid, s, a);
    }
    LKV_CHECK_LAUNCH("shared_decode");
  }
  if (parts != 1) {
    auto join = wide ? shared_join_kernel<128> : shared_join_kernel<64>;
    hipLaunchKernelGGL(join, dim3((unsigned)rows), dim3(256), 0, s, a);
    LKV_CHECK_LAUNCH("shared_decode (join)");
  }
  return LKV_OK;
}
