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
#include "lkv_mx.h"

namespace {

constexpr int kWaves = 4;      // of a workgroup; each takes every fourth tile of the workgroup's tokens
constexpr int kTile = 32;      // tokens

typedef float f32x4 __attribute__((ext_vector_type(4)));
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

// Keys of a tile: two halves of 16 tokens, a lane token lane % 16 of each. Raw as loaded.
// Model dtype: channels 32 i + 8 q .. + 8 for the i-th product. 8 bits: channels (d/4) q .. + d/4, so that a
// lane's codes lie together under one scale; the i-th product takes the i-th eight of them.
template <int D, bool MX> struct KeyRegs;
template <int D> struct KeyRegs<D, false> {
  uint4 w[2][D / 32];
  __device__ __forceinline__ void load(const Stream& s, int t0, int last) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = min(t0 + 16 * u + (lane & 15), last);
      const uint4* p = (const uint4*)(s.k + (int64_t)t * (2 * D) + (lane >> 4) * 16);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) w[u][i] = p[i * 4];
    }
  }
  template <int DT> __device__ __forceinline__ uint4 operand(int u, int i) const { return w[u][i]; }
  static __device__ __forceinline__ int channel(int q, int i) { return 32 * i + 8 * q; }
};
template <int D> struct KeyRegs<D, true> {
  uint4 w[2][D / 64];
  uint32_t scale[2];
  __device__ __forceinline__ void load(const Stream& s, int t0, int last) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = min(t0 + 16 * u + (lane & 15), last);
      const int64_t at = (int64_t)t * D + (lane >> 4) * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) w[u][i] = ((const uint4*)(s.k + at))[i];
      scale[u] = s.ks[at / kMxGroup];
    }
  }
  template <int DT> __device__ __forceinline__ uint4 operand(int u, int i) const {
    const uint4& x = w[u][i / 2];
    const uint32_t lo = i & 1 ? x.z : x.x, hi = i & 1 ? x.w : x.y;
    const float f = lkv::mx_scale(scale[u]);
    return make_uint4(Mat<DT>::template widen<false>(lo, f), Mat<DT>::template widen<true>(lo, f), Mat<DT>::template widen<false>(hi, f),
                      Mat<DT>::template widen<true>(hi, f));
  }
  static __device__ __forceinline__ int channel(int q, int i) { return (D / 4) * q + 8 * i; }
};

// Values of a tile: eight tokens a lane, d/16 neighbouring channels of each.
template <int D, bool MX> struct ValueRegs;
template <int D> struct ValueRegs<D, false> {
  uint32_t w[8][D / 32];
  __device__ __forceinline__ void load(const Stream& s, int t0, int last) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = min(t0 + (j < 4 ? 0 : 16) + 4 * (lane >> 4) + (j & 3), last);
      const uint8_t* p = s.v + (int64_t)t * (2 * D) + (lane & 15) * (D / 8);
      if constexpr (D == 128) {
        const uint4 x = *(const uint4*)p;
        w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
      } else {
        const uint2 x = *(const uint2*)p;
        w[j][0] = x.x, w[j][1] = x.y;
      }
    }
  }
  __device__ __forceinline__ void clear(int j) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) w[j][c] = 0;
  }
  template <int DT> __device__ __forceinline__ uint32_t pair(int j, int c) const { return w[j][c]; }
};
template <int D> struct ValueRegs<D, true> {
  uint32_t w[8][D / 64];
  uint32_t scale[8];
  __device__ __forceinline__ void load(const Stream& s, int t0, int last) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = min(t0 + (j < 4 ? 0 : 16) + 4 * (lane >> 4) + (j & 3), last);
      const int64_t at = (int64_t)t * D + (lane & 15) * (D / 16);
      if constexpr (D == 128) {
        const uint2 x = *(const uint2*)(s.v + at);
        w[j][0] = x.x, w[j][1] = x.y;
      } else {
        w[j][0] = *(const uint32_t*)(s.v + at);
      }
      scale[j] = s.vs[at / kMxGroup];
    }
  }
  __device__ __forceinline__ void clear(int j) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c) w[j][c] = 0;
    scale[j] = 127;
  }
  template <int DT> __device__ __forceinline__ uint32_t pair(int j, int c) const {
    const float f = lkv::mx_scale(scale[j]);
    return c & 1 ? Mat<DT>::template widen<true>(w[j][c / 2], f) : Mat<DT>::template widen<false>(w[j][c / 2], f);
  }
};

// A wave's running result for 16 * NR rows: lane l has rows l % 16 (+ 16 n) and channels (d/4)(l / 16) .. + d/4,
// channel (d/4) q + (d/16) i + e in o[n][e][i].
template <int D, int NR> struct Result {
  f32x4 o[NR][D / 16];
  float m[NR];  // the maximum so far, in base 2
  float l[NR];  // this lane's tokens' part of the sum
};

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
  uint4 qf[NR][D / 32];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      qf[n][i] = q[n] ? *(const uint4*)(q[n] + KeyRegs<D, MX>::channel(quarter, i)) : make_uint4(0, 0, 0, 0);
  KeyRegs<D, MX> k;
  ValueRegs<D, MX> v;
  k.load(s, first, end - 1);
  v.load(s, first, end - 1);
  for (int t = first; t < end; t += step) {
    f32x4 sc[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) sc[n][0] = sc[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 a = k.template operand<DT>(u, i);
#pragma unroll
        for (int n = 0; n < NR; ++n) sc[n][u] = Mat<DT>::mma(a, qf[n][i], sc[n][u]);
      }
    k.load(s, t + step, end - 1);
    if (t + kTile > end) {  // tokens behind the end: no weight, and no value that a weight of 0 could turn to NaN
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool live = t + (j < 4 ? 0 : 16) + 4 * quarter + (j & 3) < end;
        if (!live) v.clear(j);
#pragma unroll
        for (int n = 0; n < NR; ++n) sc[n][j / 4][j & 3] = live ? sc[n][j / 4][j & 3] : -INFINITY;
      }
    }
    uint4 p[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      // Scaled before they are compared: as s * scale2 - m in one step, large scores' rounding in m alone would leave
      // the largest weight far from 1.
      sc[n][0] *= scale2;
      sc[n][1] *= scale2;
      float top = fmaxf(fmaxf(fmaxf(sc[n][0][0], sc[n][0][1]), fmaxf(sc[n][0][2], sc[n][0][3])),
                        fmaxf(fmaxf(sc[n][1][0], sc[n][1][1]), fmaxf(sc[n][1][2], sc[n][1][3])));
      top = lkv::pair_max<32>(lkv::pair_max<16>(top));
      if (__any(top > r.m[n])) {
        const float next = fmaxf(top, r.m[n]);
        const float keep = r.m[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r.m[n] - next);
        r.m[n] = next;
        r.l[n] *= keep;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) r.o[n][e] *= keep;
      }
      const float base = r.m[n] == -INFINITY ? 0.0f : r.m[n];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(sc[n][j / 4][j & 3] - base);
      r.l[n] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      p[n] = make_uint4(Mat<DT>::pack(w[0], w[1]), Mat<DT>::pack(w[2], w[3]), Mat<DT>::pack(w[4], w[5]), Mat<DT>::pack(w[6], w[7]));
    }
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = v.template pair<DT>(j, c);
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
    v.load(s, t + step, end - 1);
  }
#pragma unroll
  for (int n = 0; n < NR; ++n) r.l[n] = lkv::pair_sum<32>(lkv::pair_sum<16>(r.l[n]));
}

__device__ __forceinline__ float join_factor(float m, float l, float top) {
  return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - top);
}

// The waves' results into wave 0's: waves 2 and 3 to 0 and 1, then 1 to 0, lane by lane.
template <int D, int NR>
__device__ __forceinline__ void join_waves(Result<D, NR>& r, f32x4* so, float2* sml) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int PER = NR * (D / 16);
#pragma unroll
  for (int half = kWaves / 2; half > 0; half /= 2) {
    __syncthreads();
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        sml[((wave - half) * NR + n) * 64 + lane] = make_float2(r.m[n], r.l[n]);
#pragma unroll
        for (int e = 0; e < D / 16; ++e) so[((wave - half) * PER + n * (D / 16) + e) * 64 + lane] = r.o[n][e];
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float2 other = sml[(wave * NR + n) * 64 + lane];
        const float top = fmaxf(r.m[n], other.x);
        const float f = join_factor(r.m[n], r.l[n], top), fo = join_factor(other.x, other.y, top);
        r.m[n] = top;
        r.l[n] = r.l[n] * f + other.y * fo;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) r.o[n][e] = r.o[n][e] * f + so[(wave * PER + n * (D / 16) + e) * 64 + lane] * fo;
      }
    }
  }
}

// A row's result: the output itself where this is its only part.
template <int D>
__device__ __forceinline__ void store_row(const SharedArgs& a, int64_t row, int part, float m, float l, const f32x4 (&o)[D / 16]) {
  const int parts = a.p_parts + a.o_parts, quarter = (threadIdx.x & 63) >> 4;
  if (parts == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t at = row * D + quarter * (D / 4);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < D / 16; ++e) lkv::store_any(a.out, at + (D / 16) * i + e, a.out_dtype, l == 0.0f ? 0.0f : o[e][i] * inv);
    if (quarter == 0) a.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * lkv::kLn2;
    return;
  }
  const int64_t slot = row * parts + part;
  if (quarter == 0) a.part_ml[slot] = make_float2(m, l);
  float* to = a.part_o + slot * D + quarter * (D / 4);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < D / 16; e += 4) *(f32x4*)(to + (D / 16) * i + e) = f32x4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
}

template <int DT, int D, bool PMX, bool OMX, int NR>
__global__ __launch_bounds__(256, NR == 4 ? 1 : 2) void shared_decode_kernel(SharedArgs a) {
  __shared__ f32x4 so[(kWaves / 2) * NR * (D / 16) * 64];
  __shared__ float2 sml[(kWaves / 2) * NR * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = blockIdx.x;
  const int p_blocks = a.p_groups * 8 * a.row_tiles;
  if (id < p_blocks) {
    // Workgroups go round the 8 XCDs by their number: the row tiles of one head and token range sit on
    // one of them, one after the other, and find its keys and values in that L2.
    const int unit = (id / (8 * a.row_tiles)) * 8 + id % 8, tile = id / 8 % a.row_tiles;
    if (unit >= a.p_parts * a.n_kv) return;
    const int part = unit / a.n_kv, h = unit % a.n_kv;
    const uint16_t* q[NR];
    int64_t row[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int x = (tile * NR + n) * 16 + (lane & 15), b = x / a.g;
      row[n] = b < a.n_seqs ? (int64_t)b * a.n_q + h * a.g + (x - b * a.g) : -1;
      q[n] = row[n] >= 0 ? a.q + row[n] * D : nullptr;
    }
    const int t0 = part * a.p_chunk, end = min(t0 + a.p_chunk, a.prefix_tokens);
    Result<D, NR> r;
    attend_range<DT, D, PMX, NR>(stream_of<D, PMX>(a.prefix, 0, h), q, t0 + wave * kTile, kWaves * kTile, end, a.scale2, r);
    join_waves<D, NR>(r, so, sml);
    if (wave == 0) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
        if (row[n] >= 0) store_row<D>(a, row[n], part, r.m[n], r.l[n], r.o[n]);
    }
    return;
  }
  id -= p_blocks;
  const int part = id % a.o_parts;
  id /= a.o_parts;
  const int tile = id % a.g_tiles;
  id /= a.g_tiles;
  const int h = id % a.n_kv, b = id / a.n_kv;
  const int j = tile * 16 + (lane & 15);
  const int64_t row = (int64_t)b * a.n_q + h * a.g + j;
  const int t0 = part * a.o_chunk, end = min(t0 + a.o_chunk, own_length(a, b));
  const uint16_t* q[1] = {j < a.g ? a.q + row * D : nullptr};
  Result<D, 1> r;
  attend_range<DT, D, OMX, 1>(stream_of<D, OMX>(a.own, b, h), q, t0 + wave * kTile, kWaves * kTile, end, a.scale2, r);
  join_waves<D, 1>(r, so, sml);
  if (wave == 0 && j < a.g) store_row<D>(a, row, a.p_parts + part, r.m[0], r.l[0], r.o[0]);
}

// A wave a query row: its parts' results into one.
template <int D>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.n_seqs * a.n_q) return;
  const int lane = threadIdx.x & 63, parts = a.p_parts + a.o_parts;
  const float2* ml = a.part_ml + row * parts;
  float top = -INFINITY;
  for (int p = lane; p < parts; p += 64) top = fmaxf(top, ml[p].x);
  top = lkv::wave_max_f32(top);
  float total = 0.0f, o[D / 64] = {};
  const float* from = a.part_o + row * parts * D + lane * (D / 64);
  for (int p = 0; p < parts; ++p) {
    const float2 x = ml[p];
    if (x.y == 0.0f) continue;
    const float f = join_factor(x.x, x.y, top);
    total += f * x.y;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] += f * from[(int64_t)p * D + i];
  }
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    lkv::store_any(a.out, row * D + lane * (D / 64) + i, a.out_dtype, total == 0.0f ? 0.0f : o[i] / total);
  if (lane == 0) a.lse[row] = total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * lkv::kLn2;
}

int check_desc(const lkv_shared_desc* d) {
  LKV_CHECK_ARG(d, "NULL pointer");
  LKV_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "head_dim %d unsupported (64 or 128)", d->head_dim);
  LKV_CHECK_ARG(d->n_seqs >= 0 && d->n_kv > 0 && d->n_q > 0 && d->n_q % d->n_kv == 0, "bad shape: %d sequences, %d query heads over %d",
                d->n_seqs, d->n_q, d->n_kv);
  LKV_CHECK_ARG((int64_t)d->n_seqs * d->n_q <= (1 << 24), "%lld query rows in one call", (long long)d->n_seqs * d->n_q);
  LKV_CHECK_ARG(d->scale > 0.0f && d->scale < INFINITY, "scale %g: positive and finite", (double)d->scale);
  LKV_CHECK_ARG(d->prefix_tokens >= 0 && d->max_own >= 0 && d->own_tokens >= 0, "bad extent: prefix %d, own %d of at most %d",
                d->prefix_tokens, d->own_tokens, d->max_own);
  LKV_CHECK_ARG(d->prefix_tokens <= (1 << 30) && d->max_own <= (1 << 30), "at most %d tokens: prefix %d, own %d", 1 << 30, d->prefix_tokens,
                d->max_own);
  return LKV_OK;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a call is divided: see SharedArgs.
struct Plan {
  int nr, row_tiles, p_parts, p_chunk, p_groups, g_tiles, o_parts, o_chunk;
};

Plan plan_of(const lkv_shared_desc* d) {
  Plan p = {};
  const int g = d->n_q / d->n_kv;
  const int64_t rows = (int64_t)d->n_seqs * g;
  p.nr = d->prefix_tokens == 0 || rows <= 16 ? 1 : (rows <= 32 ? 2 : 4);
  p.row_tiles = ceil_div(rows, 16 * p.nr);
  p.g_tiles = ceil_div(g, 16);
  // Tokens that a workgroup takes: as many workgroups as the card holds at once, and no fewer than one tile
  // a wave.
  const int64_t room = p.nr == 4 ? 256 : 512;
  const int64_t tokens = (int64_t)p.row_tiles * d->n_kv * d->prefix_tokens + (int64_t)d->n_seqs * d->n_kv * p.g_tiles * d->max_own;
  const int64_t least = kWaves * kTile;
  int64_t chunk = (tokens / room + least - 1) / least * least;
  if (chunk < least) chunk = least;
  p.p_chunk = p.o_chunk = (int)(chunk > (1 << 30) ? (1 << 30) : chunk);
  p.p_parts = ceil_div(d->prefix_tokens, p.p_chunk);
  p.o_parts = ceil_div(d->max_own, p.o_chunk);
  p.p_groups = ceil_div((int64_t)p.p_parts * d->n_kv, 8);
  return p;
}

template <int DT, int D, bool PMX, bool OMX>
void launch(int nr, dim3 grid, hipStream_t s, const SharedArgs& a) {
  auto kernel = nr == 1 ? shared_decode_kernel<DT, D, PMX, OMX, 1> : nr == 2 ? shared_decode_kernel<DT, D, PMX, OMX, 2> : shared_decode_kernel<DT, D, PMX, OMX, 4>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a);
}

template <int DT, int D>
void launch(bool pmx, bool omx, int nr, dim3 grid, hipStream_t s, const SharedArgs& a) {
  if (pmx) {
    omx ? launch<DT, D, true, true>(nr, grid, s, a) : launch<DT, D, true, false>(nr, grid, s, a);
  } else {
    omx ? launch<DT, D, false, true>(nr, grid, s, a) : launch<DT, D, false, false>(nr, grid, s, a);
  }
}

}  // namespace

extern "C" size_t lkv_shared_decode_workspace_bytes(const lkv_shared_desc* desc) {
  if (check_desc(desc)) return 0;
  const Plan p = plan_of(desc);
  const size_t parts = p.p_parts + p.o_parts, rows = (size_t)desc->n_seqs * desc->n_q;
  return parts < 2 ? 16 : lkv_align_up(rows * parts * sizeof(float2), 16) + rows * parts * desc->head_dim * sizeof(float);
}

extern "C" int lkv_shared_decode(uintptr_t stream, const lkv_shared_desc* desc, const void* q, int q_dtype, const lkv_kv_rows* prefix,
                                 const lkv_kv_rows* own, const int32_t* lengths, void* out, int out_dtype, float* lse, void* ws,
                                 size_t ws_bytes) {
  if (int rc = check_desc(desc)) return rc;
  LKV_CHECK_ARG(q && out && lse, "NULL pointer");
  LKV_CHECK_ARG(q_dtype == LKV_F16 || q_dtype == LKV_BF16, "queries are float16 or bfloat16, got dtype %d", q_dtype);
  LKV_CHECK_ARG(lkv_is_model_dtype(out_dtype), "unsupported output dtype %d", out_dtype);
  LKV_CHECK_ARG(((uintptr_t)q & 15) == 0, "queries must start on 16 bytes");
  LKV_CHECK_ARG(ws && ws_bytes >= lkv_shared_decode_workspace_bytes(desc), "workspace of %zu bytes: %zu are needed", ws_bytes,
                lkv_shared_decode_workspace_bytes(desc));
  LKV_CHECK_ARG(((uintptr_t)ws & 15) == 0, "the workspace must start on 16 bytes");
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
  const int64_t blocks = (int64_t)p.p_groups * 8 * p.row_tiles + (int64_t)desc->n_seqs * desc->n_kv * p.g_tiles * p.o_parts;
  LKV_CHECK_ARG(blocks < (1LL << 31) && rows * parts < (1LL << 31), "%lld workgroups in one call", (long long)blocks);
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
      wide ? launch<LKV_F16, 128>(pmx, omx, p.nr, grid, s, a) : launch<LKV_F16, 64>(pmx, omx, p.nr, grid, s, a);
    } else {
      wide ? launch<LKV_BF16, 128>(pmx, omx, p.nr, grid, s, a) : launch<LKV_BF16, 64>(pmx, omx, p.nr, grid, s, a);
    }
    LKV_CHECK_LAUNCH("shared_decode");
  }
  if (parts != 1) {
    auto join = wide ? shared_join_kernel<128> : shared_join_kernel<64>;
    hipLaunchKernelGGL(join, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    LKV_CHECK_LAUNCH("shared_decode (join)");
  }
  return LKV_OK;
}
