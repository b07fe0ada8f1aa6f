// Attention's parts that kernels over rows of dense caches share: rows to operands of the matrix units, scores to
// weights, results to memory. A wave takes 32 tokens at a time, as S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32.
#pragma once

#include "lkv_mx.h"

namespace lkv {

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
  // The tile's halves of 16 tokens from streams of their own, each placed as if the tile lay together.
  __device__ __forceinline__ void load(const Stream (&s)[2], const LaneOffsets<D, false>& at) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) w[u][i] = *(const uint4*)(s[u].k + at.key[u] + i * 64);
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
  __device__ __forceinline__ void load(const Stream (&s)[2], const LaneOffsets<D, true>& at) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) w[u][i] = *(const uint4*)(s[u].k + at.key[u] + i * 16);
      scale[u] = s[u].ks[at.key[u] / kMxGroup];
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
  __device__ __forceinline__ void load(const Stream (&s)[2], const LaneOffsets<D, false>& at) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* from = s[j / 4].v + at.value[j];
      if constexpr (D == 128) {
        const uint4 x = *(const uint4*)from;
        w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
      } else {
        const uint2 x = *(const uint2*)from;
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
  __device__ __forceinline__ void load(const Stream (&s)[2], const LaneOffsets<D, true>& at) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* from = s[j / 4].v + at.value[j];
      if constexpr (D == 128) {
        const uint2 x = *(const uint2*)from;
        w[j][0] = x.x, w[j][1] = x.y;
      } else {
        w[j][0] = *(const uint32_t*)from;
      }
    }
    if (!at.cut) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        __builtin_memcpy(scale[u], s[u].vs + (uint32_t)(((threadIdx.x & 48) / 4 + 16 * u) * (D / kMxGroup)), sizeof(scale[u]));
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* from = s[u].vs + at.value[4 * u + j] / D * (D / kMxGroup);
          if constexpr (D == 128) {
            __builtin_memcpy(&scale[u][j], from, 4);
          } else {
            uint16_t x;
            __builtin_memcpy(&x, from, 2);
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

// Settled scores to weights, the second product's operand: in the model dtype, as the matrix units take them at the full rate. Each is then off by half a
// step of it at the most, and independently of the others, so that an output of many rows is off by about as much again as its own rounding makes it: relative to
// 64 bits (root mean square, normal scores and values) 0.0017 by that rounding and 0.0022 by both in bfloat16, 0.00021 and 0.00027 in float16. Their sum is of the weights
// before they are rounded, in float32; of the rounded ones it would change no digit of these.
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

}  // namespace lkv
