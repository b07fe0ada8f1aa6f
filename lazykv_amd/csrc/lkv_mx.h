// Rows of dense caches (lkv_kv_rows): their checks, and the 8-bit rows' codes.
//
// LKV_MXFP8 holds a value as an E4M3 code (a sign, 4 exponent bits, 3 mantissa bits, largest 448) under
// a scale 2^(X - 127) that 32 neighbouring channels share: X is a byte. A power of two as the scale
// makes both directions exact but for one rounding: x * 2^(127 - X) loses nothing, the code is its
// nearest E4M3 value, and a code times its scale has four significant bits, so it is a bfloat16 or
// float16 value as it stands (bfloat16 values below the normal range apart).
#pragma once

#include "lkv_common.h"

constexpr int kMxGroup = 32;  // channels that share a scale

// Rows that are written: none of them may share an address with another (lkv_rows.hip). Strides and head_dim in elements of `bytes` bytes; v may be NULL.
int lkv_distinct_rows(const char* what, const void* k, const void* v, int bytes, int n_seqs, int n_kv, int64_t tokens, int head_dim, int64_t seq_stride,
                      int64_t head_stride, int64_t token_stride);
int lkv_distinct_dst(const lkv_kv_rows* dst, int n_kv, int head_dim);

// The arguments every rows call checks the same way. `what` names the rows in the message.
static inline int lkv_check_rows(const lkv_kv_rows* r, const char* what, int n_seqs, int dtype, int head_dim) {
  LKV_CHECK_ARG(r->k && r->v, "%s: NULL pointer", what);
  LKV_CHECK_ARG(r->dtype == dtype || r->dtype == LKV_MXFP8, "%s: rows of dtype %d under a call in dtype %d", what, r->dtype, dtype);
  LKV_CHECK_ARG(r->seqs == n_seqs, "%s: rows of %d sequences, not %d", what, r->seqs, n_seqs);
  LKV_CHECK_ARG(r->tokens >= 0 && r->tokens < (1LL << 31), "%s: %lld tokens", what, (long long)r->tokens);
  LKV_CHECK_ARG(r->seq_stride % kMxGroup == 0 && r->head_stride % kMxGroup == 0, "%s: strides must be multiples of %d elements", what,
                kMxGroup);
  LKV_CHECK_ARG((((uintptr_t)r->k | (uintptr_t)r->v) & 15) == 0, "%s: rows must start on 16 bytes", what);
  if (r->dtype == LKV_MXFP8) {
    LKV_CHECK_ARG(r->k_scale && r->v_scale, "%s: 8-bit rows need their scales", what);
    LKV_CHECK_ARG(r->deq_dtype == dtype, "%s: 8-bit rows of dtype %d under a call in dtype %d", what, r->deq_dtype, dtype);
    LKV_CHECK_ARG((((uintptr_t)r->k_scale | (uintptr_t)r->v_scale) & (head_dim / kMxGroup - 1)) == 0,
                  "%s: a row's scales must start on %d bytes", what, head_dim / kMxGroup);
  }
  return LKV_OK;
}

namespace lkv {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// 2^(X - 127) as a float: the exponent field, but for X = 0, which is below the normal range.
__device__ __forceinline__ float mx_scale(uint32_t x) { return bits_to_float(x ? x << 23 : 0x00400000u); }

// The largest value of the model dtype that four significant bits hold.
template <int DT>
__device__ __forceinline__ float mx_largest() {
  return DT == LKV_F16 ? 61440.0f : bits_to_float(0x7f700000u);
}

// The four values of a word of codes, times their scale.
__device__ __forceinline__ void mx_widen(uint32_t codes, float scale, float (&out)[4]) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  out[0] = a.x * scale;
  out[1] = a.y * scale;
  out[2] = b.x * scale;
  out[3] = b.y * scale;
}

// Eight channels of a row to codes; a quad of lanes, which hold a group, shares the scale. Every lane of the quad has to be here.
template <int DT>
__device__ __forceinline__ uint2 mx_encode(float (&x)[8], uint32_t& scale) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(x[i]);
    const bool fine = a < INFINITY;
    most = fmaxf(most, fine ? a : 0.0f);
    x[i] = fine ? x[i] : NAN;
  }
  most = fmaxf(most, dpp<kDppQuadSwap1>(most));
  most = fmaxf(most, dpp<kDppQuadSwap2>(most));
  // 448 = 1.75 * 2^8.
  const float top = fminf(most, mx_largest<DT>());
  const uint32_t bits = float_to_bits(top);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  scale = e > 0 ? e : 0;
  const float up = bits_to_float((254u - scale) << 23);
  uint32_t code[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float v = x[4 * i + j];
      // A NaN passes both comparisons' selects.
      const float lim = v > mx_largest<DT>() ? mx_largest<DT>() : (v < -mx_largest<DT>() ? -mx_largest<DT>() : v);
      y[j] = lim * up;
    }
    int packed = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], packed, true);
    code[i] = (uint32_t)packed;
  }
  return make_uint2(code[0], code[1]);
}

}  // namespace lkv
