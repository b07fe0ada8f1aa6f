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

}  // namespace lkv
