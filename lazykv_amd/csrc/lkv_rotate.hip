// New tokens' queries and keys normalised over each head and rotated, keys and values written to their rows (lkv_rotate_append).
#include <cfloat>

#include "lkv_attend.h"
#include "lkv_pages.h"

namespace {

struct RotateArgs {
  lkv_rotate_desc d;
  const uint16_t *q, *k, *v;
  const void *cos, *sin, *q_weight, *k_weight;
  uint16_t* q_out;
  lkv::PagedRows rows;
  const int32_t* starts;
  const int32_t* counts;
  int32_t start;
  uint32_t heads;   // n_q + 2 n_kv
  uint32_t splits;  // workgroups of a token
  uint32_t share;   // heads of each
};

// Eight neighbouring values in the model dtype or in float32.
template <int DT>
__device__ __forceinline__ void load_eight(const void* p, int64_t at, bool wide, float (&out)[8]) {
  if (wide) {
    const float4 a = *(const float4*)((const float*)p + at), b = *(const float4*)((const float*)p + at + 4);
    out[0] = a.x, out[1] = a.y, out[2] = a.z, out[3] = a.w, out[4] = b.x, out[5] = b.y, out[6] = b.z, out[7] = b.w;
  } else {
    const uint4 w = *(const uint4*)((const uint16_t*)p + at);
    const lkv::RowWords<DT, 8> words = {{w.x, w.y, w.z, w.w}};
    lkv::widen_row_words<DT, 8>(words, out);
  }
}

// A workgroup takes a token, or some of its heads where there are few tokens: sixteen lanes (head_dim 128) or eight (64) hold a head, 8 channels a lane, and go on to
// the head 16 further with the same tables and weights. Those are folded once: a channel becomes
//   (x a + z b) / rms,  a = weight cos, b = -+ weight' sin,
// z the channel half a rotation away. It is loaded again rather than sent by the lane that has it: it is in the cache line or the next, and any
// rotary width takes the same path.
//
// Bound by memory: 4,099 tokens of 48 heads (d 128), 103 MB, 22.6 us, 4.6 TB/s of the 5.1 that a large copy reaches; one token 4 us, a launch. With few tokens by their rounds of heads, of
// which each loads, reduces and stores before the next: 2,600 tokens of 48 heads (d 64) into 8-bit rows, 49 MB, 13.9 us, 3.5 TB/s.
constexpr int kHeads = 16;  // that a workgroup holds at a time
template <int DT, int D, bool MX>
__global__ __launch_bounds__(kHeads * D / 8) void rotate_append_kernel(RotateArgs a) {
  constexpr int LPR = D / 8;
  const uint32_t bt = blockIdx.x / a.splits, split = blockIdx.x - bt * a.splits;
  const uint32_t b = bt / (uint32_t)a.d.tokens, t = bt - b * (uint32_t)a.d.tokens;
  const int c = (threadIdx.x % LPR) * 8, half = a.d.rotary / 2, other = c < half ? c + half : c - half;
  const bool turns = c < a.d.rotary;
  // The token's row: the same in every head.
  const int64_t row = (int64_t)a.start + (a.starts ? a.starts[b] : 0) + t;
  const bool kept = (!a.counts || (int)t < a.counts[b]) && row >= 0 && row < a.rows.capacity;
  const lkv::Sixteen place = kept ? lkv::sixteen_of<D>(a.rows, (int)b, 0, (int)(row >> 4)) : lkv::Sixteen{0, false};
  const int64_t to = place.at + (row & 15) * D + c;
  float qa[8], qb[8], ka[8], kb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qa[i] = ka[i] = 1.0f, qb[i] = kb[i] = 0.0f;
  if (turns) {
    const int64_t at = b * a.d.table_seq_stride + (int64_t)t * a.d.rotary + c;
    load_eight<DT>(a.cos, at, a.d.table_dtype == LKV_F32, qa);
    load_eight<DT>(a.sin, at, a.d.table_dtype == LKV_F32, qb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qb[i] = c < half ? -qb[i] : qb[i];
      ka[i] = qa[i];
      kb[i] = qb[i];
    }
  }
  const auto weigh = [&](const void* weight, float(&wa)[8], float(&wb)[8]) {
    if (!weight) return;
    const bool wide = a.d.weight_dtype == LKV_F32;
    float w[8];
    load_eight<DT>(weight, c, wide, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) wa[i] *= w[i];
    if (!turns) return;
    load_eight<DT>(weight, other, wide, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) wb[i] *= w[i];
  };
  weigh(a.q_weight, qa, qb);
  weigh(a.k_weight, ka, kb);
  const uint32_t end = min((split + 1) * a.share, a.heads);
  for (uint32_t head = split * a.share + threadIdx.x / LPR; head < end; head += kHeads) {  // whole heads leave: the quads of the others stay complete
    const bool is_q = head < (uint32_t)a.d.n_q, is_v = head >= (uint32_t)(a.d.n_q + a.d.n_kv);
    const int h = (int)(is_q ? head : is_v ? head - a.d.n_q - a.d.n_kv : head - a.d.n_q);
    if (!is_q && !place.there) continue;
    const uint16_t* x = is_q   ? a.q + b * a.d.q_stride[0] + h * a.d.q_stride[1] + t * a.d.q_stride[2]
                        : is_v ? a.v + b * a.d.v_stride[0] + h * a.d.v_stride[1] + t * a.d.v_stride[2]
                               : a.k + b * a.d.k_stride[0] + h * a.d.k_stride[1] + t * a.d.k_stride[2];
    uint4 word = *(const uint4*)(x + c);
    if (!is_v) {
      const lkv::RowWords<DT, 8> words = {{word.x, word.y, word.z, word.w}};
      float y[8], z[8];
      lkv::widen_row_words<DT, 8>(words, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = 0.0f;
      if (turns) load_eight<DT>(x, other, false, z);
      float inverse = 1.0f;
      if (is_q ? a.q_weight != nullptr : a.k_weight != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(y[i], y[i], sum);
        // The reciprocal root takes a subnormal number for 0: such a mean square (without eps, of bfloat16 values below 2^-63) is taken times 2^48.
        const float mean = lkv::row_sum<LPR>(sum) * (1.0f / D) + a.d.eps;
        const bool tiny = mean < FLT_MIN;
        inverse = __builtin_amdgcn_rsqf(tiny ? mean * 0x1p48f : mean);
        inverse = tiny ? inverse * 0x1p24f : inverse;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(y[i], is_q ? qa[i] : ka[i], z[i] * (is_q ? qb[i] : kb[i])) * inverse;
      using M = lkv::Mat<DT>;
      word = make_uint4(M::pack(y[0], y[1]), M::pack(y[2], y[3]), M::pack(y[4], y[5]), M::pack(y[6], y[7]));
    }
    if (is_q) {
      *(uint4*)(a.q_out + b * a.d.out_stride[0] + h * a.d.out_stride[1] + t * a.d.out_stride[2] + c) = word;
      continue;
    }
    const int64_t at = to + h * a.rows.rows.head_stride;
    if constexpr (MX) {
      // From the rounded values: the cache does not tell by which call a token came.
      const lkv::RowWords<DT, 8> words = {{word.x, word.y, word.z, word.w}};
      float y[8];
      lkv::widen_row_words<DT, 8>(words, y);
      uint32_t scale;
      const uint2 codes = lkv::mx_encode<DT>(y, scale);
      *(uint2*)((uint8_t*)(is_v ? a.rows.rows.v : a.rows.rows.k) + at) = codes;
      if ((threadIdx.x & 3) == 0) ((uint8_t*)(is_v ? a.rows.rows.v_scale : a.rows.rows.k_scale))[at / kMxGroup] = (uint8_t)scale;
    } else {
      *(uint4*)((uint16_t*)(is_v ? a.rows.rows.v : a.rows.rows.k) + at) = word;
    }
  }
}

}  // namespace

extern "C" int lkv_rotate_append(uintptr_t stream, const lkv_rotate_desc* desc, const void* q, const void* k, const void* v, const void* cos, const void* sin,
                                 const void* q_weight, const void* k_weight, void* q_out, const lkv_kv_rows* dst, const lkv_pages* pages,
                                 const int32_t* starts, int start, const int32_t* counts) {
  LKV_CHECK_ARG(desc && q && k && v && q_out, "NULL pointer");
  const lkv_rotate_desc& d = *desc;
  LKV_CHECK_ARG(d.dtype == LKV_F16 || d.dtype == LKV_BF16, "tokens are float16 or bfloat16, got dtype %d", d.dtype);
  LKV_CHECK_ARG(d.head_dim == 64 || d.head_dim == 128, "head_dim %d unsupported (64 or 128)", d.head_dim);
  LKV_CHECK_ARG(d.n_seqs >= 0 && d.n_q > 0 && d.n_kv > 0 && d.tokens >= 0, "bad shape: %d sequences, %d and %d heads, %d tokens", d.n_seqs, d.n_q, d.n_kv, d.tokens);
  LKV_CHECK_ARG(d.rotary >= 0 && d.rotary <= d.head_dim && d.rotary % 16 == 0, "%d channels rotated: a multiple of 16, at most %d", d.rotary, d.head_dim);
  LKV_CHECK_ARG(d.rotary == 0 || (cos && sin), "a rotation without its tables");
  LKV_CHECK_ARG(d.rotary == 0 || d.table_dtype == d.dtype || d.table_dtype == LKV_F32, "tables of dtype %d", d.table_dtype);
  LKV_CHECK_ARG((!q_weight && !k_weight) || d.weight_dtype == d.dtype || d.weight_dtype == LKV_F32, "weights of dtype %d", d.weight_dtype);
  // Few bits would be left of a subnormal eps.
  LKV_CHECK_ARG((d.eps == 0.0f || d.eps >= FLT_MIN) && d.eps < INFINITY, "eps %g: 0 or a normal number", (double)d.eps);
  uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)q_weight | (uintptr_t)k_weight;
  if (d.rotary) all |= (uintptr_t)cos | (uintptr_t)sin;
  LKV_CHECK_ARG((all & 15) == 0, "tokens, tables and weights must start on 16 bytes");
  int64_t strides = d.table_seq_stride;
  for (int i = 0; i < 3; ++i) strides |= d.q_stride[i] | d.k_stride[i] | d.v_stride[i] | d.out_stride[i];
  LKV_CHECK_ARG((strides & 7) == 0, "strides must be multiples of 8 elements");
  RotateArgs a = {};
  if (int rc = lkv_paged_rows(dst, pages, d.n_seqs, d.dtype, d.head_dim, a.rows)) return rc;
  if (!starts) LKV_CHECK_ARG(start >= 0 && (int64_t)start + d.tokens <= a.rows.capacity, "rows %d..%lld exceed the %d there are", start,
                             (long long)start + d.tokens, a.rows.capacity);
  const int64_t heads = (int64_t)d.n_q + 2 * (int64_t)d.n_kv, tokens = (int64_t)d.n_seqs * d.tokens;
  // All heads of a token by one workgroup, or, of few tokens, as many as it has lanes for (48 heads, d 128): 64 tokens 5.6 and 4.4 us, 256 5.9 and 5.1,
  // 512 6.6 and 6.9, 1,024 8.5 and 10.4, 4,096 21.8 and 33.
  const int64_t splits = tokens >= 512 ? 1 : (heads + kHeads - 1) / kHeads;
  // (2^24 workgroups of 256 threads are more than a launch has.)
  LKV_CHECK_ARG(heads < (1LL << 31) && (__int128)heads * tokens < (1LL << 31) && (__int128)tokens * splits < (1 << 24), "%lld heads of %lld tokens in one call", (long long)heads,
                (long long)tokens);
  if (tokens == 0) return LKV_OK;
  if (int rc = lkv_distinct_dst(dst, d.n_kv, d.head_dim)) return rc;
  if (int rc = lkv_distinct_rows("q_out", q_out, nullptr, 2, d.n_seqs, d.n_q, d.tokens, d.head_dim, d.out_stride[0], d.out_stride[1], d.out_stride[2])) return rc;
  a.d = d;
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.cos = cos;
  a.sin = sin;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.q_out = (uint16_t*)q_out;
  a.starts = starts;
  a.counts = counts;
  a.start = start;
  a.heads = (uint32_t)heads;
  a.splits = (uint32_t)splits;
  a.share = splits == 1 ? a.heads : kHeads;
  const bool mx = dst->dtype == LKV_MXFP8, half = d.dtype == LKV_F16, wide = d.head_dim == 128;
  auto kernel = half ? (wide ? (mx ? rotate_append_kernel<LKV_F16, 128, true> : rotate_append_kernel<LKV_F16, 128, false>)
                             : (mx ? rotate_append_kernel<LKV_F16, 64, true> : rotate_append_kernel<LKV_F16, 64, false>))
                     : (wide ? (mx ? rotate_append_kernel<LKV_BF16, 128, true> : rotate_append_kernel<LKV_BF16, 128, false>)
                             : (mx ? rotate_append_kernel<LKV_BF16, 64, true> : rotate_append_kernel<LKV_BF16, 64, false>));
  hipLaunchKernelGGL(kernel, dim3((uint32_t)(tokens * a.splits)), dim3(kHeads * d.head_dim / 8), 0, (hipStream_t)stream, a);
  LKV_CHECK_LAUNCH("rotate_append");
  return LKV_OK;
}
