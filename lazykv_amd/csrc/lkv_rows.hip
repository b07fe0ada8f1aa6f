// Rows of dense caches: new tokens' keys and values into a cache (lkv_append_rows), in 8 bits or as they
// are, and 8-bit rows back into the model dtype (lkv_read_rows).
#include "lkv_mx.h"

namespace {

// A row's element offset in the cache and in the tensors of a call.
struct RowPlan {
  int64_t seq_stride, head_stride;                  // cache
  int64_t x_seq_stride, x_head_stride, x_tok_stride;  // tensors
  int64_t cap;
  int32_t n_kv, tokens, start;
  uint32_t rows;  // n_seqs * n_kv * tokens
  const int32_t* starts;
};

// Eight lanes (head_dim 64) or sixteen (128) hold a row, 8 channels a lane; a quad of lanes shares a scale.
// A thread takes the row's keys and its values: the quad's maximum is two DPP moves, a row's loads and stores are one piece, and one
// launch serves both. Bound by memory: a value is read and written once. 32,768 tokens of 8 heads, d 64, float16 into 8
// bits: 20.7 us (102 MB, 4.9 TB/s; a large copy reaches 5.0). One token: 2.6 us, a launch's own time.
template <int DT, int D, bool MX>
__global__ __launch_bounds__(256) void append_rows_kernel(RowPlan p, const uint16_t* __restrict__ xk, const uint16_t* __restrict__ xv,
                                                            uint8_t* __restrict__ ck, uint8_t* __restrict__ cv,
                                                            uint8_t* __restrict__ sk, uint8_t* __restrict__ sv) {
  constexpr int LPR = D / 8;
  const uint32_t r = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;
  const int c = (threadIdx.x % LPR) * 8;
  if (r >= p.rows) return;  // whole rows leave: the quads of the others stay complete
  const uint32_t bh = r / (uint32_t)p.tokens, t = r - bh * (uint32_t)p.tokens;
  const uint32_t b = bh / (uint32_t)p.n_kv, h = bh - b * (uint32_t)p.n_kv;
  const int64_t row = (int64_t)p.start + (p.starts ? p.starts[b] : 0) + t;
  if (row < 0 || row >= p.cap) return;
  const int64_t src = (int64_t)b * p.x_seq_stride + (int64_t)h * p.x_head_stride + (int64_t)t * p.x_tok_stride + c;
  const int64_t dst = (int64_t)b * p.seq_stride + (int64_t)h * p.head_stride + row * D + c;
  const uint4 wk = *(const uint4*)(xk + src), wv = *(const uint4*)(xv + src);
  if constexpr (!MX) {
    *(uint4*)((uint16_t*)ck + dst) = wk;
    *(uint4*)((uint16_t*)cv + dst) = wv;
  } else {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint4 w = which ? wv : wk;
      lkv::RowWords<DT, 8> words = {{w.x, w.y, w.z, w.w}};
      float x[8];
      lkv::widen_row_words<DT, 8>(words, x);
      uint32_t scale;
      const uint2 codes = lkv::mx_encode<DT>(x, scale);
      *(uint2*)((which ? cv : ck) + dst) = codes;
      if ((threadIdx.x & 3) == 0) (which ? sv : sk)[dst / kMxGroup] = (uint8_t)scale;
    }
  }
}

// The way back, divided alike: 131,072 tokens of 8 heads, d 128, to bfloat16 take 135 us (814 MB, 6.0 TB/s).
template <int DT, int D>
__global__ __launch_bounds__(256) void read_rows_kernel(RowPlan p, const uint8_t* __restrict__ ck, const uint8_t* __restrict__ cv,
                                                          const uint8_t* __restrict__ sk, const uint8_t* __restrict__ sv,
                                                          uint16_t* __restrict__ xk, uint16_t* __restrict__ xv) {
  constexpr int LPR = D / 8;
  const uint32_t r = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;
  const int c = (threadIdx.x % LPR) * 8;
  if (r >= p.rows) return;
  const uint32_t bh = r / (uint32_t)p.tokens, t = r - bh * (uint32_t)p.tokens;
  const uint32_t b = bh / (uint32_t)p.n_kv, h = bh - b * (uint32_t)p.n_kv;
  const int64_t src = (int64_t)b * p.seq_stride + (int64_t)h * p.head_stride + ((int64_t)p.start + t) * D + c;
  const int64_t dst = (int64_t)b * p.x_seq_stride + (int64_t)h * p.x_head_stride + (int64_t)t * p.x_tok_stride + c;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint2 code = *(const uint2*)((which ? cv : ck) + src);
    const float scale = lkv::mx_scale((which ? sv : sk)[src / kMxGroup]);
    float x[8];
    float (&lo)[4] = *(float (*)[4])x;
    float (&hi)[4] = *(float (*)[4])(x + 4);
    lkv::mx_widen(code.x, scale, lo);
    lkv::mx_widen(code.y, scale, hi);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)lkv::Elem<DT>::store(x[2 * i]) | ((uint32_t)lkv::Elem<DT>::store(x[2 * i + 1]) << 16);
    *(uint4*)((which ? xv : xk) + dst) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// One dimension of a set of rows: `count` of them, `stride` apart.
struct Dim {
  int64_t count, stride;
};

// Whether no two of the spans of `length` that start at sums of the dimensions' multiples share an address. Strides that nest, each at least
// what the smaller ones reach, are seen at once: slices, steps and permutations of contiguous tensors have such. Otherwise every difference of
// two spans is tried, along the longest dimension only the multiples that come next to zero; over 65,536 tries are not made,
// and the spans not taken for apart.
bool rows_apart(Dim (&dims)[4], int64_t length) {
  for (int i = 0; i < 4; ++i) {
    if (dims[i].count < 2) dims[i] = {1, 0};
    dims[i].stride = dims[i].stride < 0 ? -dims[i].stride : dims[i].stride;  // the same differences
    for (int j = i; j > 0 && dims[j].stride < dims[j - 1].stride; --j) {
      const Dim x = dims[j];
      dims[j] = dims[j - 1];
      dims[j - 1] = x;
    }
  }
  __int128 reach = length;
  bool nested = true;
  for (const Dim& d : dims) {
    if (d.count < 2) continue;
    nested = nested && d.stride >= reach;
    reach += (__int128)d.stride * (d.count - 1);
  }
  if (nested) return true;
  int most = 0;
  for (int i = 1; i < 4; ++i)
    if (dims[i].count > dims[most].count) most = i;
  __int128 tries = 1;
  for (int i = 0; i < 4; ++i)
    if (i != most) tries *= 2 * dims[i].count - 1;
  const Dim along = dims[most];
  if (tries > (1 << 16) || along.stride == 0 || along.stride < length) return false;
  dims[most] = {1, 0};
  for (int64_t t = 0; t < (int64_t)tries; ++t) {
    __int128 at = 0;
    int64_t rest = t;
    bool same = true;
    for (const Dim& d : dims) {
      const int64_t by = rest % (2 * d.count - 1) - (d.count - 1);
      rest /= 2 * d.count - 1;
      at += (__int128)by * d.stride;
      same = same && by == 0;
    }
    if (same) continue;  // along one dimension: a stride of `length` or more
    const __int128 m = -at / along.stride;
    for (__int128 x = m - 1; x <= m + 1; ++x) {
      const __int128 gap = at + x * along.stride;
      if (x > -along.count && x < along.count && gap < length && gap > -length) return false;
    }
  }
  return true;
}

// The checks that both calls share; a plan without rows is a call without work.
int row_plan(const lkv_kv_rows* rows, const void* k, const void* v, int dtype, int64_t seq_stride, int64_t head_stride,
             int64_t token_stride, int n_seqs, int n_kv, int head_dim, int tokens, RowPlan& p) {
  LKV_CHECK_ARG(rows && k && v, "NULL pointer");
  LKV_CHECK_ARG(dtype == LKV_F16 || dtype == LKV_BF16, "rows are float16 or bfloat16, got dtype %d", dtype);
  LKV_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d unsupported (64 or 128)", head_dim);
  LKV_CHECK_ARG(n_seqs >= 0 && n_kv > 0 && tokens >= 0, "bad shape: %d sequences, %d heads, %d tokens", n_seqs, n_kv, tokens);
  if (int rc = lkv_check_rows(rows, "rows", n_seqs, dtype, head_dim)) return rc;
  LKV_CHECK_ARG((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "keys and values must start on 16 bytes");
  LKV_CHECK_ARG(seq_stride % 8 == 0 && head_stride % 8 == 0 && token_stride % 8 == 0, "strides must be multiples of 8 elements");
  const int64_t n = (int64_t)n_seqs * n_kv * tokens;
  LKV_CHECK_ARG(n <= (1LL << 31) - 1, "%lld rows in one call", (long long)n);
  p = {rows->seq_stride, rows->head_stride, seq_stride, head_stride, token_stride, rows->tokens, n_kv, tokens, 0, (uint32_t)n, nullptr};
  return LKV_OK;
}

}  // namespace

// Two rows that are written must not share an address. Strides and head_dim are in elements of `bytes` bytes.
int lkv_distinct_rows(const char* what, const void* k, const void* v, int bytes, int n_seqs, int n_kv, int64_t tokens, int head_dim, int64_t seq_stride,
                  int64_t head_stride, int64_t token_stride) {
  const int64_t apart = (int64_t)((uintptr_t)v - (uintptr_t)k);
  Dim dims[4] = {{v ? 2 : 1, apart}, {n_seqs, seq_stride * bytes}, {n_kv, head_stride * bytes}, {tokens, token_stride * bytes}};
  if (token_stride == head_dim) dims[3] = {1, 0};
  LKV_CHECK_ARG(rows_apart(dims, (token_stride == head_dim ? tokens : 1) * head_dim * bytes), "%s: rows that are written share an address", what);
  return LKV_OK;
}

int lkv_distinct_dst(const lkv_kv_rows* dst, int n_kv, int head_dim) {
  const int es = dst->dtype == LKV_MXFP8 ? 1 : 2;
  if (int rc = lkv_distinct_rows("dst", dst->k, dst->v, es, dst->seqs, n_kv, dst->tokens, head_dim, dst->seq_stride, dst->head_stride, head_dim)) return rc;
  if (es == 2) return LKV_OK;
  return lkv_distinct_rows("dst's scales", dst->k_scale, dst->v_scale, 1, dst->seqs, n_kv, dst->tokens, head_dim / kMxGroup, dst->seq_stride / kMxGroup,
                           dst->head_stride / kMxGroup, head_dim / kMxGroup);
}

extern "C" int lkv_append_rows(uintptr_t stream, const lkv_kv_rows* dst, const void* k, const void* v, int dtype, int64_t seq_stride,
                               int64_t head_stride, int64_t token_stride, int n_seqs, int n_kv, int head_dim, int tokens,
                               const int32_t* starts, int start) {
  RowPlan p;
  if (int rc = row_plan(dst, k, v, dtype, seq_stride, head_stride, token_stride, n_seqs, n_kv, head_dim, tokens, p)) return rc;
  if (!starts) LKV_CHECK_ARG(start >= 0 && (int64_t)start + tokens <= dst->tokens, "rows %d..%lld exceed the %lld there are", start,
                             (long long)start + tokens, (long long)dst->tokens);
  if (p.rows == 0) return LKV_OK;
  if (int rc = lkv_distinct_dst(dst, n_kv, head_dim)) return rc;
  p.start = start;
  p.starts = starts;
  const bool mx = dst->dtype == LKV_MXFP8, half = dtype == LKV_F16, wide = head_dim == 128;
  auto kernel = mx ? (half ? (wide ? append_rows_kernel<LKV_F16, 128, true> : append_rows_kernel<LKV_F16, 64, true>)
                           : (wide ? append_rows_kernel<LKV_BF16, 128, true> : append_rows_kernel<LKV_BF16, 64, true>))
                   : (wide ? append_rows_kernel<LKV_BF16, 128, false> : append_rows_kernel<LKV_BF16, 64, false>);
  const uint32_t per = 256 / (head_dim / 8);
  hipLaunchKernelGGL(kernel, dim3((p.rows + per - 1) / per), dim3(256), 0, (hipStream_t)stream, p, (const uint16_t*)k,
                     (const uint16_t*)v, (uint8_t*)dst->k, (uint8_t*)dst->v, (uint8_t*)dst->k_scale, (uint8_t*)dst->v_scale);
  LKV_CHECK_LAUNCH("append_rows");
  return LKV_OK;
}

extern "C" int lkv_read_rows(uintptr_t stream, const lkv_kv_rows* src, int n_seqs, int n_kv, int head_dim, int first, int tokens, void* k,
                             void* v, int dtype, int64_t seq_stride, int64_t head_stride, int64_t token_stride) {
  RowPlan p;
  if (int rc = row_plan(src, k, v, dtype, seq_stride, head_stride, token_stride, n_seqs, n_kv, head_dim, tokens, p)) return rc;
  LKV_CHECK_ARG(src->dtype == LKV_MXFP8, "rows in the model dtype are read where they are");
  LKV_CHECK_ARG(first >= 0 && (int64_t)first + tokens <= src->tokens, "rows %d..%lld exceed the %lld there are", first,
                (long long)first + tokens, (long long)src->tokens);
  if (p.rows == 0) return LKV_OK;
  if (int rc = lkv_distinct_rows("out", k, v, 2, n_seqs, n_kv, tokens, head_dim, seq_stride, head_stride, token_stride)) return rc;
  p.start = first;
  const bool half = dtype == LKV_F16, wide = head_dim == 128;
  auto kernel = half ? (wide ? read_rows_kernel<LKV_F16, 128> : read_rows_kernel<LKV_F16, 64>)
                     : (wide ? read_rows_kernel<LKV_BF16, 128> : read_rows_kernel<LKV_BF16, 64>);
  const uint32_t per = 256 / (head_dim / 8);
  hipLaunchKernelGGL(kernel, dim3((p.rows + per - 1) / per), dim3(256), 0, (hipStream_t)stream, p, (const uint8_t*)src->k,
                     (const uint8_t*)src->v, src->k_scale, src->v_scale, (uint16_t*)k, (uint16_t*)v);
  LKV_CHECK_LAUNCH("read_rows");
  return LKV_OK;
}
