// Rows over a budget evicted by the sums of the weights that they got (lkv_evict_rows).
//
// Which rows stay is a whole-number matter: a row's rank is its sum as an unsigned number of the same order, one above all others for the first
// and newest tokens' rows, and the keep-th largest rank is found digit by digit. A kept row moves only if it lies behind row keep - 1, to a
// row before it that is not kept: every source is behind every destination, so that rows move in any order and at once, and no more of them
// than must. What a row holds is told by its position, not by its place.
#include "lkv_pages.h"

namespace {

using namespace lkv;

struct EvictArgs {
  PagedRows rows;
  const int32_t* lengths;
  const float* sums;
  const int32_t* positions;
  float* sums_out;
  int32_t* positions_out;
  int64_t sums_stride[2], positions_stride[2], sums_out_stride[2], positions_out_stride[2];
  int32_t* count;  // [sequences * KV heads]: rows that move
  int32_t* list;   // [sequences * KV heads][2][moves]: where to, and from where
  int32_t n_seqs, n_kv, keep, sinks, recent, tokens, max_tokens, moves;
};

__device__ __forceinline__ int length_of(const EvictArgs& a, int b) {
  const int64_t n = (int64_t)a.tokens + (a.lengths ? a.lengths[b] : 0);
  return (int)(n < 0 ? 0 : (n > a.max_tokens ? a.max_tokens : n));
}

// A row's rank: larger sums have larger ones, NaN has none.
__device__ __forceinline__ uint32_t rank_of(const EvictArgs& a, float sum, int position, int64_t newest) {
  if (position < a.sinks || position > newest - a.recent) return ~0u;
  if (!(sum == sum)) return 0;
  const uint32_t u = float_to_bits(sum + 0.0f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kThreads = 1024;
constexpr int kEach = 4;  // neighbouring rows of a thread in a step

// The sum of x over the threads before this one, and over all in `total`.
__device__ __forceinline__ uint32_t block_before(uint32_t x, uint32_t* lds, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t up_to = wave_inclusive_sum(x);
  __syncthreads();
  if (lane == 63) lds[wave] = up_to;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    const uint32_t y = lds[i];
    before += i < wave ? y : 0;
    total += y;
  }
  return before + up_to - x;
}

// One workgroup a KV head.
__global__ __launch_bounds__(kThreads) void evict_plan_kernel(EvictArgs a) {
  __shared__ uint32_t digits[256];
  __shared__ uint32_t sums[kThreads / 64];
  __shared__ uint32_t found[2];
  const int bh = blockIdx.x, b = bh / a.n_kv, h = bh % a.n_kv, n = length_of(a, b);
  const float* sum = a.sums + b * a.sums_stride[0] + h * a.sums_stride[1];
  const int32_t* position = a.positions + b * a.positions_stride[0] + h * a.positions_stride[1];
  float* sum_out = a.sums_out + b * a.sums_out_stride[0] + h * a.sums_out_stride[1];
  int32_t* position_out = a.positions_out + b * a.positions_out_stride[0] + h * a.positions_out_stride[1];
  const bool copies = sum != sum_out || position != position_out;
  if (n <= a.keep) {  // all stay
    if (threadIdx.x == 0) a.count[bh] = 0;
    if (copies)
      for (int i = threadIdx.x; i < n; i += kThreads) {
        sum_out[i] = sum[i];
        position_out[i] = position[i];
      }
    return;
  }
  int most = INT32_MIN;
  for (int i = threadIdx.x; i < n; i += kThreads) most = max(most, position[i]);
  if (threadIdx.x == 0) found[0] = 0;
  __syncthreads();
  atomicMax(&found[0], (uint32_t)most ^ 0x80000000u);
  __syncthreads();
  const int64_t newest = (int32_t)(found[0] ^ 0x80000000u);
  uint32_t prefix = 0, wanted = (uint32_t)a.keep;  // of the ranks that start with the prefix's digits, the wanted-th largest
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) digits[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t r = rank_of(a, sum[i], position[i], newest);
      if (shift == 24 || r >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&digits[r >> shift & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
      // Four digits a lane, the largest first.
      uint32_t of[4], all = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        of[i] = digits[255 - 4 * threadIdx.x - i];
        all += of[i];
      }
      uint32_t before = wave_inclusive_sum(all) - all;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < wanted && wanted <= before + of[i]) {
          found[0] = prefix | (uint32_t)(255 - 4 * threadIdx.x - i) << shift;
          found[1] = wanted - before;
        }
        before += of[i];
      }
    }
    __syncthreads();
    prefix = found[0];
    wanted = found[1];
    __syncthreads();
  }
  // Ranks above `prefix` stay, and of those equal to it the first `wanted`.
  uint32_t ties = 0, holes = 0, movers = 0;
  int32_t* to = a.list + (int64_t)bh * 2 * a.moves;
  int32_t* from = to + a.moves;
  for (int64_t i0 = 0; i0 < n; i0 += kThreads * kEach) {
    const int64_t first = i0 + threadIdx.x * kEach;
    uint32_t r[kEach], equal = 0;
    float s[kEach];
    int at[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int64_t i = first + j;
      s[j] = i < n ? sum[i] : 0.0f;
      at[j] = i < n ? position[i] : 0;
      r[j] = i < n ? rank_of(a, s[j], at[j], newest) : 0;
      equal += i < n && r[j] == prefix ? 1 : 0;
    }
    uint32_t total;
    uint32_t tie = ties + block_before(equal, sums, total);
    ties += total;
    bool kept[kEach];
    uint32_t mine = 0;  // holes in the low half, movers in the high one
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int64_t i = first + j;
      kept[j] = i < n && (r[j] > prefix || (r[j] == prefix && tie < wanted));
      tie += i < n && r[j] == prefix ? 1 : 0;
      mine += i < a.keep && !kept[j] ? 1u : i >= a.keep && kept[j] ? 1u << 16 : 0u;
    }
    const uint32_t before = block_before(mine, sums, total);
    uint32_t hole = holes + (before & 0xffffu), mover = movers + (before >> 16);
    holes += total & 0xffffu;
    movers += total >> 16;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int64_t i = first + j;
      if (i < a.keep) {
        if (!kept[j]) {
          to[hole++] = (int32_t)i;
        } else if (copies) {
          sum_out[i] = s[j];
          position_out[i] = at[j];
        }
      } else if (kept[j]) {
        from[mover++] = (int32_t)i;
      }
    }
  }
  if (threadIdx.x == 0) a.count[bh] = (int32_t)movers;
}

// Sixteen lanes (head_dim 128) or eight move a row's keys and values.
template <int D, bool MX>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
  constexpr int LPR = D / 8;
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, b = bh / a.n_kv, h = bh % a.n_kv;
  const int move = blockIdx.x / heads * (256 / LPR) + threadIdx.x / LPR, c = threadIdx.x % LPR * 8;
  if (move >= a.count[bh]) return;
  const int32_t* list = a.list + (int64_t)bh * 2 * a.moves;
  const int to = list[move], from = list[a.moves + move];
  if (c == 0) {
    a.sums_out[b * a.sums_out_stride[0] + h * a.sums_out_stride[1] + to] = a.sums[b * a.sums_stride[0] + h * a.sums_stride[1] + from];
    a.positions_out[b * a.positions_out_stride[0] + h * a.positions_out_stride[1] + to] = a.positions[b * a.positions_stride[0] + h * a.positions_stride[1] + from];
  }
  const int64_t dst = row_of<D>(a.rows, b, h, to), src = row_of<D>(a.rows, b, h, from);
  if (dst < 0 || src < 0) return;
  if constexpr (MX) {
    uint8_t *k = (uint8_t*)a.rows.rows.k, *v = (uint8_t*)a.rows.rows.v;
    const uint2 x = *(const uint2*)(k + src + c), y = *(const uint2*)(v + src + c);
    *(uint2*)(k + dst + c) = x;
    *(uint2*)(v + dst + c) = y;
    if ((threadIdx.x & 3) == 0) {
      ((uint8_t*)a.rows.rows.k_scale)[(dst + c) / kMxGroup] = a.rows.rows.k_scale[(src + c) / kMxGroup];
      ((uint8_t*)a.rows.rows.v_scale)[(dst + c) / kMxGroup] = a.rows.rows.v_scale[(src + c) / kMxGroup];
    }
  } else {
    uint16_t *k = (uint16_t*)a.rows.rows.k, *v = (uint16_t*)a.rows.rows.v;
    const uint4 x = *(const uint4*)(k + src + c), y = *(const uint4*)(v + src + c);
    *(uint4*)(k + dst + c) = x;
    *(uint4*)(v + dst + c) = y;
  }
}

int check_evict(const lkv_evict_desc* d) {
  LKV_CHECK_ARG(d, "NULL pointer");
  LKV_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "head_dim %d unsupported (64 or 128)", d->head_dim);
  LKV_CHECK_ARG(d->dtype == LKV_F16 || d->dtype == LKV_BF16, "rows are float16 or bfloat16, got dtype %d", d->dtype);
  LKV_CHECK_ARG(d->n_seqs >= 0 && d->n_kv > 0, "bad shape: %d sequences, %d heads", d->n_seqs, d->n_kv);
  LKV_CHECK_ARG(d->tokens >= 0 && d->max_tokens >= 0 && d->max_tokens <= (1 << 30), "bad extent: %d rows of at most %d", d->tokens, d->max_tokens);
  LKV_CHECK_ARG(d->keep > 0 && d->sinks >= 0 && d->recent >= 0 && (int64_t)d->sinks + d->recent <= d->keep, "%d first and %d newest of %d rows that are kept", d->sinks,
                d->recent, d->keep);
  return LKV_OK;
}

// The most rows that a head can move: those kept behind `keep`, and those there is a place for.
int moves_of(const lkv_evict_desc* d) {
  const int over = d->max_tokens - d->keep;
  return over <= 0 ? 0 : over < d->keep ? over : d->keep;
}

}  // namespace

extern "C" size_t lkv_evict_rows_workspace_bytes(const lkv_evict_desc* desc) {
  if (check_evict(desc)) return 0;
  const size_t heads = (size_t)desc->n_seqs * desc->n_kv;
  return lkv_align_up(heads * sizeof(int32_t), 16) + heads * 2 * moves_of(desc) * sizeof(int32_t);
}

extern "C" int lkv_evict_rows(uintptr_t stream, const lkv_evict_desc* desc, const lkv_kv_rows* rows, const lkv_pages* pages, const int32_t* lengths, const float* sums,
                              const int64_t* sums_stride, const int32_t* positions, const int64_t* positions_stride, float* sums_out,
                              const int64_t* sums_out_stride, int32_t* positions_out, const int64_t* positions_out_stride, void* ws, size_t ws_bytes) {
  if (int rc = check_evict(desc)) return rc;
  LKV_CHECK_ARG(sums && sums_stride && positions && positions_stride && sums_out && sums_out_stride && positions_out && positions_out_stride, "NULL pointer");
  EvictArgs a = {};
  if (int rc = lkv_paged_rows(rows, pages, desc->n_seqs, desc->dtype, desc->head_dim, a.rows)) return rc;
  LKV_CHECK_ARG(desc->max_tokens <= a.rows.capacity, "%d rows of a sequence over %d", desc->max_tokens, a.rows.capacity);
  const size_t need = lkv_evict_rows_workspace_bytes(desc);
  LKV_CHECK_ARG(ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0, "workspace of %zu bytes, on 16: %zu are needed", ws_bytes, need);
  const int64_t heads = (int64_t)desc->n_seqs * desc->n_kv;
  a.moves = moves_of(desc);
  const int64_t per = 256 / (desc->head_dim / 8), blocks = heads * ((a.moves + per - 1) / per);
  LKV_CHECK_ARG(heads < (1LL << 31) && blocks < (1LL << 31), "%lld workgroups in one call", (long long)blocks);
  if (heads == 0 || desc->max_tokens == 0) return LKV_OK;
  if (int rc = lkv_distinct_dst(rows, desc->n_kv, desc->head_dim)) return rc;
  a.lengths = lengths;
  a.sums = sums;
  a.positions = positions;
  a.sums_out = sums_out;
  a.positions_out = positions_out;
  for (int i = 0; i < 2; ++i) {
    a.sums_stride[i] = sums_stride[i];
    a.positions_stride[i] = positions_stride[i];
    a.sums_out_stride[i] = sums_out_stride[i];
    a.positions_out_stride[i] = positions_out_stride[i];
  }
  a.count = (int32_t*)ws;
  a.list = (int32_t*)((uint8_t*)ws + lkv_align_up(heads * sizeof(int32_t), 16));
  a.n_seqs = desc->n_seqs;
  a.n_kv = desc->n_kv;
  a.keep = desc->keep;
  a.sinks = desc->sinks;
  a.recent = desc->recent;
  a.tokens = desc->tokens;
  a.max_tokens = desc->max_tokens;
  const hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(evict_plan_kernel, dim3((unsigned)heads), dim3(kThreads), 0, s, a);
  LKV_CHECK_LAUNCH("evict_rows (plan)");
  if (blocks > 0) {
    const bool mx = rows->dtype == LKV_MXFP8, wide = desc->head_dim == 128;
    auto kernel = wide ? (mx ? evict_move_kernel<128, true> : evict_move_kernel<128, false>) : (mx ? evict_move_kernel<64, true> : evict_move_kernel<64, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
    LKV_CHECK_LAUNCH("evict_rows");
  }
  return LKV_OK;
}
