// Rows over a budget evicted by the sums of the weights that they got (lkv_evict_rows).
//
// Which rows stay is a whole-number matter: a row's rank is its sum as an unsigned number of the same order, one above all others for the first
// and newest tokens' rows, and the keep-th largest rank is found digit by digit. A kept row moves only if it lies behind row keep - 1, to a
// row before it that is not kept: every source is behind every destination, so that rows move in any order and at once, and no more of them
// than must. What a row holds is told by its position, not by its place.
//
// The moves are bound by memory: 131,072 rows of 8 heads (d 128) cut to 32,768 take 43 us, 4.6 TB/s of rows that are read one by one, and the planning before it another
// 43, six launches whose ends are most of that. A decode step's one row over 2,048, of sixteen sequences: 9.5 us, one launch's latency from length to move.
#include "lkv_pages.h"

namespace {

using namespace lkv;

// Of the rows whose ranks begin with these digits, how many are wanted.
struct Wanted {
  uint32_t prefix, left;
};

struct EvictArgs {
  PagedRows rows;
  const int32_t* lengths;
  const float* sums;
  const int32_t* positions;
  float* sums_out;
  int32_t* positions_out;
  int64_t sums_stride[2], positions_stride[2], sums_out_stride[2], positions_out_stride[2];
  int32_t* count;      // [sequences * KV heads]: rows that move
  int32_t* list;       // [sequences * KV heads][2][moves]: where to, and from where
  int32_t* newest;     // [sequences * KV heads][spans]: largest positions
  uint32_t* digits;    // [sequences * KV heads][3][kDigits]: how many rows have each digit
  Wanted* wanted;      // [sequences * KV heads][3]: after each of them
  uint32_t* split;     // [sequences * KV heads][spans][4]: see Split
  int32_t n_seqs, n_kv, keep, sinks, recent, tokens, max_tokens, moves;
  int32_t spans;       // of a head's rows, kSpan each
};

__device__ __forceinline__ int length_of(const EvictArgs& a, int b) {
  const int64_t n = (int64_t)a.tokens + (a.lengths ? a.lengths[b] : 0);
  return (int)(n < 0 ? 0 : (n > a.max_tokens ? a.max_tokens : n));
}

// A row's rank: larger sums have larger ones, NaN has none.
__device__ __forceinline__ uint32_t rank_of(const EvictArgs& a, float sum, int position, int newest) {
  if (position < a.sinks || (int64_t)position > (int64_t)newest - a.recent) return ~0u;
  if (!(sum == sum)) return 0;
  const uint32_t u = float_to_bits(sum + 0.0f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kThreads = 1024, kWaves = kThreads / 64;
// A rank is found in three digits of 11, 11 and 10 bits: an 8-bit one would put all sums of a few octaves, which have the same exponents but for a bit or
// two, on a few counters.
constexpr int kDigits = 2048;
__device__ __forceinline__ uint32_t digit_of(uint32_t rank, int place) { return place == 0 ? rank >> 21 : place == 1 ? rank >> 10 & 2047 : rank & 1023; }
__device__ __forceinline__ bool starts_with(uint32_t rank, uint32_t prefix, int places) { return places == 0 || (places == 1 ? (rank ^ prefix) >> 21 == 0 : (rank ^ prefix) >> 10 == 0); }

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
  for (int i = 0; i < kWaves; ++i) {
    const uint32_t y = lds[i];
    before += i < wave ? y : 0;
    total += y;
  }
  return before + up_to - x;
}

// `digits`: LDS or memory.
__device__ __forceinline__ Wanted next_digit(const uint32_t* digits, int place, Wanted w, uint32_t* lds, Wanted* found) {
  // Two digits a thread, the largest first.
  const int d = place == 2 ? 1023 - (int)threadIdx.x : kDigits - 1 - 2 * (int)threadIdx.x;
  const uint32_t x = digits[d], y = place == 2 ? 0 : digits[d - 1];
  uint32_t total;
  const uint32_t before = block_before(x + y, lds, total);
  const int shift = place == 0 ? 21 : place == 1 ? 10 : 0;
  if (before < w.left && w.left <= before + x) *found = {w.prefix | (uint32_t)d << shift, w.left - before};
  if (before + x < w.left && w.left <= before + x + y) *found = {w.prefix | (uint32_t)(d - 1) << shift, w.left - before - x};
  __syncthreads();
  return *found;
}

// Neighbouring rows of a workgroup, in registers: row first + 64 EACH wave + 64 j + lane in place j.
template <int EACH> struct Span {
  float sum[EACH];
  int position[EACH];
  uint32_t rank[EACH];
  int first, n;  // this lane's first row; rows that the head has
  const float* sums;
  const int32_t* positions;
  __device__ __forceinline__ void load(const EvictArgs& a, int b, int h, int span, int length) {
    sums = a.sums + b * a.sums_stride[0] + h * a.sums_stride[1];
    positions = a.positions + b * a.positions_stride[0] + h * a.positions_stride[1];
    first = span * kThreads * EACH + (int)(threadIdx.x >> 6) * 64 * EACH + (int)(threadIdx.x & 63);
    n = length;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = row(j);
      sum[j] = i < n ? sums[i] : 0.0f;
      position[j] = i < n ? positions[i] : INT32_MIN;
    }
  }
  __device__ __forceinline__ int row(int j) const { return first + 64 * j; }
  // The largest position, in all threads.
  __device__ __forceinline__ int newest(uint32_t* lds) const {
    int most = INT32_MIN;
#pragma unroll
    for (int j = 0; j < EACH; ++j) most = max(most, position[j]);
    const uint32_t wave_most = wave_max_u32((uint32_t)most ^ 0x80000000u);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = wave_most;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) all = max(all, lds[i]);
    __syncthreads();
    return (int)(all ^ 0x80000000u);
  }
  __device__ __forceinline__ void order(const EvictArgs& a, int newest) {
#pragma unroll
    for (int j = 0; j < EACH; ++j) rank[j] = rank_of(a, sum[j], position[j], newest);
  }
  __device__ __forceinline__ void count_digits(uint32_t* lds, int place, uint32_t prefix) const {
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (row(j) < n && starts_with(rank[j], prefix, place)) atomicAdd(&lds[digit_of(rank[j], place)], 1u);
  }
};

__device__ __forceinline__ void clear_digits(uint32_t* lds) {
  __syncthreads();
  lds[threadIdx.x] = lds[threadIdx.x + kThreads] = 0;
  __syncthreads();
}
__device__ __forceinline__ uint32_t lanes_before(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0)); }

// What lies before a span: rows of the last rank, holes and rows that move.
struct Before {
  uint32_t ties, holes, movers;
};

// The span's holes and moving rows to their lists, its rows that stay to where they are copied.
template <int EACH>
__device__ __forceinline__ void write_lists(const EvictArgs& a, const Span<EACH>& x, int b, int h, Wanted last, Before before, uint32_t* lds, int32_t* to, int32_t* from,
                                            uint32_t& moving) {
  float* sum_out = a.sums_out + b * a.sums_out_stride[0] + h * a.sums_out_stride[1];
  int32_t* position_out = a.positions_out + b * a.positions_out_stride[0] + h * a.positions_out_stride[1];
  const bool copies = x.sums != sum_out || x.positions != position_out;
  const int lane = threadIdx.x & 63, keep = min(a.keep, x.n);
  // Rows of the last rank in the waves before, in their order.
  uint32_t mine = 0, total;
#pragma unroll
  for (int j = 0; j < EACH; ++j) mine += __popcll(__ballot(x.row(j) < x.n && x.rank[j] == last.prefix));
  uint32_t tie = before.ties + block_before(lane == 0 ? mine : 0, lds, total);
  tie = __builtin_amdgcn_readfirstlane(tie);
  uint64_t kept[EACH];
  uint32_t holes = 0, movers = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const bool live = x.row(j) < x.n, equal = live && x.rank[j] == last.prefix;
    const uint64_t equals = __ballot(equal);
    const bool stays = live && (x.rank[j] > last.prefix || (equal && tie + lanes_before(equals) < last.left));
    tie += __popcll(equals);
    kept[j] = __ballot(stays);
    const uint64_t front = __ballot(x.row(j) < keep);
    holes += __popcll(front & ~kept[j]);
    movers += __popcll(kept[j] & ~front);
  }
  // The two counts in one sum: a span has less than 2^16 of each.
  const uint32_t wave_before = __builtin_amdgcn_readfirstlane(block_before(lane == 0 ? holes | movers << 16 : 0, lds, total));
  uint32_t hole = before.holes + (wave_before & 0xffffu), mover = before.movers + (wave_before >> 16);
  moving = before.movers + (total >> 16);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = x.row(j);
    const uint64_t front = __ballot(i < keep), empty = front & ~kept[j], moves = kept[j] & ~front;
    const bool stays = kept[j] >> lane & 1;
    if (i < keep) {
      if (!stays) {
        to[hole + lanes_before(empty)] = i;
      } else if (copies) {
        sum_out[i] = x.sum[j];
        position_out[i] = x.position[j];
      }
    } else if (stays) {
      from[mover + lanes_before(moves)] = i;
    }
    hole += __popcll(empty);
    mover += __popcll(moves);
  }
}

// A row from one place to another: D / 8 lanes, 8 channels each.
template <int D, bool MX>
__device__ __forceinline__ void move_row(const EvictArgs& a, int b, int h, int from, int to, int c) {
  if (c == 0) {
    a.sums_out[b * a.sums_out_stride[0] + h * a.sums_out_stride[1] + to] = a.sums[b * a.sums_stride[0] + h * a.sums_stride[1] + from];
    a.positions_out[b * a.positions_out_stride[0] + h * a.positions_out_stride[1] + to] = a.positions[b * a.positions_stride[0] + h * a.positions_stride[1] + from];
  }
  const int64_t dst = row_of<D>(a.rows, b, h, to), src = row_of<D>(a.rows, b, h, from);
  if (dst < 0 || src < 0) return;
  if constexpr (MX) {
    uint8_t *k = (uint8_t*)a.rows.rows.k, *v = (uint8_t*)a.rows.rows.v, *ks = (uint8_t*)a.rows.rows.k_scale, *vs = (uint8_t*)a.rows.rows.v_scale;
    const uint2 x = *(const uint2*)(k + src + c), y = *(const uint2*)(v + src + c);
    *(uint2*)(k + dst + c) = x;
    *(uint2*)(v + dst + c) = y;
    if (c % kMxGroup == 0) {
      ks[(dst + c) / kMxGroup] = ks[(src + c) / kMxGroup];
      vs[(dst + c) / kMxGroup] = vs[(src + c) / kMxGroup];
    }
  } else {
    uint16_t *k = (uint16_t*)a.rows.rows.k, *v = (uint16_t*)a.rows.rows.v;
    const uint4 x = *(const uint4*)(k + src + c), y = *(const uint4*)(v + src + c);
    *(uint4*)(k + dst + c) = x;
    *(uint4*)(v + dst + c) = y;
  }
}

constexpr int kFew = 256;  // moves that the planning workgroup makes by itself

// A head's rows in one workgroup's registers. Where a head can move few rows, as when a decode step is over its budget by one, they are moved here.
template <int EACH, int D, bool MX, bool MOVES>
__global__ __launch_bounds__(kThreads) void evict_short_kernel(EvictArgs a) {
  __shared__ uint32_t digits[kDigits];
  __shared__ uint32_t sums[kWaves];
  __shared__ Wanted found;
  __shared__ int32_t few[2][kFew];
  const int bh = blockIdx.x, b = bh / a.n_kv, h = bh % a.n_kv, n = length_of(a, b);
  Span<EACH> x;
  x.load(a, b, h, 0, n);
  x.order(a, x.newest(sums));
  Wanted last = {0, (uint32_t)a.keep};  // where all rows stay: every rank is at least 0, and as many ties stay as there can be
  if (n > a.keep) {
    for (int place = 0; place < 3; ++place) {
      clear_digits(digits);
      x.count_digits(digits, place, last.prefix);
      __syncthreads();
      last = next_digit(digits, place, last, sums, &found);
    }
  }
  int32_t* to = MOVES ? few[0] : a.list + (int64_t)bh * 2 * a.moves;
  uint32_t moving;
  write_lists<EACH>(a, x, b, h, last, {0, 0, 0}, sums, to, MOVES ? few[1] : to + a.moves, moving);
  if constexpr (MOVES) {
    __syncthreads();
    for (uint32_t i = threadIdx.x / (D / 8); i < moving; i += kThreads / (D / 8)) move_row<D, MX>(a, b, h, few[1][i], few[0][i], threadIdx.x % (D / 8) * 8);
  } else {
    if (threadIdx.x == 0) a.count[bh] = (int32_t)moving;
  }
}

// ---- long caches: a head's rows in spans of a workgroup each, a launch for each step ---------------------
// The steps' counts are whole numbers added in memory: their order changes nothing. Four rows a thread: 131,072 rows of eight heads are 256 workgroups, one a
// CU, 86.1 us with the move; eight rows 94.0, two (twice the counters to add) 88.4.
constexpr int kEach = 4, kSpan = kThreads * kEach;

__global__ __launch_bounds__(kThreads) void evict_newest_kernel(EvictArgs a) {
  __shared__ uint32_t lds[kWaves];
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, span = blockIdx.x / heads, b = bh / a.n_kv, h = bh % a.n_kv;
  Span<kEach> x;
  x.load(a, b, h, span, length_of(a, b));
  const int newest = x.newest(lds);
  if (threadIdx.x == 0) a.newest[(int64_t)bh * a.spans + span] = newest;
  if (span == 0)
    for (int i = threadIdx.x; i < 3 * kDigits; i += kThreads) a.digits[(int64_t)bh * 3 * kDigits + i] = 0;
}

template <int EACH>
__device__ __forceinline__ void load_ranks(const EvictArgs& a, Span<EACH>& x, int bh, int span, int n) {
  x.load(a, bh / a.n_kv, bh % a.n_kv, span, n);
  int newest = INT32_MIN;
  for (int i = threadIdx.x & 63; i < a.spans; i += 64) newest = max(newest, a.newest[(int64_t)bh * a.spans + i]);
  x.order(a, (int)(wave_max_u32((uint32_t)newest ^ 0x80000000u) ^ 0x80000000u));
}

// The rank's first `places` digits, of which the steps before left all but the last; the first span leaves them for the next step.
__device__ __forceinline__ Wanted found_digits(const EvictArgs& a, int bh, int span, int places, uint32_t* lds, Wanted* found) {
  if (places == 0) return {0, (uint32_t)a.keep};
  Wanted* steps = a.wanted + (int64_t)bh * 3;
  const Wanted w = next_digit(a.digits + ((int64_t)bh * 3 + places - 1) * kDigits, places - 1, places == 1 ? Wanted{0, (uint32_t)a.keep} : steps[places - 2], lds, found);
  if (span == 0 && threadIdx.x == 0) steps[places - 1] = w;
  return w;
}

__global__ __launch_bounds__(kThreads) void evict_digit_kernel(EvictArgs a, int place) {
  __shared__ uint32_t digits[kDigits];
  __shared__ uint32_t lds[kWaves];
  __shared__ Wanted found;
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, span = blockIdx.x / heads, n = length_of(a, bh / a.n_kv);
  if (n <= a.keep || (int64_t)span * kSpan >= n) return;
  Span<kEach> x;
  load_ranks(a, x, bh, span, n);
  const Wanted w = found_digits(a, bh, span, place, lds, &found);
  clear_digits(digits);
  x.count_digits(digits, place, w.prefix);
  __syncthreads();
  uint32_t* all = a.digits + ((int64_t)bh * 3 + place) * kDigits;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t y = digits[threadIdx.x + i * kThreads];
    if (y) atomicAdd(&all[threadIdx.x + i * kThreads], y);
  }
}

// Of a span's rows: those of the last rank before row `keep`, all of them, and those above it, before row `keep` and all.
struct Split {
  uint32_t front_equal, equal, front_above, above;
};

__global__ __launch_bounds__(kThreads) void evict_split_kernel(EvictArgs a) {
  __shared__ uint32_t lds[kWaves];
  __shared__ Wanted found;
  __shared__ uint32_t counts[4];
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, span = blockIdx.x / heads, n = length_of(a, bh / a.n_kv);
  if (n <= a.keep || (int64_t)span * kSpan >= n) return;
  Span<kEach> x;
  load_ranks(a, x, bh, span, n);
  if (threadIdx.x < 4) counts[threadIdx.x] = 0;
  const Wanted last = found_digits(a, bh, span, 3, lds, &found);
  uint32_t c[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const bool live = x.row(j) < n;
    const uint64_t front = __ballot(x.row(j) < a.keep), equal = __ballot(live && x.rank[j] == last.prefix), above = __ballot(live && x.rank[j] > last.prefix);
    c[0] += __popcll(front & equal);
    c[1] += __popcll(equal);
    c[2] += __popcll(front & above);
    c[3] += __popcll(above);
  }
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) atomicAdd(&counts[i], c[i]);
  __syncthreads();
  if (threadIdx.x < 4) a.split[((int64_t)bh * a.spans + span) * 4 + threadIdx.x] = counts[threadIdx.x];
}

__global__ __launch_bounds__(kThreads) void evict_list_kernel(EvictArgs a) {
  __shared__ uint32_t lds[kWaves];
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, span = blockIdx.x / heads, b = bh / a.n_kv, n = length_of(a, b);
  if (span == 0 && threadIdx.x == 0 && n <= a.keep) a.count[bh] = 0;
  if ((int64_t)span * kSpan >= n) return;
  Span<kEach> x;
  load_ranks(a, x, bh, span, n);
  Wanted last = {0, (uint32_t)a.keep};
  uint32_t c[4] = {0, 0, 0, 0}, all_front_equal = 0;
  if (n > a.keep) {
    last = a.wanted[(int64_t)bh * 3 + 2];
    const int spans = (n + kSpan - 1) / kSpan;
    for (int i = threadIdx.x & 63; i < spans; i += 64) {
      const uint4 y = *(const uint4*)(a.split + ((int64_t)bh * a.spans + i) * 4);
      all_front_equal += y.x;
      if (i < span) c[0] += y.x, c[1] += y.y, c[2] += y.z, c[3] += y.w;
    }
    all_front_equal = __shfl(wave_inclusive_sum(all_front_equal), 63);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __shfl(wave_inclusive_sum(c[i]), 63);
  }
  // Rows of the last rank stay in their order, those before row `keep` first.
  const uint32_t front_rows = (uint32_t)min((int64_t)span * kSpan, (int64_t)a.keep);
  const uint32_t stay_front = min(all_front_equal, last.left), back_equal = c[1] - c[0];
  const Before before = {c[1], front_rows - c[2] - min(c[0], last.left), c[3] - c[2] + min(back_equal, last.left - stay_front)};
  int32_t* to = a.list + (int64_t)bh * 2 * a.moves;
  uint32_t moving;
  write_lists<kEach>(a, x, b, bh % a.n_kv, last, before, lds, to, to + a.moves, moving);
  if (n > a.keep && (int64_t)(span + 1) * kSpan >= n && threadIdx.x == 0) a.count[bh] = (int32_t)moving;
}

// Sixteen lanes (head_dim 128) or eight move a row's keys and values.
template <int D, bool MX>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
  constexpr int LPR = D / 8;
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, b = bh / a.n_kv, h = bh % a.n_kv;
  const int move = blockIdx.x / heads * (256 / LPR) + threadIdx.x / LPR, c = threadIdx.x % LPR * 8;
  if (move >= a.count[bh]) return;
  const int32_t* list = a.list + (int64_t)bh * 2 * a.moves;
  move_row<D, MX>(a, b, h, list[a.moves + move], list[move], c);
}

int check_evict(const lkv_evict_desc* d) {
  LKV_CHECK_ARG(d, "NULL pointer");
  LKV_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "head_dim %d unsupported (64 or 128)", d->head_dim);
  LKV_CHECK_ARG(d->dtype == LKV_F16 || d->dtype == LKV_BF16, "rows are float16 or bfloat16, got dtype %d", d->dtype);
  LKV_CHECK_ARG(d->n_seqs >= 0 && d->n_kv > 0, "bad shape: %d sequences, %d heads", d->n_seqs, d->n_kv);
  LKV_CHECK_ARG((int64_t)d->n_seqs * d->n_kv < (1 << 22), "%d x %d heads in one call", d->n_seqs, d->n_kv);
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

// The scratch: offsets of its parts.
struct Layout {
  int spans;  // 0: a head's rows fit one workgroup
  size_t list, newest, digits, wanted, split, bytes;
};
Layout layout_of(const lkv_evict_desc* d) {
  Layout l = {};
  const size_t heads = (size_t)d->n_seqs * d->n_kv;
  l.list = lkv_align_up(heads * sizeof(int32_t), 16);
  l.bytes = l.newest = l.list + lkv_align_up(heads * 2 * moves_of(d) * sizeof(int32_t), 16);
  // One workgroup's registers hold 16,384 rows: that many take 26.0 us (8,000 of one sequence stay), by spans 36.8; 6,000 15.0 and 31.9, 2,049 of sixteen sequences 9.5 and 30.3.
  if (d->max_tokens <= kThreads * 16) return l;
  l.spans = (int)(((int64_t)d->max_tokens + kSpan - 1) / kSpan);
  l.digits = l.newest + lkv_align_up(heads * l.spans * sizeof(int32_t), 16);
  l.wanted = l.digits + heads * 3 * kDigits * sizeof(uint32_t);
  l.split = l.wanted + lkv_align_up(heads * 3 * sizeof(Wanted), 16);
  l.bytes = l.split + heads * l.spans * sizeof(Split);
  return l;
}

template <int D, bool MX>
int launch(const EvictArgs& a, hipStream_t s, int64_t heads) {
  const dim3 block(kThreads);
  const bool few = a.spans == 0 && a.moves <= kFew;
  if (a.spans == 0) {
    // Rows a thread, no more than needed (sixteen sequences over their budget by one): 2,048 rows 8.6 us by two and 16.0 by sixteen, 2,049 9.5 by four; 6,000 of one, cut to 2,000, 15.0 by
    // eight and 19.7.
    const int each = a.max_tokens <= 2 * kThreads ? 2 : a.max_tokens <= 4 * kThreads ? 4 : a.max_tokens <= 8 * kThreads ? 8 : 16;
    auto kernel = each == 2   ? (few ? evict_short_kernel<2, D, MX, true> : evict_short_kernel<2, D, MX, false>)
                  : each == 4 ? (few ? evict_short_kernel<4, D, MX, true> : evict_short_kernel<4, D, MX, false>)
                  : each == 8 ? (few ? evict_short_kernel<8, D, MX, true> : evict_short_kernel<8, D, MX, false>)
                              : (few ? evict_short_kernel<16, D, MX, true> : evict_short_kernel<16, D, MX, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)heads), block, 0, s, a);
    LKV_CHECK_LAUNCH("evict_rows (plan)");
  } else {
    const dim3 grid((unsigned)(heads * a.spans));
    hipLaunchKernelGGL(evict_newest_kernel, grid, block, 0, s, a);
    for (int place = 0; place < 3; ++place) hipLaunchKernelGGL(evict_digit_kernel, grid, block, 0, s, a, place);
    hipLaunchKernelGGL(evict_split_kernel, grid, block, 0, s, a);
    hipLaunchKernelGGL(evict_list_kernel, grid, block, 0, s, a);
    LKV_CHECK_LAUNCH("evict_rows (plan)");
  }
  if (few || a.moves == 0) return LKV_OK;
  const int64_t per = 256 / (D / 8);
  hipLaunchKernelGGL((evict_move_kernel<D, MX>), dim3((unsigned)(heads * ((a.moves + per - 1) / per))), dim3(256), 0, s, a);
  LKV_CHECK_LAUNCH("evict_rows");
  return LKV_OK;
}

}  // namespace

extern "C" size_t lkv_evict_rows_workspace_bytes(const lkv_evict_desc* desc) {
  if (check_evict(desc)) return 0;
  return layout_of(desc).bytes;
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
  const Layout l = layout_of(desc);
  a.moves = moves_of(desc);
  a.spans = l.spans;
  const int64_t per = 256 / (desc->head_dim / 8), moving = (a.moves + per - 1) / per, planning = heads * (l.spans ? l.spans : 1);
  LKV_CHECK_ARG(planning < (1 << 22) && heads * moving < (1 << 24), "%lld and %lld workgroups in one call", (long long)planning, (long long)(heads * moving));
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
  uint8_t* const at = (uint8_t*)ws;
  a.count = (int32_t*)at;
  a.list = (int32_t*)(at + l.list);
  a.newest = (int32_t*)(at + l.newest);
  a.digits = (uint32_t*)(at + l.digits);
  a.wanted = (Wanted*)(at + l.wanted);
  a.split = (uint32_t*)(at + l.split);
  a.n_seqs = desc->n_seqs;
  a.n_kv = desc->n_kv;
  a.keep = desc->keep;
  a.sinks = desc->sinks;
  a.recent = desc->recent;
  a.tokens = desc->tokens;
  a.max_tokens = desc->max_tokens;
  const hipStream_t s = (hipStream_t)stream;
  const bool mx = rows->dtype == LKV_MXFP8;
  if (desc->head_dim == 128) return mx ? launch<128, true>(a, s, heads) : launch<128, false>(a, s, heads);
  return mx ? launch<64, true>(a, s, heads) : launch<64, false>(a, s, heads);
}
