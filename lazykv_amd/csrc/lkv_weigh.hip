// The weights that rows get from a chunk's tokens, summed up (lkv_weigh_rows):
//   sum_i = sum over the KV head's query heads and the tokens that attend row i of exp(scale q . k_i - lse).
//
// A wave holds 64 rows' keys as the second operand of v_mfma_f32_16x16x32 and takes the query rows 16 at a time as the first,
// S [16 queries x 16 rows] = Q K^T, so that a row's scores lie in one lane of each quarter: its sum stays there from the first query to the last.
// The accumulators start at -lse / scale, and the scores come out relative to it. That form reads the queries from memory, for up to 32 query rows of
// a KV head. More of them go through LDS, 64 at a time for four waves, on v_mfma_f32_32x32x16; there -lse is the addend of the exponent's one
// multiply-add.
//
// Bound by issue, and by products and vector operations that hardly overlap: behind each 32 x 32 x 16 product of 32 cycles, at 128 channels, the stage's loop has six vector operations, two of
// them exponentials, and some two and a half more bring a stage's queries to LDS. 1,024 tokens over 16,384 rows (32 heads on 8, d 128): 178 us, 0.75 PFLOP/s, the matrix
// units busy for 39% of the cycles, the vector units for 57%. One token over 4,099 (d 64): 4.9 us on the device, launch and latency.
#include <type_traits>

#include "lkv_attend.h"
#include "lkv_pages.h"

int lkv_check_chunk(const lkv_chunk_desc* d);  // lkv_chunk.hip

namespace {

using namespace lkv;

constexpr int kWaves = 4;
constexpr int kWaveRows = 64;
constexpr int kBlockRows = kWaves * kWaveRows;

struct WeighArgs {
  const uint16_t* q;
  const float* lse;
  PagedRows rows;
  const int32_t *lengths, *counts, *seen;
  const float* sums;
  float* out;
  int32_t* positions;
  float* part;  // [parts][sequences * KV heads][padded rows]
  int64_t q_stride[3], sums_stride[2], out_stride[2], positions_stride[2];
  float scale2, per_scale;  // scale * log2(e), 1 / scale
  int32_t n_seqs, n_q, n_kv, g, new_tokens, tokens, max_tokens;
  int32_t blocks, parts, chunk;  // of a KV head's rows; of its query rows, in ranges of `chunk`
  int32_t step_t, step_j;        // a stage of query rows further: tokens, heads of the group; and in elements
  int64_t step_at, wrap_at;      // , and from the last head of a token to the first of the next beyond a head's step
};

struct Extent {
  int len, n;
};
__device__ __forceinline__ Extent extent_of(const WeighArgs& a, int b) {
  const int64_t len = (int64_t)a.tokens + (a.lengths ? a.lengths[b] : 0);
  const int n = a.counts ? a.counts[b] : a.new_tokens;
  return {(int)(len < 0 ? 0 : (len > a.max_tokens ? a.max_tokens : len)), n < 0 ? 0 : (n > a.new_tokens ? a.new_tokens : n)};
}

// A row's sum of the call, where it belongs.
__device__ __forceinline__ void store_sum(const WeighArgs& a, const Extent& e, int b, int h, int row, float got) {
  if (row >= e.len) return;
  const int past = e.len - e.n;
  if (row < past && a.sums) got += a.sums[b * a.sums_stride[0] + h * a.sums_stride[1] + row];
  a.out[b * a.out_stride[0] + h * a.out_stride[1] + row] = got;
  if (a.positions && row >= past && row >= 0)
    a.positions[b * a.positions_stride[0] + h * a.positions_stride[1] + row] = (a.seen ? a.seen[b] : max(past, 0)) + row - past;
}

// A query row without weight, one that is not there or whose lse is -inf, attends nothing: its limit is 0. Its scores may be NaN, whatever its query is taken for, where a key
// is not finite, so that sixteen or a stage with such a row takes the form that looks at the limits.

// Sixteen query rows as the lanes hold them.
template <int D, bool MX> struct QueryRegs {
  uint4 w[D / 32];
  float start;  // -lse / scale; -inf for a row without weight
  int limit;
  __device__ __forceinline__ void load(const WeighArgs& a, const Extent& e, int b, int h, int x) {
    const int quarter = (threadIdx.x & 63) >> 4;
    const int t = x / a.g, j = h * a.g + (x - t * a.g);
    const bool live = t < e.n;
    const int tt = live ? t : 0, jj = live ? j : h * a.g;  // the first row in the place of one that is not there
    const uint16_t* q = a.q + b * a.q_stride[0] + jj * a.q_stride[1] + tt * a.q_stride[2];
    const float lse = a.lse[((int64_t)b * a.n_q + jj) * a.new_tokens + tt];
    const bool weighs = live && lse != -INFINITY;
    limit = weighs ? e.len - e.n + t + 1 : 0;
    start = weighs ? -lse * a.per_scale : -INFINITY;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) w[i] = *(const uint4*)(q + KeyRegs<D, MX>::channel(quarter, i));
  }
};

template <int DT, int D, bool MX>
__global__ __launch_bounds__(64 * kWaves, 2) void weigh_rows_kernel(WeighArgs a) {
  const int lane = threadIdx.x & 63, quarter = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, block = blockIdx.x / heads, b = bh / a.n_kv, h = bh % a.n_kv;
  const Extent e = extent_of(a, b);
  const int row0 = block * kBlockRows + wave * kWaveRows;
  if (row0 >= e.len) return;
  KeyRegs<D, MX> k[2];
  bool there[2][2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = min(row0 + 32 * u, (e.len - 1) & ~31), last = min(kTile, e.len - t) - 1;
    LaneOffsets<D, MX> at;
    at.set(last);
    Stream s[2];
    const Sixteen x0 = sixteen_of<D>(a.rows, b, h, t >> 4), x1 = last >= 16 ? sixteen_of<D>(a.rows, b, h, (t >> 4) + 1) : Sixteen{x0.at + 16 * D, x0.there};
    const int64_t e0 = x0.at, e1 = x1.at - 16 * D;  // as if the tile lay together
    s[0] = {(const uint8_t*)a.rows.rows.k + (MX ? e0 : 2 * e0), nullptr, MX ? a.rows.rows.k_scale + e0 / kMxGroup : nullptr, nullptr};
    s[1] = {(const uint8_t*)a.rows.rows.k + (MX ? e1 : 2 * e1), nullptr, MX ? a.rows.rows.k_scale + e1 / kMxGroup : nullptr, nullptr};
    there[u][0] = x0.there;
    there[u][1] = x1.there;
    k[u].load(s, at);
  }
  float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
  // The first query that attends the wave's first row, and the first one that attends all its rows.
  const int past = e.len - e.n, x_end = e.n * a.g;
  const int x_first = max(row0 - past, 0) * a.g & ~15, x_whole = max(row0 + kWaveRows - 1 - past, 0) * a.g;
  if (x_first < x_end) {
    QueryRegs<D, MX> now, next;
    now.load(a, e, b, h, x_first + (lane & 15));
    for (int x = x_first; x < x_end; x += 16) {
      next.load(a, e, b, h, min(x + 16, x_end - 1) + (lane & 15));
      load_fence();
      f32x4 start;
#pragma unroll
      for (int i = 0; i < 4; ++i) start[i] = __shfl(now.start, (lane & 48) + 4 * quarter + i);
      f32x4 sc[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          sc[u][w] = start;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) sc[u][w] = Mat<DT>::mma(now.w[i], k[u].template operand<DT>(w, i), sc[u][w]);
        }
      if (x < x_whole || __any(now.start == -INFINITY)) {
        int limit[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) limit[i] = __shfl(now.limit, (lane & 48) + 4 * quarter + i) - row0 - (lane & 15);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float y = 32 * u + 16 * w < limit[i] ? sc[u][w][i] : -INFINITY;
              keep_here(y);
              sc[u][w][i] = y;
            }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(sc[u][w][i] * a.scale2);
          sum[u][w] += (p[0] + p[1]) + (p[2] + p[3]);
        }
      now = next;
    }
  }
  // Each quarter stores sixteen of the wave's rows.
  float mine = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float total = pair_sum<32>(pair_sum<16>(sum[u][w]));
      mine = quarter == 2 * u + w ? (there[u][w] ? total : 0.0f) : mine;
    }
  store_sum(a, e, b, h, row0 + lane, mine);
}

// ---- many query rows: through LDS ------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT> __device__ __forceinline__ f32x16 wide_mma(uint4 a, uint4 b, f32x16 c) {
  if constexpr (DT == LKV_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

constexpr int kStage = 64;  // query rows
template <int D> __device__ __forceinline__ int swizzle(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }

// A query row that goes on by a stage at a time: its token, its head in the group and where it is, without a division for each.
struct Walk {
  int t, j;
  int64_t at;
  __device__ __forceinline__ void begin(const WeighArgs& a, int b, int h, int x) {
    t = x / a.g;
    j = x - t * a.g;
    at = b * a.q_stride[0] + (h * a.g + j) * a.q_stride[1] + t * a.q_stride[2];
  }
  __device__ __forceinline__ void next(const WeighArgs& a) {
    t += a.step_t;
    j += a.step_j;
    at += a.step_at;
    if (j >= a.g) {
      j -= a.g;
      t += 1;
      at += a.wrap_at;
    }
  }
};

// A stage's query rows on their way to LDS, what is added to their exponents, and how many of a sequence's rows they attend. Every wave's lane l knows row l; a
// row's 16-byte pieces are loaded by other lanes, which ask it where it is. In the place of rows from x_end on the first one of the range lies, without weight.
template <int D> struct StageQueries {
  static_assert(kStage == 64, "a row of the stage for each lane");
  static constexpr int PIECES = D / 8, LOADS = kStage * PIECES / (64 * kWaves);
  u32x4 w[LOADS];
  float less;
  int limit;
  Walk mine;
  int x;  // the stage's first row
  __device__ __forceinline__ void begin(const WeighArgs& a, int b, int h, int x0) {
    x = x0;
    mine.begin(a, b, h, x0 + (int)(threadIdx.x & 63));
  }
  __device__ __forceinline__ void load(const WeighArgs& a, const Extent& e, int b, int h, const Walk& first, int x_end) {
    const bool live = x + (int)(threadIdx.x & 63) < x_end;
    const int64_t at = live ? mine.at : first.at;
    const int lo = (int)(uint32_t)at, hi = (int)(at >> 32);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int r = (i * 64 * kWaves + (int)threadIdx.x) / PIECES;
      const int64_t from = (int64_t)((uint64_t)(uint32_t)__shfl(hi, r) << 32 | (uint32_t)__shfl(lo, r));
      w[i] = *(const u32x4*)(a.q + from + threadIdx.x % PIECES * 8);
    }
    const float l = a.lse[((int64_t)b * a.n_q + h * a.g + (live ? mine.j : first.j)) * a.new_tokens + (live ? mine.t : first.t)];
    less = live && l != -INFINITY ? -l * kLog2e : -INFINITY;
    limit = less != -INFINITY ? e.len - e.n + mine.t + 1 : 0;
    mine.next(a);
    x += kStage;
  }
  __device__ __forceinline__ void store(uint8_t* lds, float* less_at, int* limit_at) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int y = i * 64 * kWaves + threadIdx.x, r = y / PIECES;
      *(u32x4*)(lds + r * (2 * D) + ((y % PIECES) ^ swizzle<D>(r)) * 16) = w[i];
    }
    if (threadIdx.x < kStage) {
      less_at[threadIdx.x] = less;
      limit_at[threadIdx.x] = limit;
    }
  }
};

// The weights of 32 staged queries for a tile of 32 keys, summed. CUT: not all of them attend all keys, or have weight; `row` is the lane's.
template <int DT, int D, bool CUT>
__device__ __forceinline__ float tile_sum(const uint4 (&q)[D / 16], const uint4 (&k)[D / 16], const f32x4 (&less)[4], const int* limits, int row, float scale2) {
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) s = wide_mma<DT>(q[i], k[i], s);
  float p[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float y = __builtin_fmaf(s[i], scale2, less[i / 4][i % 4]);
    if constexpr (CUT) {
      y = row < limits[8 * (i / 4) + i % 4] ? y : -INFINITY;
      keep_here(y);
    }
    p[i] = __builtin_amdgcn_exp2f(y);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] += p[i + 8];
  return ((p[0] + p[4]) + (p[1] + p[5])) + ((p[2] + p[6]) + (p[3] + p[7]));
}

template <int DT, int D, bool MX>
__global__ __launch_bounds__(64 * kWaves, 2) void weigh_wide_kernel(WeighArgs a) {
  constexpr int BYTES = kStage * 2 * D;
  __shared__ u32x4 lds4[2 * BYTES / 16];
  __shared__ __attribute__((aligned(16))) float less_at[2][kStage];
  __shared__ __attribute__((aligned(16))) int limit_at[2][kStage];
  uint8_t* const lds = (uint8_t*)lds4;
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = blockIdx.x;
  const int heads = a.n_seqs * a.n_kv, bh = id % heads;
  id /= heads;
  const int part = id % a.parts, block = id / a.parts, b = bh / a.n_kv, h = bh % a.n_kv;
  const Extent e = extent_of(a, b);
  if (block * kBlockRows >= e.len) return;
  const int row0 = block * kBlockRows + wave * kWaveRows;
  // A lane's key of each tile of 32, channels 16 i + 8 half .. + 8 for the i-th product; behind the end the last one.
  uint4 k[2][D / 16];
  bool there[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = min(row0 + 32 * u + (lane & 31), e.len - 1);
    const Sixteen s = sixteen_of<D, false>(a.rows, b, h, row >> 4);
    const int64_t at = s.at + (row & 15) * D + 8 * half;
    there[u] = s.there;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      if constexpr (MX) {
        const uint2 c = *(const uint2*)((const uint8_t*)a.rows.rows.k + at + 16 * i);
        const float f = bits_to_float((uint32_t)a.rows.rows.k_scale[(at + 16 * i) / kMxGroup] << 23);
        k[u][i] = make_uint4(Mat<DT>::template widen<false>(c.x, f), Mat<DT>::template widen<true>(c.x, f), Mat<DT>::template widen<false>(c.y, f),
                             Mat<DT>::template widen<true>(c.y, f));
      } else {
        k[u][i] = *(const uint4*)((const uint16_t*)a.rows.rows.k + at + 16 * i);
      }
    }
  }
  // The first query that attends the workgroup's first row, and the first one that attends all its rows.
  const int past = e.len - e.n, x_end = min(e.n * a.g, (part + 1) * a.chunk);
  const int x_first = max(part * a.chunk, max(block * kBlockRows - past, 0) * a.g), x_whole = max(min(block * kBlockRows + kBlockRows, e.len) - 1 - past, 0) * a.g;
  float sum[2] = {0.0f, 0.0f};
  if (x_first < x_end) {
    LdsPointer at[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      at[i] = (LdsPointer)lds + (lane & 31) * (2 * D) + ((2 * i + half) ^ swizzle<D>(lane & 31)) * 16;
      keep_here(at[i]);
    }
    Walk first;
    first.begin(a, b, h, x_first);
    StageQueries<D> stage;
    stage.begin(a, b, h, x_first);
    stage.load(a, e, b, h, first, x_end);
    int buffer = 0;
    const auto tiles = [&](auto cut) __attribute__((always_inline)) {
#pragma unroll
      for (int sub = 0; sub < kStage / 32; ++sub) {
        uint4 q[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) q[i] = read_piece(at[i] + buffer * BYTES + sub * 32 * 2 * D);
        f32x4 less[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) less[i] = *(const f32x4*)&less_at[buffer][32 * sub + 8 * i + 4 * half];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          sum[u] += tile_sum<DT, D, decltype(cut)::value>(q, k[u], less, &limit_at[buffer][32 * sub + 4 * half], row0 + 32 * u + (lane & 31), a.scale2);
      }
    };
    for (int x = x_first; x < x_end; x += kStage) {
      const bool cut = x < x_whole || __any(stage.less == -INFINITY);
      stage.store(lds + buffer * BYTES, less_at[buffer], limit_at[buffer]);
      __syncthreads();
      if (x + kStage < x_end) stage.load(a, e, b, h, first, x_end);
      load_fence();
      if (cut) {
        tiles(std::true_type());
      } else {
        tiles(std::false_type());
      }
      buffer ^= 1;
    }
  }
  // Each half stores a tile's rows.
  const float first = pair_sum<32>(sum[0]), second = pair_sum<32>(sum[1]);
  const float mine = half ? (there[1] ? second : 0.0f) : (there[0] ? first : 0.0f);
  if (a.parts > 1) {
    a.part[((int64_t)part * heads + bh) * a.blocks * kBlockRows + row0 + lane] = mine;
  } else {
    store_sum(a, e, b, h, row0 + lane, mine);
  }
}

// The parts' sums of a row, in their order.
__global__ __launch_bounds__(256) void weigh_join_kernel(WeighArgs a) {
  const int heads = a.n_seqs * a.n_kv, bh = blockIdx.x % heads, row = blockIdx.x / heads * kBlockRows + threadIdx.x, b = bh / a.n_kv, h = bh % a.n_kv;
  const Extent e = extent_of(a, b);
  if (row >= e.len) return;
  float got = 0.0f;
  for (int p = 0; p < a.parts; ++p) got += a.part[((int64_t)p * heads + bh) * a.blocks * kBlockRows + row];
  store_sum(a, e, b, h, row, got);
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

struct Plan {
  bool wide;
  int blocks, parts, chunk;
};
Plan plan_of(const lkv_chunk_desc* d) {
  Plan p = {};
  const int64_t x = (int64_t)d->new_tokens * (d->n_q / d->n_kv);
  // Few query rows from memory, many through LDS (8 heads, d 128): 32 over 4,096 rows 6.2 us and by the other form 6.5, over 65,536 29.5 and 33.3; 36 over 4,096
  // 6.6 and 6.5; 64 over 65,536 38.3 and 33.8; 4,096 over 16,384 258 and 187.
  p.wide = x > 32;
  p.blocks = ceil_div(d->max_tokens, kBlockRows);
  const int64_t units = (int64_t)d->n_seqs * d->n_kv * p.blocks;
  // Query rows in parts for 2,048 workgroups, a stage each at the least, which few rows are not: 8,192 of them over 4,096 rows 97 us, by 1,024 workgroups 108, by 4,096 100; 800 over 700
  // 12.2, by four stages each 20.4.
  int64_t parts = units > 0 ? 2048 / units : 1;
  const int64_t most = x / kStage;
  parts = parts > most ? most : parts;
  parts = parts < 1 ? 1 : parts;
  p.chunk = ceil_div(ceil_div(x, parts), kStage) * kStage;
  p.chunk = p.chunk < kStage ? kStage : p.chunk;
  p.parts = ceil_div(x, p.chunk);
  p.parts = p.parts < 1 ? 1 : p.parts;
  return p;
}

template <int DT, int D, bool MX>
void (*kernel_of(const Plan& p))(WeighArgs) {
  return p.wide ? weigh_wide_kernel<DT, D, MX> : weigh_rows_kernel<DT, D, MX>;
}

}  // namespace

extern "C" size_t lkv_weigh_rows_workspace_bytes(const lkv_chunk_desc* desc) {
  if (lkv_check_chunk(desc)) return 0;
  const Plan p = plan_of(desc);
  return p.parts < 2 ? 0 : (size_t)p.parts * desc->n_seqs * desc->n_kv * p.blocks * kBlockRows * sizeof(float);
}

extern "C" int lkv_weigh_rows(uintptr_t stream, const lkv_chunk_desc* desc, const void* q, int q_dtype, const float* lse, const lkv_kv_rows* rows,
                              const lkv_pages* pages, const int32_t* lengths, const int32_t* counts, const float* sums, const int64_t* sums_stride, float* out,
                              const int64_t* out_stride, int32_t* positions, const int64_t* positions_stride, const int32_t* seen, void* ws, size_t ws_bytes) {
  if (int rc = lkv_check_chunk(desc)) return rc;
  // Of few query rows the scores start from -lse / scale. A weight that float32 holds, or one above, has an lse of -89 to 104 beside a score of about 0 at such scales: 104 * 2^120 is
  // finite, and an lse beyond that gives 0 or infinity as it should.
  LKV_CHECK_ARG(desc->scale >= 0x1p-120f, "scale %g: at least 2^-120, its reciprocal times an lse would not be finite", (double)desc->scale);
  LKV_CHECK_ARG(q && lse && out && out_stride && (!sums || sums_stride) && (!positions || positions_stride), "NULL pointer");
  LKV_CHECK_ARG(q_dtype == LKV_F16 || q_dtype == LKV_BF16, "queries are float16 or bfloat16, got dtype %d", q_dtype);
  LKV_CHECK_ARG(((uintptr_t)q & 15) == 0, "queries must start on 16 bytes");
  WeighArgs a = {};
  if (int rc = lkv_paged_rows(rows, pages, desc->n_seqs, q_dtype, desc->head_dim, a.rows)) return rc;
  LKV_CHECK_ARG(desc->max_tokens <= a.rows.capacity, "%d rows of a sequence over %d", desc->max_tokens, a.rows.capacity);
  const size_t need = lkv_weigh_rows_workspace_bytes(desc);
  LKV_CHECK_ARG(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0), "workspace of %zu bytes, on 16: %zu are needed", ws_bytes, need);
  const Plan p = plan_of(desc);
  const int64_t blocks = (int64_t)desc->n_seqs * desc->n_kv * p.blocks;
  LKV_CHECK_ARG(blocks * p.parts < (1 << 24), "%lld workgroups in one call", (long long)blocks * p.parts);
  if (blocks == 0) return LKV_OK;
  a.q = (const uint16_t*)q;
  a.lse = lse;
  a.lengths = lengths;
  a.counts = counts;
  a.seen = seen;
  a.sums = sums;
  a.out = out;
  a.positions = positions;
  a.part = (float*)ws;
  for (int i = 0; i < 3; ++i) a.q_stride[i] = desc->q_stride[i];
  for (int i = 0; i < 2; ++i) {
    a.sums_stride[i] = sums ? sums_stride[i] : 0;
    a.out_stride[i] = out_stride[i];
    a.positions_stride[i] = positions ? positions_stride[i] : 0;
  }
  a.scale2 = desc->scale * kLog2e;
  a.per_scale = 1.0f / desc->scale;
  a.n_seqs = desc->n_seqs;
  a.n_q = desc->n_q;
  a.n_kv = desc->n_kv;
  a.g = desc->n_q / desc->n_kv;
  a.new_tokens = desc->new_tokens;
  a.tokens = desc->tokens;
  a.max_tokens = desc->max_tokens;
  a.blocks = p.blocks;
  a.parts = p.parts;
  a.chunk = p.chunk;
  a.step_t = kStage / a.g;
  a.step_j = kStage % a.g;
  a.step_at = a.step_t * a.q_stride[2] + a.step_j * a.q_stride[1];
  a.wrap_at = a.q_stride[2] - a.g * a.q_stride[1];
  const hipStream_t s = (hipStream_t)stream;
  const bool half = q_dtype == LKV_F16, wide = desc->head_dim == 128, mx = rows->dtype == LKV_MXFP8;
  auto kernel = half ? (wide ? (mx ? kernel_of<LKV_F16, 128, true>(p) : kernel_of<LKV_F16, 128, false>(p)) : (mx ? kernel_of<LKV_F16, 64, true>(p) : kernel_of<LKV_F16, 64, false>(p)))
                     : (wide ? (mx ? kernel_of<LKV_BF16, 128, true>(p) : kernel_of<LKV_BF16, 128, false>(p)) : (mx ? kernel_of<LKV_BF16, 64, true>(p) : kernel_of<LKV_BF16, 64, false>(p)));
  hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks * p.parts)), dim3(64 * kWaves), 0, s, a);
  LKV_CHECK_LAUNCH("weigh_rows");
  if (p.parts > 1) {
    hipLaunchKernelGGL(weigh_join_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
    LKV_CHECK_LAUNCH("weigh_rows (join)");
  }
  return LKV_OK;
}
