// Block selection for sparse attention over the 8-bit block-scaled cache.
//
// A row q as whole numbers c = round(q (127 / max|q|)) can have at most
//   I = sum_d max(c_d hi_d, c_d lo_d) = sum_d c+_d hi_d + c-_d lo_d
// with a key inside a block's bounds (c+ and c- its positive and negative parts), so the scores
// of all rows and blocks are one int8 matrix product over 2 D, exact in
// int32; a score is fp32(I) u step, two roundings, whatever the order of the sum.
// Three launches: the rows' codes, the scores (16 blocks x 16 rows per
// MFMA tile, the largest over a run's rows kept in registers), and
// the choice of the `budget` highest (radix selection on the scores' ordered
// bit patterns).
#include "uc_block8.h"

#include <type_traits>

namespace uc {
namespace b8 {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));

struct Run {
  const uint16_t *q;
  int64_t ss, st, sh;
  const int32_t *lens;
  int32_t len, heads, group, run, runs;
  int32_t fp16, causal;
  int32_t budget, sink, recent;

  __device__ __forceinline__ int32_t count(int32_t s) const {
    if (lens == nullptr) return len;
    const int32_t n = lens[s];
    return n < 0 ? 0 : n > len ? len : n;
  }
  // Of a run: the last keys that its first and its last row see; false where no row counts or sees one.
  __device__ __forceinline__ bool keys(int32_t length, int32_t count, int32_t index, int32_t &first, int32_t &last) const {
    const int32_t t0 = index * run;
    if (t0 >= count) return false;
    int32_t t1 = t0 + run - 1;
    t1 = t1 < count ? t1 : count - 1;
    first = causal ? length - count + t0 : length - 1;
    last = causal ? length - count + t1 : length - 1;
    first = first < 0 ? 0 : first;
    return last >= 0;
  }
};

// One wave per query row: its codes and their step; step -1 marks a row that does not count.
template <int D>
__global__ __launch_bounds__(256) void codes_kernel(Cache c, Run q, int8_t *codes, float *steps, int64_t rows) {
  constexpr int kE = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int32_t h = static_cast<int32_t>(row % q.heads), t = static_cast<int32_t>(row / q.heads % q.len);
  const int32_t s = static_cast<int32_t>(row / q.heads / q.len);
  float x[kE], a = 0.0f;
  bool bad = t >= q.count(s);
  if (!bad) {
    const uint16_t *p = q.q + s * q.ss + t * q.st + h * q.sh + lane * kE;
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      x[j] = q.fp16 ? f16_bits_to_f32(p[j]) : bf16_bits_to_f32(p[j]);
      a = fmaxf(a, fabsf(x[j]));
      bad = bad || !(fabsf(x[j]) < __builtin_huge_valf());
    }
    a = wave_max(a);
  }
  bad = __any(bad);
  const float inverse = bad || a == 0.0f ? 0.0f : div_rn(127.0f, a);
#pragma unroll
  for (int j = 0; j < kE; ++j) {
    const float y = bad ? 0.0f : __builtin_amdgcn_fmed3f(rintf(mul_rn(x[j], inverse)), -127.0f, 127.0f);
    codes[row * D + lane * kE + j] = static_cast<int8_t>(static_cast<int>(y));
  }
  if (lane == 0) steps[row] = bad ? -1.0f : mul_rn(a, 1.0f / 127.0f);
}

// The bytes of w that are positive, and those that are negative.
__device__ __forceinline__ void parts(int w, int &pos, int &neg) {
  const uint32_t m = ((static_cast<uint32_t>(w) >> 7) & 0x01010101u) * 255u;
  neg = static_cast<int>(static_cast<uint32_t>(w) & m);
  pos = static_cast<int>(static_cast<uint32_t>(w) & ~m);
}

// A wave scores 16 blocks for one run: S = bounds x codes^T, so a lane holds
// four blocks of one row, and the largest over the rows stays in its registers.
template <int D>
__global__ __launch_bounds__(256) void score_kernel(Cache c, Run q, const int8_t *codes, const float *steps,
                                                    float unit_factor, float *score, int32_t chunks) {
  constexpr int kK = D / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int32_t unit = blockIdx.x / chunks, chunk = blockIdx.x % chunks;  // unit: (sequence, run, head)
  const int32_t h = unit % c.heads, run = unit / c.heads % q.runs, s = unit / c.heads / q.runs;
  const int32_t length = c.length(s), count = q.count(s);
  int32_t first, last;
  if (!q.keys(length, count, run, first, last)) return;
  const int32_t blocks = (last >> c.shift) + 1;
  const int32_t t0 = run * q.run;
  const int32_t rows = ((count - t0 < q.run) ? count - t0 : q.run) * q.group;
  const int64_t sh = int64_t(s) * c.heads + h;
  for (int32_t b0 = (chunk * 4 + wave) * 16; b0 < blocks; b0 += chunks * 64) {
    i4 hi[kK], lo[kK];
    const int32_t mine = b0 + col < blocks ? b0 + col : blocks - 1;
    const int8_t *p = c.bounds + (sh * c.blocks + mine) * 2 * D + quad * 16;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      hi[k] = *reinterpret_cast<const i4 *>(p + k * 64);
      lo[k] = *reinterpret_cast<const i4 *>(p + D + k * 64);
    }
    float u[4], best[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t b = b0 + quad * 4 + i;
      u[i] = mul_rn(c.key_scale[sh * c.blocks + (b < blocks ? b : blocks - 1)], unit_factor);
      best[i] = mf::kNegInf;
    }
    for (int32_t r0 = 0; r0 < rows; r0 += 16) {
      const int32_t r = r0 + col < rows ? r0 + col : rows - 1;  // the last row again: it changes no maximum
      const int64_t at = (int64_t(s) * q.len + t0 + r / q.group) * q.heads + h * q.group + r % q.group;
      const float step = steps[at];
      i4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const i4 w = *reinterpret_cast<const i4 *>(codes + at * D + k * 64 + quad * 16);
        i4 pos, neg;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          int a, b;
          parts(w[j], a, b);
          pos[j] = a;
          neg[j] = b;
        }
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi[k], pos, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo[k], neg, acc, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = mul_rn(mul_rn(static_cast<float>(acc[i]), u[i]), step);
        best[i] = step >= 0.0f ? fmaxf(best[i], v) : best[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) best[i] = fmaxf(best[i], __shfl_xor(best[i], o, kWave));
      const int32_t b = b0 + quad * 4 + i;
      if (col == 0 && b < blocks) {
        // a block whose scale is no finite number is chosen, so that its NaN shows
        score[int64_t(unit) * c.blocks + b] = u[i] < __builtin_huge_valf() ? best[i] : __builtin_huge_valf();
      }
    }
  }
}

// Bits of a score that order as it does.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

// One workgroup per (sequence, run, head).  Blocks before `low` and from
// `high` on are chosen anyway; of the others the `want` highest.
__global__ __launch_bounds__(256) void choose_kernel(Cache c, Run q, const float *score, int32_t *out) {
  __shared__ int32_t hist[256];
  __shared__ int32_t shared[4];
  __shared__ int32_t wave_eq[4], wave_in[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t unit = blockIdx.x;
  const int32_t run = unit / c.heads % q.runs, s = unit / c.heads / q.runs;
  const int32_t length = c.length(s), count = q.count(s);
  const float *sc = score + int64_t(unit) * c.blocks;
  int32_t *list = out + int64_t(unit) * q.budget;
  int32_t first, last, blocks = 0, low = 0, high = 0;
  if (q.keys(length, count, run, first, last)) {
    blocks = (last >> c.shift) + 1;
    high = (first >> c.shift) - q.recent + 1;
    low = q.sink < blocks ? q.sink : blocks;
    high = high < low ? low : high;
  }
  const int32_t want = q.budget - low - (blocks - high);
  uint32_t threshold = 0;
  int32_t equals = 0;  // blocks at the threshold that are chosen
  if (want < high - low) {
    // the want-th highest of [low, high), eight bits at a time
    int32_t need = want > 0 ? want : 0;
    if (need == 0) {
      threshold = 0xffffffffu;
    } else {
      for (int shift = 24; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int32_t b = low + tid; b < high; b += 256) {
          const uint32_t key = ordered(sc[b]);
          if (shift == 24 || (key >> (shift + 8)) == (threshold >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        // thread i: keys in bins above i
        int32_t above = 0;
        for (int i = tid + 1; i < 256; ++i) above += hist[i];
        if (above < need && above + hist[tid] >= need) {
          shared[0] = tid;
          shared[1] = above;
        }
        __syncthreads();
        threshold |= static_cast<uint32_t>(shared[0]) << shift;
        need -= shared[1];
        __syncthreads();
      }
      equals = need;
    }
  }
  const bool all = want >= high - low;
  int32_t written = 0, seen_equal = 0;
  for (int32_t b0 = 0; b0 < blocks; b0 += 256) {
    const int32_t b = b0 + tid;
    const bool live = b < blocks, must = live && (b < low || b >= high || all);
    const uint32_t key = live && !must ? ordered(sc[b]) : 0;
    const bool equal = live && !must && key == threshold;
    const uint64_t eq = __ballot(equal);
    if (lane == 0) wave_eq[wave] = __popcll(eq);
    __syncthreads();
    int32_t rank = seen_equal + __popcll(eq & ((uint64_t(1) << lane) - 1));
    for (int w = 0; w < 4; ++w) {
      if (w < wave) rank += wave_eq[w];
      seen_equal += wave_eq[w];
    }
    const bool in = must || (live && (key > threshold || (equal && rank < equals)));
    const uint64_t chosen = __ballot(in);
    if (lane == 0) wave_in[wave] = __popcll(chosen);
    __syncthreads();
    int32_t at = written + __popcll(chosen & ((uint64_t(1) << lane) - 1));
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += wave_in[w];
      written += wave_in[w];
    }
    if (in && at < q.budget) list[at] = b;
  }
  for (int32_t i = written + tid; i < q.budget; i += 256) list[i] = -1;
}

int make_run(const uc_block8_cache *cache, const uc_block8_query *query, int64_t query_block, const char *what, Run &q) {
  UC_REQUIRE(query != nullptr, "%s: query is NULL", what);
  UC_REQUIRE(half_dtype(query->dtype), "%s: queries must be bf16 or fp16", what);
  UC_REQUIRE(query->heads_q > 0 && query->heads_q % cache->heads_kv == 0,
             "%s: query heads must be a multiple of KV heads", what);
  UC_REQUIRE(query->query_len >= 0 && query->query_len < (1 << 24), "%s: bad query_len", what);
  UC_REQUIRE(query->heads_q / cache->heads_kv * query->query_len < (int64_t(1) << 30), "%s: too many query rows", what);
  UC_REQUIRE(query->max_tokens >= 0, "%s: negative max_tokens", what);
  UC_REQUIRE(query_block > 0, "%s: query_block must be positive", what);
  const int64_t len = query->query_len > 0 ? query->query_len : 1;
  const int64_t run = query_block < len ? query_block : len;
  q = Run{static_cast<const uint16_t *>(query->query), query->q_ss, query->q_st, query->q_sh, query->query_lengths,
          static_cast<int32_t>(query->query_len), static_cast<int32_t>(query->heads_q),
          static_cast<int32_t>(query->heads_q / cache->heads_kv), static_cast<int32_t>(run),
          static_cast<int32_t>(ceil_div(query->query_len, run)), query->dtype == UC_FP16, query->causal != 0, 0, 0, 0};
  return UC_OK;
}

struct Space {
  int64_t codes, steps, scores, total;  // byte offsets
};

Space space_of(const uc_block8_cache *cache, const Run &q) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t rows = cache->sequences * q.len * q.heads;
  Space w;
  w.codes = 0;
  w.steps = up(rows * cache->head_dim);
  w.scores = w.steps + up(rows * 4);
  w.total = w.scores + up(cache->sequences * q.runs * cache->heads_kv * cache->blocks * 4);
  return w;
}

}  // namespace
}  // namespace b8
}  // namespace uc

extern "C" int64_t uc_block8_select_workspace_bytes(const uc_block8_cache *cache, const uc_block8_query *query,
                                                    int64_t query_block) {
  using namespace uc::b8;
  Cache c;
  Run q;
  if (check_cache(cache, "uc_block8_select", c) || make_run(cache, query, query_block, "uc_block8_select", q)) return -1;
  return space_of(cache, q).total;
}

extern "C" int uc_block8_select(const uc_block8_cache *cache, const uc_block8_query *query, int64_t budget,
                                int64_t sink, int64_t recent, int64_t query_block, int32_t *blocks, void *workspace,
                                int64_t workspace_bytes, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::b8;
  Cache c;
  Run q;
  if (int rc = check_cache(cache, "uc_block8_select", c)) return rc;
  if (int rc = make_run(cache, query, query_block, "uc_block8_select", q)) return rc;
  UC_REQUIRE(budget > 0 && budget < (1 << 24), "uc_block8_select: budget must be positive");
  UC_REQUIRE(sink >= 0 && recent >= 1, "uc_block8_select: sink must not be negative and recent must be positive");
  const int64_t span = q.causal ? ceil_div(int64_t(q.run) - 1, int64_t(c.block)) : 0;
  UC_REQUIRE(sink + recent + span <= budget, "uc_block8_select: budget %lld is less than the %lld blocks always chosen",
             static_cast<long long>(budget), static_cast<long long>(sink + recent + span));
  if (q.len == 0) return UC_OK;
  UC_REQUIRE(q.q != nullptr && (reinterpret_cast<uintptr_t>(q.q) & 15) == 0 && ((q.ss | q.st | q.sh) & 7) == 0,
             "uc_block8_select: query must be 16-byte aligned with strides that are multiples of 8");
  UC_REQUIRE(blocks != nullptr, "uc_block8_select: blocks is NULL");
  const Space w = space_of(cache, q);
  UC_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= w.total,
             "uc_block8_select: workspace too small");
  q.budget = static_cast<int32_t>(budget);
  q.sink = static_cast<int32_t>(sink);
  q.recent = static_cast<int32_t>(recent);
  char *ws = static_cast<char *>(workspace);
  int8_t *codes = reinterpret_cast<int8_t *>(ws + w.codes);
  float *steps = reinterpret_cast<float *>(ws + w.steps), *score = reinterpret_cast<float *>(ws + w.scores);
  const int64_t rows = cache->sequences * q.len * q.heads, units = cache->sequences * q.runs * cache->heads_kv;
  const int64_t capacity = cache->blocks * cache->block_tokens;
  const int64_t expected = query->max_tokens < capacity ? query->max_tokens : capacity;
  const int64_t chunks = expected > 0 ? ceil_div(ceil_div(expected, int64_t(c.block)), 64) : 1;
  UC_REQUIRE(rows < (int64_t(1) << 32) && units * chunks < (int64_t(1) << 31), "uc_block8_select: too many query rows");
  const float factor = cache->code_dtype == UC_INT8 ? 1.0f : static_cast<float>(448.0 / 127.0);
  auto launch = [&](auto d_tag) {
    constexpr int D = decltype(d_tag)::value;
    hipLaunchKernelGGL((codes_kernel<D>), dim3(static_cast<uint32_t>(ceil_div(rows, 4))), dim3(256), 0,
                       as_stream(stream), c, q, codes, steps, rows);
    if (int rc = check_launch("uc_block8_select (codes)")) return rc;
    hipLaunchKernelGGL((score_kernel<D>), dim3(static_cast<uint32_t>(units * chunks)), dim3(256), 0, as_stream(stream),
                       c, q, codes, steps, factor, score, static_cast<int32_t>(chunks));
    return check_launch("uc_block8_select (scores)");
  };
  if (int rc = cache->head_dim == 128 ? launch(std::integral_constant<int, 128>())
                                      : launch(std::integral_constant<int, 64>()))
    return rc;
  hipLaunchKernelGGL(choose_kernel, dim3(static_cast<uint32_t>(units)), dim3(256), 0, as_stream(stream), c, q, score,
                     blocks);
  return check_launch("uc_block8_select");
}
