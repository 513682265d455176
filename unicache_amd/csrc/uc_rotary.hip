// Rotary positions of several axes, alone and on the way into a paged cache.
//
// Pair i of a head turns by angle 2 pi positions[axis[i]] turns[i]:
//   (a, b) -> (a cos - b sin, b cos + a sin).
// A position of 2^20 is 2^17 revolutions of the fastest pair, of which only the fraction counts: fp32
// would leave 2^-7 of a revolution of it.  So the product is 64-bit, its whole revolutions are taken
// off there, and the fraction in [-1/2, 1/2] goes on in fp32, whose sine and cosine of pi x are exact
// to a few units.  The rest is fp32, rounded once at the end.
//
// A workgroup takes one or a few tokens: it works out each pair's sine and cosine once, into LDS, and
// turns all heads of the token by them, 16 channels (two 16-byte vectors, both sides of eight pairs) a
// thread.  The values on their way into a cache ride along as rows without pairs.
//
// Bound by HBM: 7k tokens of 32 + 8 heads 29.3 us (4.9 TB/s over reads and writes), 16k tokens into a cache 66.6 (4.5).  Four
// tokens a workgroup from 2048 tokens on, where their pairs fill its threads; below that one, for more workgroups.
#include "uc_paged.h"

namespace uc {
namespace pg {
namespace {

constexpr int kMostPairs = 256;

struct Rows {  // dense [S, n, heads, D]; heads 0: none
  const uint16_t *p;
  int64_t ss, st, sh;
  int32_t heads;
};

struct Turn {
  const double *turns;
  const int32_t *axis;
  const void *positions;
  int32_t axes, pairs, bytes, adjacent, inverse;
};

struct Job {
  Rows query, key, value;
  uint16_t *out_query, *out_key;  // contiguous; out_key NULL: key and value go to the cache
  const int32_t *counts;
  int32_t sequences, tokens, chunks;  // chunks: 16 channels each, of a head
  FastDiv by_tokens, by_chunks, by_units;
};

__device__ __forceinline__ int64_t position(const Turn &t, int64_t i) {
  return t.bytes == 8 ? static_cast<const int64_t *>(t.positions)[i] : static_cast<const int32_t *>(t.positions)[i];
}

template <int DT>
__device__ __forceinline__ void widen(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = half_bits_to_f32<DT>(j % 2 ? w[j / 2] >> 16 : w[j / 2]);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == UC_FP16) return f32_to_f16_bits(a) | (static_cast<uint32_t>(f32_to_f16_bits(b)) << 16);
  return f32_to_bf16_bits(a) | (static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16);
}

template <int DT>
__device__ __forceinline__ uint4 narrow(const float (&x)[8]) {
  return uint4{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7])};
}

template <int DT, int T>
__global__ __launch_bounds__(256) void rotary_kernel(Cache c, Job job, Turn t) {
  __shared__ float2 turn[T][kMostPairs];  // (cos, sin)
  const int32_t rows = job.sequences * job.tokens, first = blockIdx.x * T;
  const int32_t here = rows - first < T ? rows - first : T;
  for (int32_t i = threadIdx.x; i < here * t.pairs; i += 256) {
    const int32_t k = T == 1 ? 0 : i / t.pairs, pair = i - k * t.pairs, row = first + k;
    int64_t at;
    if (t.positions != nullptr) {
      const int32_t a = t.axis[pair];
      at = position(t, int64_t(a < 0 || a >= t.axes ? 0 : a) * rows + row);
    } else {  // the token's place in its sequence
      const int32_t s = fast_div(row, job.by_tokens), n = row - s * job.tokens;
      int32_t count = job.counts != nullptr ? job.counts[s] : job.tokens;
      count = count < 0 ? 0 : count > job.tokens ? job.tokens : count;
      at = c.length(s) - count + n;
    }
    const double turns = static_cast<double>(at) * t.turns[pair];
    float sine, cosine;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sine, &cosine);
    turn[k][pair] = float2{cosine, t.inverse ? -sine : sine};
  }
  __syncthreads();
  const int32_t heads = job.query.heads + job.key.heads + job.value.heads, units = heads * job.chunks;
  for (int32_t i = threadIdx.x; i < here * units; i += 256) {
    const int32_t k = T == 1 ? 0 : fast_div(i, job.by_units), unit = i - k * units;
    const int32_t row = first + k, s = fast_div(row, job.by_tokens), n = row - s * job.tokens;
    int32_t head = fast_div(unit, job.by_chunks);
    const int32_t chunk = unit - head * job.chunks;
    const bool of_query = head < job.query.heads, of_value = head >= job.query.heads + job.key.heads;
    const Rows &r = of_query ? job.query : of_value ? job.value : job.key;
    if (!of_query) head -= job.query.heads;
    if (of_value) head -= job.key.heads;
    const int32_t d = job.chunks * 16;
    const uint16_t *src = r.p + s * r.ss + n * r.st + head * r.sh;
    uint16_t *dst;
    if (of_query) {
      dst = job.out_query + (int64_t(row) * r.heads + head) * d;
    } else if (job.out_key != nullptr) {
      dst = job.out_key + (int64_t(row) * r.heads + head) * d;
    } else {
      int32_t count = job.counts != nullptr ? job.counts[s] : job.tokens;
      count = count < 0 ? 0 : count > job.tokens ? job.tokens : count;
      const int32_t token = c.length(s) - count + n;
      if (n >= count || token < 0) continue;
      const int32_t page = c.table[int64_t(s) * c.width + (token >> c.shift)];
      if (!c.is_page(page)) continue;
      dst = (of_value ? c.value : c.key) + int64_t(page) * c.page_elems + ((head << c.shift) + (token & (c.page - 1))) * d;
    }
    const bool turned = !of_value && chunk * 8 < t.pairs;
    const bool halves = turned && !t.adjacent;
    const int32_t a = halves ? 8 * chunk : 16 * chunk, b = halves ? 8 * chunk + t.pairs : 16 * chunk + 8;
    uint4 va = *reinterpret_cast<const uint4 *>(src + a), vb = *reinterpret_cast<const uint4 *>(src + b);
    if (turned) {
      float x[8], y[8], u[8], w[8];
      widen<DT>(va, x);
      widen<DT>(vb, y);
      float2 cs[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) cs[j] = turn[k][8 * chunk + j];
      if (halves) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[j] = __builtin_fmaf(x[j], cs[j].x, -(y[j] * cs[j].y));
          w[j] = __builtin_fmaf(y[j], cs[j].x, x[j] * cs[j].y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u[2 * j] = __builtin_fmaf(x[2 * j], cs[j].x, -(x[2 * j + 1] * cs[j].y));
          u[2 * j + 1] = __builtin_fmaf(x[2 * j + 1], cs[j].x, x[2 * j] * cs[j].y);
          w[2 * j] = __builtin_fmaf(y[2 * j], cs[4 + j].x, -(y[2 * j + 1] * cs[4 + j].y));
          w[2 * j + 1] = __builtin_fmaf(y[2 * j + 1], cs[4 + j].x, y[2 * j] * cs[4 + j].y);
        }
      }
      va = narrow<DT>(u);
      vb = narrow<DT>(w);
    }
    *reinterpret_cast<uint4 *>(dst + a) = va;
    *reinterpret_cast<uint4 *>(dst + b) = vb;
  }
}

int check_plan(const uc_rotary_plan *plan, int64_t head_dim, bool positions, const char *what, Turn &t) {
  UC_REQUIRE(plan->turns != nullptr && plan->axis != nullptr, "%s: the plan's turns and axes are NULL", what);
  UC_REQUIRE(plan->pairs > 0 && plan->pairs % 8 == 0 && 2 * plan->pairs <= head_dim,
             "%s: pairs must be a multiple of 8, and twice as many no more than head_dim", what);
  UC_REQUIRE(plan->axes > 0 && plan->axes < (1 << 16), "%s: bad number of axes", what);
  UC_REQUIRE(!positions || plan->positions != nullptr, "%s: positions are NULL", what);
  UC_REQUIRE(plan->positions == nullptr || plan->position_bytes == 4 || plan->position_bytes == 8,
             "%s: positions must have 4 or 8 bytes", what);
  t = Turn{plan->turns, plan->axis, plan->positions, static_cast<int32_t>(plan->axes), static_cast<int32_t>(plan->pairs),
           plan->position_bytes, plan->adjacent != 0, plan->inverse != 0};
  return UC_OK;
}

int check_rows(const Rows &r, const char *what, const char *name) {
  UC_REQUIRE(r.p != nullptr && (reinterpret_cast<uintptr_t>(r.p) & 15) == 0 && ((r.ss | r.st | r.sh) & 7) == 0,
             "%s: %s must be 16-byte aligned with strides that are multiples of 8", what, name);
  return UC_OK;
}

int launch(const char *what, int dtype, const Cache &c, Job &job, const Turn &t, hipStream_t stream) {
  const int64_t rows = int64_t(job.sequences) * job.tokens;
  const int32_t units = (job.query.heads + job.key.heads + job.value.heads) * job.chunks;
  job.by_tokens = make_fastdiv(static_cast<uint32_t>(job.tokens));
  job.by_chunks = make_fastdiv(static_cast<uint32_t>(job.chunks));
  job.by_units = make_fastdiv(static_cast<uint32_t>(units));
  auto go = [&](auto kernel, int tokens) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(ceil_div(rows, int64_t(tokens)))), dim3(256), 0, stream, c, job,
                       t);
  };
  if (rows < 2048) {
    dtype == UC_FP16 ? go(rotary_kernel<UC_FP16, 1>, 1) : go(rotary_kernel<UC_BF16, 1>, 1);
  } else {
    dtype == UC_FP16 ? go(rotary_kernel<UC_FP16, 4>, 4) : go(rotary_kernel<UC_BF16, 4>, 4);
  }
  return check_launch(what);
}

// (a launch has less than 2^32 threads; a workgroup's units stay in 31 bits)
int check_sizes(int64_t sequences, int64_t tokens, int64_t heads, const char *what) {
  UC_REQUIRE(sequences >= 0 && tokens >= 0 && sequences < (1 << 24) && tokens < (1 << 24) &&
                 sequences * tokens < (1 << 24),
             "%s: too many rows", what);
  UC_REQUIRE(heads < (1 << 20), "%s: too many heads", what);
  return UC_OK;
}

}  // namespace
}  // namespace pg
}  // namespace uc

extern "C" int uc_rotary(const uc_rotary_plan *plan, int64_t sequences, int64_t tokens, int64_t head_dim, int dtype,
                         const void *query, int64_t q_ss, int64_t q_st, int64_t q_sh, int64_t heads_q, void *out_query,
                         const void *key, int64_t k_ss, int64_t k_st, int64_t k_sh, int64_t heads_k, void *out_key,
                         uc_stream_t stream) {
  using namespace uc;
  using namespace uc::pg;
  const char *what = "uc_rotary";
  UC_REQUIRE(plan != nullptr, "%s: plan is NULL", what);
  UC_REQUIRE(half_dtype(dtype), "%s: rows must be bf16 or fp16", what);
  UC_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 2 * kMostPairs,
             "%s: head_dim must be a multiple of 16, and %d at most", what, 2 * kMostPairs);
  UC_REQUIRE(heads_q > 0 && heads_k >= 0, "%s: bad number of heads", what);
  if (int rc = check_sizes(sequences, tokens, heads_q > heads_k ? heads_q : heads_k, what)) return rc;
  Turn t;
  if (int rc = check_plan(plan, head_dim, sequences * tokens > 0, what, t)) return rc;
  if (sequences * tokens == 0) return UC_OK;
  Job job = {};
  job.query = Rows{static_cast<const uint16_t *>(query), q_ss, q_st, q_sh, static_cast<int32_t>(heads_q)};
  job.key = Rows{static_cast<const uint16_t *>(key), k_ss, k_st, k_sh, static_cast<int32_t>(heads_k)};
  job.out_query = static_cast<uint16_t *>(out_query);
  job.out_key = static_cast<uint16_t *>(out_key);
  if (int rc = check_rows(job.query, what, "query")) return rc;
  UC_REQUIRE(out_query != nullptr && (reinterpret_cast<uintptr_t>(out_query) & 15) == 0, "%s: out must be 16-byte aligned", what);
  if (heads_k > 0) {
    if (int rc = check_rows(job.key, what, "key")) return rc;
    UC_REQUIRE(out_key != nullptr && (reinterpret_cast<uintptr_t>(out_key) & 15) == 0, "%s: out must be 16-byte aligned", what);
  }
  job.sequences = static_cast<int32_t>(sequences);
  job.tokens = static_cast<int32_t>(tokens);
  job.chunks = static_cast<int32_t>(head_dim / 16);
  return launch(what, dtype, Cache{}, job, t, as_stream(stream));
}

extern "C" int uc_paged_write(const uc_paged_cache *cache, int64_t layer, const void *key, int64_t k_ss, int64_t k_st,
                              int64_t k_sh, const void *value, int64_t v_ss, int64_t v_st, int64_t v_sh, int64_t tokens,
                              const int32_t *counts, const uc_rotary_plan *plan, const void *query, int64_t q_ss,
                              int64_t q_st, int64_t q_sh, int64_t heads_q, void *out_query, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::pg;
  const char *what = "uc_paged_write";
  Cache c;
  if (int rc = check_cache(cache, layer, what, c)) return rc;
  UC_REQUIRE(query == nullptr || plan != nullptr, "%s: a query without a plan", what);
  UC_REQUIRE(query == nullptr || heads_q > 0, "%s: bad number of query heads", what);
  if (int rc = check_sizes(c.sequences, tokens, query != nullptr && heads_q > c.heads ? heads_q : c.heads, what)) return rc;
  Turn t = {};
  if (plan != nullptr) {
    if (int rc = check_plan(plan, cache->head_dim, false, what, t)) return rc;
  }
  if (tokens == 0) return UC_OK;
  Job job = {};
  job.key = Rows{static_cast<const uint16_t *>(key), k_ss, k_st, k_sh, c.heads};
  job.value = Rows{static_cast<const uint16_t *>(value), v_ss, v_st, v_sh, c.heads};
  if (int rc = check_rows(job.key, what, "key")) return rc;
  if (int rc = check_rows(job.value, what, "value")) return rc;
  if (query != nullptr) {
    job.query = Rows{static_cast<const uint16_t *>(query), q_ss, q_st, q_sh, static_cast<int32_t>(heads_q)};
    job.out_query = static_cast<uint16_t *>(out_query);
    if (int rc = check_rows(job.query, what, "query")) return rc;
    UC_REQUIRE(out_query != nullptr && (reinterpret_cast<uintptr_t>(out_query) & 15) == 0, "%s: out must be 16-byte aligned", what);
  }
  job.counts = counts;
  job.sequences = c.sequences;
  job.tokens = static_cast<int32_t>(tokens);
  job.chunks = static_cast<int32_t>(cache->head_dim / 16);
  return launch(what, cache->dtype, c, job, t, as_stream(stream));
}
