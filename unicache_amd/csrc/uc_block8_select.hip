// Block selection for sparse attention over the 8-bit block-scaled cache.
//
// A row q as whole numbers c = round(q (127 / max|q|)) (of 2^64 q for rows below 2^-100) can have at most
//   I = sum_d max(c_d hi_d, c_d lo_d) = sum_d c+_d hi_d + c-_d lo_d
// with a key inside a block's bounds (c+ and c- its positive and negative parts), so the scores
// of all rows and blocks are one int8 matrix product over 2 D, exact in
// int32; a score is fp32(I) u step, two roundings, whatever the order of the sum.
// Runs of at most 16 rows (decode) take one launch, a workgroup per run and
// head: scores into LDS, then the `budget` highest by histograms of eight bits of their ordered
// patterns; or, few runs of many blocks, one for the scores and one for the choice.  512 blocks 9.4 us
// (latency: lengths, rows, bounds, four histogram rounds), 2048 blocks of 128 heads 14.2 + 9.6 us
// (67 MB of bounds at 4.7 TB/s, and the choice).  Longer runs take three: the rows' codes, the
// scores (MFMA tiles of 16 rows x 16 blocks, the largest over a run's rows kept in registers), and the
// choice; 2048 tokens of 28/4 heads by 512 blocks 7.4 + 14.5 + 5.6 us.
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
  FastDiv by_group;

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

// Eight 16-bit values as floats.
__device__ __forceinline__ void to_floats(uint4 raw, bool fp16, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t bits = (j % 2 ? w[j / 2] >> 16 : w[j / 2]) & 0xffffu;
    x[j] = fp16 ? f16_bits_to_f32(static_cast<uint16_t>(bits)) : bf16_bits_to_f32(bits);
  }
}

// round(x inverse) of four values as bytes.
__device__ __forceinline__ uint32_t four_codes(const float *x, float inverse) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float y = __builtin_amdgcn_fmed3f(rintf(mul_rn(x[j], inverse)), -127.0f, 127.0f);
    w |= (static_cast<uint32_t>(static_cast<int>(y)) & 0xffu) << (8 * j);
  }
  return w;
}

// The codes' factor of a row with largest magnitude a, and their step.
__device__ __forceinline__ float code_factor(float a) { return a > 0.0f ? div_rn(127.0f, a) : 0.0f; }
// Rows below 2^-100 are multiplied by this first, exactly: 127 / a is past fp32's range below 2^-121.
__device__ __forceinline__ float code_lift(float a) { return a < 0x1p-100f ? 0x1p64f : 1.0f; }
__device__ __forceinline__ float code_step(float a) { return mul_rn(a, 1.0f / 127.0f); }

// The bytes of w that are positive, and those that are negative.
__device__ __forceinline__ void parts(int w, int &pos, int &neg) {
  const uint32_t m = ((static_cast<uint32_t>(w) >> 7) & 0x01010101u) * 255u;
  neg = static_cast<int>(static_cast<uint32_t>(w) & m);
  pos = static_cast<int>(static_cast<uint32_t>(w) & ~m);
}

// The codes and steps of all query rows, D / 8 lanes a row; a NaN step marks a row that does not count
// (no maximum takes it).
template <int D>
__global__ __launch_bounds__(256) void codes_kernel(Cache c, Run q, int8_t *codes, float *steps, int64_t rows) {
  constexpr int kLanes = D / 8;
  const int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) / kLanes;
  const int part = threadIdx.x % kLanes;
  if (row >= rows) return;
  const int32_t h = static_cast<int32_t>(row % q.heads), t = static_cast<int32_t>(row / q.heads % q.len);
  const int32_t s = static_cast<int32_t>(row / q.heads / q.len);
  const bool counts = t < q.count(s);
  float x[8], a = 0.0f;
  to_floats(counts ? *reinterpret_cast<const uint4 *>(q.q + s * q.ss + t * q.st + h * q.sh + part * 8) : uint4{0, 0, 0, 0},
            q.fp16, x);
  int bad = !counts;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a = fmaxf(a, fabsf(x[j]));
    bad |= !(fabsf(x[j]) < __builtin_huge_valf());
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    a = fmaxf(a, __shfl_xor(a, o, kWave));
    bad |= __shfl_xor(bad, o, kWave);
  }
  const float up = code_lift(a), f = bad ? 0.0f : code_factor(mul_rn(a, up));
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = bad ? 0.0f : mul_rn(x[j], up);
  *reinterpret_cast<uint2 *>(codes + row * D + part * 8) = uint2{four_codes(x, f), four_codes(x + 4, f)};
  if (part == 0) steps[row] = bad ? __builtin_nanf("") : code_step(a);
}

// Codes of 16 rows as the A operand: lane % 16 is the row, lane / 16 and k name 16 channels; and the
// steps of the lane's four rows of the results, 4 (lane / 16) + i.
template <int D>
struct RowCodes {
  i4 pos[D / 64], neg[D / 64];
  f4 step;

  __device__ __forceinline__ void split(int k, i4 w) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int a, b;
      parts(w[j], a, b);
      pos[k][j] = a;
      neg[k][j] = b;
    }
  }
};

// Bounds of 16 blocks as the B operand, lane % 16 the block, and that block's step.
template <int D>
struct BlockBounds {
  i4 hi[D / 64], lo[D / 64];
  float u;
};

template <int D>
__device__ __forceinline__ void load_bounds(BlockBounds<D> &x, const Cache &c, int64_t sh, int32_t b0, int32_t blocks,
                                            float unit_factor) {
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int64_t mine = sh * c.blocks + (b0 + col < blocks ? b0 + col : blocks - 1);
  const int8_t *p = c.bounds + mine * 2 * D + quad * 16;
#pragma unroll
  for (int k = 0; k < D / 64; ++k) {
    x.hi[k] = *reinterpret_cast<const i4 *>(p + k * 64);
    x.lo[k] = *reinterpret_cast<const i4 *>(p + D + k * 64);
  }
  x.u = mul_rn(c.key_scale[mine], unit_factor);
}

// best = max(best, the scores of the lane's block in its four rows)
template <int D>
__device__ __forceinline__ void score16(const BlockBounds<D> &x, const RowCodes<D> &r, float &best) {
  i4 acc = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < D / 64; ++k) {
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(r.pos[k], x.hi[k], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(r.neg[k], x.lo[k], acc, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) best = fmaxf(best, mul_rn(mul_rn(static_cast<float>(acc[i]), x.u), r.step[i]));
}

// The largest over all rows; a block whose scale is no finite number is
// chosen, so that its NaN shows.
__device__ __forceinline__ float over_rows(float best, float u) {
  best = mf::max_over_slices(best);
  return u < __builtin_huge_valf() ? best : __builtin_huge_valf();
}

// The codes of a run's at most 16 rows into LDS, D / 8 lanes a row.
template <int D>
struct OwnCodes {
  int8_t codes[16][D];
  float step[16];
};

template <int D>
__device__ __forceinline__ void own_codes(OwnCodes<D> &own, const Run &q, int32_t s, int32_t h, int32_t t0, int32_t rows) {
  constexpr int kLanes = D / 8;
  const int r = threadIdx.x / kLanes, part = threadIdx.x % kLanes;
  if (r >= 16) return;
  const bool counts = r < rows;
  float x[8], a = 0.0f;
  const int32_t token = t0 + r / q.group, head = h * q.group + r % q.group;
  to_floats(counts ? *reinterpret_cast<const uint4 *>(q.q + s * q.ss + token * q.st + head * q.sh + part * 8)
                   : uint4{0, 0, 0, 0}, q.fp16, x);
  int bad = !counts;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a = fmaxf(a, fabsf(x[j]));
    bad |= !(fabsf(x[j]) < __builtin_huge_valf());
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    a = fmaxf(a, __shfl_xor(a, o, kWave));
    bad |= __shfl_xor(bad, o, kWave);
  }
  const float up = code_lift(a), f = bad ? 0.0f : code_factor(mul_rn(a, up));
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = bad ? 0.0f : mul_rn(x[j], up);
  *reinterpret_cast<uint2 *>(&own.codes[r][part * 8]) = uint2{four_codes(x, f), four_codes(x + 4, f)};
  if (part == 0) own.step[r] = bad ? __builtin_nanf("") : code_step(a);
}

// Scores for runs of many rows.  A wave takes 64 blocks, whose bounds stay in registers; a workgroup
// takes 64 rows at a time into LDS, split into their positive and negative parts, for its four
// waves, the next 64 on their way (each wave loading all rows for itself was bound by L2: 20 us for 28 x 2048 rows
// by 512 blocks).
constexpr int kScored = 4;      // 16-block groups of a wave
constexpr int kFewBlocks = 256; // blocks of a workgroup and step of score_few_kernel
constexpr int kStageRows = 64;

template <int D>
__global__ __launch_bounds__(256) void score_kernel(Cache c, Run q, const int8_t *codes, const float *steps,
                                                    float unit_factor, float *score, int32_t chunks) {
  constexpr int kPitch = 2 * D + 16;  // bytes of a row: eight rows' chunks lie in different banks
  constexpr int kLanes = D / 16, kLoads = kStageRows * kLanes / 256;
  __shared__ __attribute__((aligned(16))) int8_t sh_codes[kStageRows * kPitch];
  __shared__ __attribute__((aligned(16))) float sh_step[kStageRows];
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
  const int64_t row0 = (int64_t(s) * q.len + t0) * q.heads + h * q.group;
  auto index_of = [&](int32_t r) {  // rows past the last are the last again: they change no maximum
    r = r < rows ? r : rows - 1;
    const int32_t token = static_cast<int32_t>(fast_div(r, q.by_group));
    return row0 + int64_t(token) * q.heads + (r - token * q.group);
  };
  for (int32_t base = chunk * 64 * kScored; base < blocks; base += chunks * 64 * kScored) {
    const int32_t b0 = base + wave * 16 * kScored;
    BlockBounds<D> x[kScored];
    float best[kScored];
#pragma unroll
    for (int n = 0; n < kScored; ++n) {
      load_bounds<D>(x[n], c, sh, b0 + 16 * n, blocks, unit_factor);
      best[n] = mf::kNegInf;
    }
    i4 next[kLoads];
    float next_step = 0.0f;
    auto fetch = [&](int32_t r0) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = threadIdx.x + i * 256;
        next[i] = *reinterpret_cast<const i4 *>(codes + index_of(r0 + at / kLanes) * D + at % kLanes * 16);
      }
      if (threadIdx.x < kStageRows) next_step = steps[index_of(r0 + threadIdx.x)];
    };
    fetch(0);
    for (int32_t r0 = 0; r0 < rows; r0 += kStageRows) {
      __syncthreads();  // the rows before have been read
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = threadIdx.x + i * 256;
        i4 pos, neg;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          int a, b;
          parts(next[i][j], a, b);
          pos[j] = a;
          neg[j] = b;
        }
        int8_t *dst = sh_codes + at / kLanes * kPitch + at % kLanes * 16;
        *reinterpret_cast<i4 *>(dst) = pos;
        *reinterpret_cast<i4 *>(dst + D) = neg;
      }
      if (threadIdx.x < kStageRows) sh_step[threadIdx.x] = next_step;
      __syncthreads();
      if (r0 + kStageRows < rows) fetch(r0 + kStageRows);
      for (int g = 0; g < kStageRows / 16 && r0 + 16 * g < rows; ++g) {
        RowCodes<D> rc;
        rc.step = *reinterpret_cast<const f4 *>(&sh_step[16 * g + 4 * quad]);
        const int8_t *src = sh_codes + (16 * g + col) * kPitch + quad * 16;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
          rc.pos[k] = *reinterpret_cast<const i4 *>(src + k * 64);
          rc.neg[k] = *reinterpret_cast<const i4 *>(src + D + k * 64);
        }
#pragma unroll
        for (int n = 0; n < kScored; ++n) score16<D>(x[n], rc, best[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < kScored; ++n) {
      const float v = over_rows(best[n], x[n].u);
      const int32_t b = b0 + 16 * n + col;
      if (quad == 0 && b < blocks) score[int64_t(unit) * c.blocks + b] = v;
    }
  }
}

// The blocks of a run: those before `low` and from `high` on (up to `blocks`) are chosen anyway, of the
// others the `want` highest.
struct Candidates {
  int32_t blocks, low, high, want;
  __device__ __forceinline__ bool all() const { return want >= high - low; }
};

__device__ __forceinline__ Candidates candidates(const Cache &c, const Run &q, int32_t length, int32_t count, int32_t run) {
  Candidates x = {0, 0, 0, 0};
  int32_t first, last;
  if (q.keys(length, count, run, first, last)) {
    x.blocks = (last >> c.shift) + 1;
    x.high = (first >> c.shift) - q.recent + 1;
    x.low = q.sink < x.blocks ? q.sink : x.blocks;
    x.high = x.high < x.low ? x.low : x.high;
  }
  x.want = q.budget - x.low - (x.blocks - x.high);
  return x;
}

// Scores of a run's at most 16 rows by 16 * GROUPS blocks a wave and step, for the blocks from b0 on below
// `high` in steps of `stride`: the rows' codes go through `own`, take(block, score) gets the outcomes.
template <int D, int GROUPS, class Take>
__device__ __forceinline__ void score_run(const Cache &c, const Run &q, int32_t s, int32_t h, int32_t run, int32_t count,
                                          int32_t b0, int32_t high, int32_t stride, float unit_factor, OwnCodes<D> &own,
                                          const Take &take) {
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int64_t sh = int64_t(s) * c.heads + h;
  BlockBounds<D> bb[GROUPS];
  if (b0 < high) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) load_bounds<D>(bb[g], c, sh, b0 + 16 * g, high, unit_factor);
  }
  const int32_t t0 = run * q.run;
  own_codes<D>(own, q, s, h, t0, ((count - t0 < q.run) ? count - t0 : q.run) * q.group);
  __syncthreads();
  RowCodes<D> rc;
  rc.step = *reinterpret_cast<const f4 *>(&own.step[4 * quad]);
#pragma unroll
  for (int k = 0; k < D / 64; ++k) rc.split(k, *reinterpret_cast<const i4 *>(&own.codes[col][k * 64 + quad * 16]));
  for (int32_t b1 = b0; b1 < high; b1 += stride) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      float best = mf::kNegInf;
      score16<D>(bb[g], rc, best);
      const float v = over_rows(best, bb[g].u);
      const int32_t b = b1 + 16 * g + col;
      if (quad == 0 && b < high) take(b, v);
    }
    if (b1 + stride < high) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) load_bounds<D>(bb[g], c, sh, b1 + stride + 16 * g, high, unit_factor);
    }
  }
}

// The scores of a run of at most 16 rows by `chunks` workgroups, for choose_kernel.
template <int D>
__global__ __launch_bounds__(256) void score_few_kernel(Cache c, Run q, float unit_factor, float *score, int32_t chunks) {
  __shared__ __attribute__((aligned(16))) OwnCodes<D> own;
  const int32_t unit = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int32_t h = unit % c.heads, run = unit / c.heads % q.runs, s = unit / c.heads / q.runs;
  const int32_t count = q.count(s);
  const Candidates x = candidates(c, q, c.length(s), count, run);
  const int32_t begin = x.low + chunk * kFewBlocks;
  if (x.all() || begin >= x.high) return;
  float *sc = score + int64_t(unit) * c.blocks;
  score_run<D, kFewBlocks / 64>(c, q, s, h, run, count, begin + (threadIdx.x >> 6) * (kFewBlocks / 4), x.high,
                                chunks * kFewBlocks, unit_factor, own, [&](int32_t b, float v) { sc[b] = v; });
}

// Bits of a score that order as it does.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int32_t kKept = 8192;  // scores that choose_kernel holds in LDS

// One workgroup per (sequence, run, head).  The smallest of the `want` highest scores is found eight
// bits a round by histograms in LDS, then the chosen are written by prefix sums.  With FUSED (runs of
// at most 16 rows) the scores are computed here, so that a decode step's choice is one launch.
template <int T, int D, bool FUSED>
__global__ __launch_bounds__(T) void choose_kernel(Cache c, Run q, float unit_factor, float *score, int32_t *out) {
  constexpr int kWaves = T / kWave;
  __shared__ uint32_t kept[kKept];
  __shared__ __attribute__((aligned(16))) int32_t hist[256];
  __shared__ __attribute__((aligned(16))) OwnCodes<D> own;
  __shared__ int32_t found[2];
  __shared__ int32_t wave_eq[kWaves], wave_in[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t unit = blockIdx.x;
  const int32_t h = unit % c.heads, run = unit / c.heads % q.runs, s = unit / c.heads / q.runs;
  const int32_t length = c.length(s), count = q.count(s);
  float *sc = score + int64_t(unit) * c.blocks;
  int32_t *list = out + int64_t(unit) * q.budget;
  const Candidates x = candidates(c, q, length, count, run);
  const int32_t blocks = x.blocks, low = x.low, high = x.high, want = x.want;
  const int32_t n = high - low;  // blocks to choose from
  const bool all = x.all(), held = n <= kKept;
  if (!all) {
    if constexpr (FUSED) {
      score_run<D, 4>(c, q, s, h, run, count, low + wave * 64, high, kWaves * 64, unit_factor, own,
                      [&](int32_t b, float v) {
                        if (held) {
                          kept[b - low] = ordered(v);
                        } else {
                          sc[b] = v;
                        }
                      });
    } else if (held) {
      for (int32_t i = tid; i < n; i += T) kept[i] = ordered(sc[low + i]);
    }
  }
  __syncthreads();  // also orders this workgroup's writes of `score` before its reads
  auto key = [&](int32_t i) { return held ? kept[i] : ordered(sc[low + i]); };

  uint32_t threshold = 0;
  int32_t equals = 0;  // blocks at the threshold that are chosen
  if (!all && want > 0) {
    int32_t need = want;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += T) hist[i] = 0;
      __syncthreads();
      // bin 0 holds the highest digit
      for (int32_t i = tid; i < n; i += T) {
        const uint32_t k = key(i);
        if (shift == 24 || (k >> (shift + 8)) == (threshold >> (shift + 8))) {
          atomicAdd(&hist[255 - ((k >> shift) & 255u)], 1);
        }
      }
      __syncthreads();
      if (wave == 0) {  // the bin that the need-th key falls into
        const int4 v = *reinterpret_cast<const int4 *>(&hist[4 * lane]);
        const int32_t mine = v.x + v.y + v.z + v.w;
        const int32_t sum = wave_prefix(mine);
        int32_t above = sum - mine;
        if (above < need && sum >= need) {
          int bin = 4 * lane;
          const int32_t w[3] = {v.x, v.y, v.z};
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            if (bin == 4 * lane + i && above + w[i] < need) {
              above += w[i];
              ++bin;
            }
          }
          found[0] = 255 - bin;
          found[1] = above;
        }
      }
      __syncthreads();
      threshold |= static_cast<uint32_t>(found[0]) << shift;
      need -= found[1];
    }
    equals = need;
  }
  for (int32_t i = tid; i < low; i += T) list[i] = i;
  int32_t written = low, seen_equal = 0;
  if (all) {
    for (int32_t i = tid; i < n; i += T) list[low + i] = low + i;
    written += n;
  } else if (want > 0) {
    for (int32_t i0 = 0; i0 < n; i0 += T) {
      const int32_t i = i0 + tid;
      const uint32_t k = i < n ? key(i) : 0;
      const bool equal = i < n && k == threshold;
      const uint64_t eq = __ballot(equal), before = (uint64_t(1) << lane) - 1;
      if (lane == 0) wave_eq[wave] = __popcll(eq);
      __syncthreads();
      int32_t rank = seen_equal + __popcll(eq & before);
      for (int v = 0; v < kWaves; ++v) {
        if (v < wave) rank += wave_eq[v];
        seen_equal += wave_eq[v];
      }
      const bool in = i < n && (k > threshold || (equal && rank < equals));
      const uint64_t chosen = __ballot(in);
      if (lane == 0) wave_in[wave] = __popcll(chosen);
      __syncthreads();
      int32_t at = written + __popcll(chosen & before);
      for (int v = 0; v < kWaves; ++v) {
        if (v < wave) at += wave_in[v];
        written += wave_in[v];
      }
      if (in) list[at] = low + i;
    }
  }
  for (int32_t i = tid; i < blocks - high; i += T) list[written + i] = high + i;
  for (int32_t i = written + blocks - high + tid; i < q.budget; i += T) list[i] = -1;
}

int make_run(const uc_block8_cache *cache, const uc_block8_query *query, int64_t query_block, const char *what, Run &q) {
  UC_REQUIRE(query != nullptr, "%s: query is NULL", what);
  UC_REQUIRE(half_dtype(query->dtype), "%s: queries must be bf16 or fp16", what);
  UC_REQUIRE(query->heads_q > 0 && query->heads_q % cache->heads_kv == 0,
             "%s: query heads must be a multiple of KV heads", what);
  UC_REQUIRE(query->query_len >= 0 && query->query_len < (1 << 24), "%s: bad query_len", what);
  UC_REQUIRE(query->heads_q < (1 << 24), "%s: too many query heads", what);  // (the products below stay in 64 bits)
  UC_REQUIRE(query->heads_q / cache->heads_kv * query->query_len < (int64_t(1) << 30), "%s: too many query rows", what);
  UC_REQUIRE(query->max_tokens >= 0, "%s: negative max_tokens", what);
  UC_REQUIRE(query_block > 0, "%s: query_block must be positive", what);
  const int64_t len = query->query_len > 0 ? query->query_len : 1;
  const int64_t run = query_block < len ? query_block : len;
  q = Run{static_cast<const uint16_t *>(query->query), query->q_ss, query->q_st, query->q_sh, query->query_lengths,
          static_cast<int32_t>(query->query_len), static_cast<int32_t>(query->heads_q),
          static_cast<int32_t>(query->heads_q / cache->heads_kv), static_cast<int32_t>(run),
          static_cast<int32_t>(ceil_div(query->query_len, run)), query->dtype == UC_FP16, query->causal != 0, 0, 0, 0,
          make_fastdiv(static_cast<uint32_t>(query->heads_q / cache->heads_kv))};
  return UC_OK;
}

// Runs whose rows fit one product: their codes need no memory.
bool few(const Run &q) { return q.run * q.group <= 16; }

// Whether a launch of its own computes their scores, with a workgroup per 256 blocks: where a workgroup per
// run would take more than one step over its 512 blocks and leave half of the CUs idle (a CU takes
// in 24 bytes a ns at most, 6 TB/s in all).  One launch, then two, us: 8 runs of 512 blocks 9.2, 9.9; 1024 14.5, 11.6; 8192
// 80, 30; 128 runs of 512 10.0, 11.2; 1024 16.9, 16.0; 2048 29.2, 24.3; 256 runs of 1024 19.8, 21.7; 4096
// 60, 65.
bool scored_apart(int64_t units, int64_t blocks) { return blocks > 512 && units <= 128; }

struct Space {
  int64_t codes, steps, scores, total;  // byte offsets
};

Space space_of(const uc_block8_cache *cache, const Run &q) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t rows = few(q) ? 0 : cache->sequences * q.len * q.heads;
  const int64_t units = cache->sequences * q.runs * cache->heads_kv;
  const bool scores = !few(q) || cache->blocks > kKept || scored_apart(units, cache->blocks);
  Space w;
  w.codes = 0;
  w.steps = up(rows * cache->head_dim);
  w.scores = w.steps + up(rows * 4);
  w.total = w.scores + up(scores ? units * cache->blocks * 4 : 1);
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
  UC_REQUIRE(budget > 0 && budget <= (1 << 30) / cache->block_tokens, "uc_block8_select: bad budget");
  UC_REQUIRE(sink >= 0 && recent >= 1, "uc_block8_select: sink must not be negative and recent must be positive");
  const int64_t span = q.causal ? ceil_div(int64_t(q.run) - 1, int64_t(c.block)) : 0;
  // (each by itself first: the sum of large ones would pass 64 bits)
  UC_REQUIRE(sink <= budget && recent <= budget, "uc_block8_select: budget %lld is less than the blocks always chosen",
             static_cast<long long>(budget));
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
  const int64_t chunks = expected > 0 ? ceil_div(ceil_div(expected, int64_t(c.block)), 64 * kScored) : 1;
  // a launch has less than 2^32 threads
  UC_REQUIRE(few(q) ? units < (1 << 23)
                      : rows * (cache->head_dim / 8) < (int64_t(1) << 32) - 256 && units * chunks < (1 << 24),
             "uc_block8_select: too many query rows");
  const float factor = cache->code_dtype == UC_INT8 ? 1.0f : static_cast<float>(448.0 / 127.0);
  auto launch = [&](auto d_tag) {
    constexpr int D = decltype(d_tag)::value;
    if (few(q)) {
      if (scored_apart(units, ceil_div(expected, int64_t(c.block)))) {
        hipLaunchKernelGGL((score_few_kernel<D>), dim3(static_cast<uint32_t>(units * chunks)), dim3(256), 0,
                           as_stream(stream), c, q, factor, score, static_cast<int32_t>(chunks));
        if (int rc = check_launch("uc_block8_select (scores)")) return rc;
        hipLaunchKernelGGL((choose_kernel<512, D, false>), dim3(static_cast<uint32_t>(units)), dim3(512), 0,
                           as_stream(stream), c, q, factor, score, blocks);
        return check_launch("uc_block8_select");
      }
      hipLaunchKernelGGL((choose_kernel<512, D, true>), dim3(static_cast<uint32_t>(units)), dim3(512), 0,
                         as_stream(stream), c, q, factor, score, blocks);
      return check_launch("uc_block8_select");
    }
    hipLaunchKernelGGL((codes_kernel<D>), dim3(static_cast<uint32_t>(ceil_div(rows, 256 / (D / 8)))), dim3(256), 0,
                       as_stream(stream), c, q, codes, steps, rows);
    if (int rc = check_launch("uc_block8_select (codes)")) return rc;
    hipLaunchKernelGGL((score_kernel<D>), dim3(static_cast<uint32_t>(units * chunks)), dim3(256), 0, as_stream(stream),
                       c, q, codes, steps, factor, score, static_cast<int32_t>(chunks));
    if (int rc = check_launch("uc_block8_select (scores)")) return rc;
    hipLaunchKernelGGL((choose_kernel<256, D, false>), dim3(static_cast<uint32_t>(units)), dim3(256), 0,
                       as_stream(stream), c, q, factor, score, blocks);
    return check_launch("uc_block8_select");
  };
  return cache->head_dim == 128 ? launch(std::integral_constant<int, 128>()) : launch(std::integral_constant<int, 64>());
}
