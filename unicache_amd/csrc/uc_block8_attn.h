// What the attention kernels of the 8-bit block-scaled cache share: the query
// and launch arguments, the rows and keys of a workgroup, and the arithmetic of the
// scales (uc_block8_attn.hip has the mathematics).
#pragma once
#include "uc_block8.h"

namespace uc {
namespace b8 {

constexpr int kTile = 64;                // keys of a tile
constexpr int32_t kNone = 1 << 30;       // a half tile without keys: behind every length
constexpr float kRaise = 8.0f;           // P stays below 2^8

struct Query {
  const uint16_t *p;
  int64_t ss, st, sh;
  const int32_t *lens;
  int32_t len, heads, group;
  int32_t fp16, causal;
  float scale;  // sm_scale * log2(e)
  FastDiv by_group;

  __device__ __forceinline__ int32_t count(int32_t s) const {
    if (lens == nullptr) return len;
    const int32_t n = lens[s];
    return n < 0 ? 0 : n > len ? len : n;
  }
};

struct Plan {
  const int32_t *list;  // block lists, or NULL: every block
  int32_t budget;
  int32_t run, runs;    // query tokens that share a list (without lists: all), and how many such runs
  int32_t groups, rows; // row groups of a run, and their rows
  int32_t splits, split_tiles;
  int32_t key_groups;   // many rows: 1, or 2 groups of waves in a workgroup that share its tiles
  int32_t workgroups;   // few rows: workgroups that share all tiles; 0: one workgroup a unit
};

// The rows of a workgroup: `first` + r / group is row r's query token.
struct Rows {
  int32_t s, h, length, count;
  int32_t run0, run_rows, r0;  // first token and rows of the run, first row of the group
  int32_t end_first, end_last; // keys that the first and the last row that counts see
};

__device__ __forceinline__ int32_t visible(const Query &q, int32_t length, int32_t count, int32_t token) {
  if (!q.causal) return length;
  const int32_t e = length - count + token + 1;
  return e < 0 ? 0 : e;
}

// Row r's token, counted from the run's first, and its head in the group.
__device__ __forceinline__ int32_t token_of(const Query &q, int32_t r) { return static_cast<int32_t>(fast_div(r, q.by_group)); }

// Rows of group g of a run, with its sequence's length and number of queries.
__device__ __forceinline__ Rows rows_at(const Query &q, const Plan &p, int32_t s, int32_t h, int32_t run, int32_t g, int rows,
                                        int32_t length, int32_t count) {
  Rows w;
  w.s = s;
  w.h = h;
  w.length = length;
  w.count = count;
  w.run0 = run * p.run;
  const int32_t tokens = q.len - w.run0 < p.run ? q.len - w.run0 : p.run;
  w.run_rows = tokens * q.group;
  w.r0 = g * rows;
  const int32_t t0 = w.run0 + token_of(q, w.r0);
  const int32_t r1 = (w.r0 + rows < w.run_rows ? w.r0 + rows : w.run_rows) - 1;
  int32_t t1 = w.run0 + token_of(q, r1);
  t1 = t1 < w.count ? t1 : w.count - 1;
  const bool none = w.r0 >= w.run_rows || t0 >= w.count;
  w.end_first = none ? 0 : visible(q, w.length, w.count, t0);
  w.end_last = none ? 0 : visible(q, w.length, w.count, t1);
  return w;
}

// Rows of unit ((sequence, head, run, group) in order).
__device__ __forceinline__ Rows rows_of(const Cache &c, const Query &q, const Plan &p, int32_t unit, int rows) {
  const int32_t g = unit % p.groups, run = unit / p.groups % p.runs, sh = unit / p.groups / p.runs;
  const int32_t s = sh / c.heads;
  return rows_at(q, p, s, sh % c.heads, run, g, rows, c.length(s), q.count(s));
}

// Tiles of a workgroup's rows, over all splits.
__device__ __forceinline__ int32_t tiles_of(const Cache &c, const Plan &p, const Rows &w) {
  if (p.list == nullptr) return (w.end_last + kTile - 1) / kTile;
  return w.end_last == 0 ? 0 : (p.budget * c.block + kTile - 1) / kTile;
}

// Tiles of one split: the host's figure, or more where a sequence is longer than it expected.
__device__ __forceinline__ int32_t split_tiles_of(const Plan &p, int32_t tiles) {
  const int32_t least = (tiles + p.splits - 1) / p.splits;
  return least > p.split_tiles ? least : p.split_tiles;
}

// Few rows: the tiles of all units ((sequence, head, run) in order) are cut into runs of equal
// length for the workgroups, so that sequences of any lengths load them alike (32 sequences of 8k
// tokens down to none: 74 us by equal splits of the longest, 59 so).  A unit's piece in
// workgroup g leaves its partial in slot g + unit: of two pieces in order one of the two is larger.

// Steps of one (head, run) of a sequence of so many keys: its tiles, rounded up to one for each of
// the four waves.
__device__ __forceinline__ int32_t steps_of(int32_t keys) { return (keys + 4 * kTile - 1) / (4 * kTile) * 4; }

// Keys that a sequence's rows read.
__device__ __forceinline__ int32_t keys_of(const Cache &c, const Plan &p, int32_t length, int32_t count) {
  return p.list != nullptr ? p.budget * c.block : count > 0 ? length : 0;
}

__device__ __forceinline__ int32_t per_of(const Plan &p, int32_t total) {
  return ((total + p.workgroups - 1) / p.workgroups + 3) / 4 * 4;
}

// A wave's sum, the same in every lane.
__device__ __forceinline__ int32_t wave_total(int32_t v) { return __builtin_amdgcn_readlane(wave_prefix(v), 63); }

// For a whole wave: steps of all sequences (of one head and run), of those before a lane's s, and of s.
struct Steps {
  int32_t total, before, mine;
};

__device__ __forceinline__ Steps steps_before(const Cache &c, const Query &q, const Plan &p, int32_t s) {
  Steps w = {0, 0, 0};
  if (p.list != nullptr) {
    w.mine = steps_of(keys_of(c, p, 0, 0));
    w.total = w.mine * c.sequences;
    w.before = w.mine * s;
    return w;
  }
  for (int32_t s0 = 0; s0 < c.sequences; s0 += 64) {
    const int32_t i = s0 + (threadIdx.x & 63);
    const int32_t n = i < c.sequences ? steps_of(keys_of(c, p, c.length(i), q.count(i))) : 0;
    const int32_t sum = wave_prefix(n);
    const int32_t m = __shfl(n, s - s0, kWave), b = __shfl(sum, s - s0, kWave);
    if (s >= s0 && s < s0 + 64) {
      w.mine = m;
      w.before = w.total + b - m;
    }
    w.total += __builtin_amdgcn_readlane(sum, 63);
  }
  return w;
}

// A run's block list, 64 entries at a time in a wave's lanes, so that a tile's entry is no load that
// its codes' loads would wait for.  An index that is none, that lies outside the cache or that is given twice in a row reads as -1.
struct BlockList {
  const int32_t *list;  // NULL: every block in turn
  int32_t budget, blocks, chunk, held;

  __device__ __forceinline__ BlockList(const Cache &c, const Plan &p, const Rows &w)
      : list(p.list), budget(p.budget), blocks(c.blocks), chunk(-1), held(-1) {
    if (list != nullptr) list += ((int64_t(w.s) * p.runs + w.run0 / p.run) * c.heads + w.h) * p.budget;
  }

  __device__ __forceinline__ int32_t entry(int32_t e) {
    if (e >= budget) return -1;
    if ((e >> 6) != chunk) {
      chunk = e >> 6;
      const int32_t i = chunk * 64 + (threadIdx.x & 63);
      const int32_t b = i < budget ? list[i] : -1, before = i > 0 && i < budget ? list[i - 1] : -1;
      held = b < 0 || b >= blocks || b == before ? -1 : b;
    }
    return __builtin_amdgcn_readlane(held, e & 63);
  }
};

// First key of a half tile (32 keys); kNone where there is none.
template <bool LISTED>
__device__ __forceinline__ int32_t half_of(const Cache &c, BlockList &list, int32_t half) {
  if constexpr (!LISTED) return half < c.blocks << (c.shift - 5) ? half * 32 : kNone;
  const int32_t b = list.entry(half >> (c.shift - 5));
  return b < 0 ? kNone : (b << c.shift) + (half & ((c.block >> 5) - 1)) * 32;
}

// Keep the first n of 16 bytes.
__device__ __forceinline__ uint4 first_bytes(uint4 v, int32_t n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int32_t k = n - 4 * i;
    w[i] = k >= 4 ? w[i] : k <= 0 ? 0u : w[i] & ((1u << (8 * k)) - 1u);
  }
  return uint4{w[0], w[1], w[2], w[3]};
}

// The value scale that keys count with in their weights' exponents.  A weight is relative to the largest
// logit + log2(scale) of its row, so a scale far below another's would leave fp32's range there: it counts as
// 2^-60 of `most`, the largest scale of the blocks that the row has seen, the present tile's among them
// (its weights then keep their place in l, whose terms are P / scale).  And where no larger one has been seen it counts as
// 2^-88 at least: a key adds 2^88 to l at most, a raised reference 2^8, so the 2^30 keys of the
// longest sequence stay below 2^128.  (A scale of 0 comes from another program; the quantizer's smallest is 2^-60.)
constexpr float kLeastScale = 0x1p-88f;

__device__ __forceinline__ float larger_scale(float most, float vs) {
  return vs < __builtin_huge_valf() ? fmaxf(most, vs) : most;  // an infinity or a NaN is no scale to go by
}

__device__ __forceinline__ float counted_scale(float vs, float most) {
  const float least = fmaxf(most * 0x1p-60f, kLeastScale);
  return vs < least ? least : vs;  // a NaN stays
}

// l 2^d: in two steps, since 2^d may be below fp32's range where the product is not.
__device__ __forceinline__ float rescaled(float l, float d) {
  const float a = mf::fast_exp2(0.5f * d);
  return l * a * a;
}

template <int DT, int N>
__device__ __forceinline__ void widen(const uint4 (&raw)[N], float (&x)[N][8]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) x[k][j] = half_bits_to_f32<DT>(j % 2 ? u[j / 2] >> 16 : u[j / 2]);
  }
}

// One query row's fragments, scaled by a power of two into fp16; returns the
// factor of its logits: sm_scale log2(e) / the power.  Lane quad x holds channels
// 32 k + 8 x .. + 7 of fragment k; with PAIRS 64 (k / 2) + 16 x + 8 (k % 2) .. + 7, so that 16 bytes
// of codes feed two fragments.
template <int D, bool PAIRS>
__device__ __forceinline__ float load_query(const Query &q, const Rows &w, int32_t r, h8 (&frag)[D / 32]) {
  const int quad = (threadIdx.x & 63) >> 4;
  const int32_t token = w.run0 + token_of(q, r);
  uint4 raw[D / 32];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) raw[k] = uint4{0, 0, 0, 0};
  if (r < w.run_rows && token < w.count) {
    const uint16_t *p = q.p + w.s * q.ss + token * q.st + (w.h * q.group + r - token_of(q, r) * q.group) * q.sh;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      raw[k] = *reinterpret_cast<const uint4 *>(p + (PAIRS ? (k / 2) * 64 + quad * 16 + (k % 2) * 8 : k * 32 + quad * 8));
    }
  }
  float x[D / 32][8], a = 0.0f;
  if (q.fp16) {
    widen<UC_FP16>(raw, x);
  } else {
    widen<UC_BF16>(raw, x);
  }
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) a = fmaxf(a, fabsf(x[k][j]));
  }
  a = mf::max_over_slices(a);
  int e = static_cast<int>((__float_as_uint(a) >> 23) & 0xff) - 127;
  // a row of zeros, or one with an infinity (whose logits are what they are); below 2^-100 the
  // power stays in fp32's range
  e = a == 0.0f || e == 128 ? 14 : e < -100 ? -100 : e;
  const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
  const float down = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) frag[k][j] = mf::to_h(x[k][j] * up);
  }
  return q.scale * down;
}

// Two outputs of the query's type.  (A select, not a branch: both are a few instructions.)
__device__ __forceinline__ uint32_t pack2(float a, float b, bool fp16) {
  const uint32_t h = __builtin_bit_cast(uint32_t, h2{mf::to_h(a), mf::to_h(b)});
  const uint32_t w = f32_to_bf16_bits(a) | (static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16);
  return fp16 ? h : w;
}

// uc_block8_mq.hip: 128 rows a workgroup, keys staged through LDS.
constexpr int kTileRows = 128;
int launch_tiles(const uc_block8_cache *cache, const Cache &c, const Query &q, const Plan &p, uint16_t *out, float *lse, float *part, float *stat, hipStream_t stream);

}  // namespace b8
}  // namespace uc
