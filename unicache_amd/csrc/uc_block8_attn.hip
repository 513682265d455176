// Attention over the 8-bit block-scaled cache, by split keys: every workgroup
// takes up to 16 NR query rows of one KV head (its query heads x query tokens)
// and a run of 64-key tiles, its four waves alternate tiles, and what they hold is
// joined at the end; a second launch joins the splits.
//
// Mathematics, per row r and key t of block b, in base 2:
//   x = (q_r . k_t) ks_b sm_scale log2(e) + log2(vs_b)
//   P = 2^(x - m), O = sum P v_code, l = sum P / vs_b, out = O / l, lse = ln2 (m + log2 l)
// so both scales cost nothing per key: the key's scale is the factor that the
// logit needs anyway and the value's scale is an addend of the exponent.  m is a
// running reference of x (not of the logit): P stays in fp16's range
// whatever the blocks' scales are, and its rounding (half a step, 2^-11) is
// relative to the largest contribution.  Sums, m and O are fp32.  A block whose
// value scale is less than 2^-60 of one read before it (a block of zeros has
// 2^-60) counts as 2^-60 of that one: its weights then keep their place in l, and
// what its values add is below 2^-51 of the head's largest either way.
//
// Codes become fp16 exactly (int8 and e4m3 both fit); a query row is
// multiplied by a power of two that brings its largest value to [2^14, 2^15),
// so bf16 rows keep all their bits down to 2^-28 of it, and the power goes into the
// logit's factor.
//
// Layout: S^T = K Q^T on 16x16x32 MFMAs.  Row r of key tile j is key
// 16 (r / 4) + 4 j + r % 4 of the 64, so that a lane's 16 logits are 16
// consecutive keys of one query row, which is the operand that
// O^T = V^T P^T takes, with no exchange between lanes: the values' blocks are
// stored channel-major for that, 16 codes of a channel in one 16-byte load.
#include "uc_block8.h"

#include <type_traits>

namespace uc {
namespace b8 {
namespace {

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
  int32_t groups;       // row groups of a run
  int32_t splits, split_tiles;
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

__device__ __forceinline__ Rows rows_of(const Cache &c, const Query &q, const Plan &p, int32_t unit, int rows) {
  Rows w;
  const int32_t g = unit % p.groups, run = unit / p.groups % p.runs, sh = unit / p.groups / p.runs;
  w.s = sh / c.heads;
  w.h = sh % c.heads;
  w.length = c.length(w.s);
  w.count = q.count(w.s);
  w.run0 = run * p.run;
  const int32_t tokens = q.len - w.run0 < p.run ? q.len - w.run0 : p.run;
  w.run_rows = tokens * q.group;
  w.r0 = g * rows;
  const int32_t t0 = w.run0 + w.r0 / q.group;
  const int32_t r1 = (w.r0 + rows < w.run_rows ? w.r0 + rows : w.run_rows) - 1;
  int32_t t1 = w.run0 + r1 / q.group;
  t1 = t1 < w.count ? t1 : w.count - 1;
  const bool none = w.r0 >= w.run_rows || t0 >= w.count;
  w.end_first = none ? 0 : visible(q, w.length, w.count, t0);
  w.end_last = none ? 0 : visible(q, w.length, w.count, t1);
  return w;
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

// First key of a half tile (32 keys); kNone where the list has none there.
__device__ __forceinline__ int32_t half_of(const Cache &c, const Plan &p, const int32_t *list, int32_t half) {
  if (list == nullptr) return half * 32;
  const int32_t e = half >> (c.shift - 5), sub = half & ((c.block >> 5) - 1);
  if (e >= p.budget) return kNone;
  const int32_t b = list[e];
  const bool again = e > 0 && list[e - 1] == b;  // an index given twice counts once
  return b < 0 || b >= c.blocks || again ? kNone : (b << c.shift) + sub * 32;
}

// Codes of one tile as they come from memory, with the scales of the lane's keys.
template <int D>
struct Raw {
  uint4 k[4][D / 64];
  uint4 v[D / 16];
  float ks, vs;
};

template <int D>
struct Lane {
  const uint8_t *kcode, *vcode;   // of the (sequence, head), at the lane's offset in a tile
  const float *kscale, *vscale;
  int32_t key;                    // the lane's key offset in its half: 0 or 16
};

template <int D>
__device__ __forceinline__ void load_keys(Raw<D> &raw, const Cache &c, const Lane<D> &l, int32_t t0, int32_t t1) {
  const int r = threadIdx.x & 15, lane = threadIdx.x & 63;
  const int32_t tk = (r & 8) ? t1 : t0, tq = (lane & 32) ? t1 : t0;
  const uint8_t *p = l.kcode + int64_t(tk == kNone ? 0 : tk) * D;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int x = 0; x < D / 64; ++x) raw.k[j][x] = *reinterpret_cast<const uint4 *>(p + j * 4 * D + x * 64);
  }
  const int32_t b = tq == kNone ? 0 : tq >> c.shift;
  raw.ks = l.kscale[b];
  raw.vs = l.vscale[b];
}

template <int D>
__device__ __forceinline__ void load_values(Raw<D> &raw, const Cache &c, const Lane<D> &l, int32_t t0, int32_t t1) {
  const int lane = threadIdx.x & 63;
  const int32_t tq = (lane & 32) ? t1 : t0;
  const int32_t t = tq == kNone ? 0 : tq;
  const uint8_t *p = l.vcode + (int64_t(t >> c.shift) << c.shift) * D + (t & (c.block - 1));
  const int32_t step = 16 * c.block;
#pragma unroll
  for (int n = 0; n < D / 16; ++n) raw.v[n] = *reinterpret_cast<const uint4 *>(p + n * step);
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

// One query row's fragments, scaled by a power of two into fp16; returns the
// factor of its logits: sm_scale log2(e) / the power.
template <int D>
__device__ __forceinline__ float load_query(const Query &q, const Rows &w, int32_t r, h8 (&frag)[D / 32]) {
  const int quad = (threadIdx.x & 63) >> 4;
  const int32_t token = w.run0 + r / q.group;
  uint4 raw[D / 32];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) raw[k] = uint4{0, 0, 0, 0};
  if (r < w.run_rows && token < w.count) {
    const uint16_t *p = q.p + w.s * q.ss + token * q.st + (w.h * q.group + r % q.group) * q.sh;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      raw[k] = *reinterpret_cast<const uint4 *>(p + (k / 2) * 64 + quad * 16 + (k % 2) * 8);
    }
  }
  float x[D / 32][8], a = 0.0f;
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = j % 2 ? u[j / 2] >> 16 : u[j / 2];
      x[k][j] = q.fp16 ? f16_bits_to_f32(static_cast<uint16_t>(bits)) : bf16_bits_to_f32(bits & 0xffffu);
      a = fmaxf(a, fabsf(x[k][j]));
    }
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

// The value scale that a tile's keys count with; `most` is the largest so far.
__device__ __forceinline__ float counted_scale(float vs, float &most) {
  if (vs < __builtin_huge_valf()) most = fmaxf(most, vs);
  const float least = most * 0x1p-60f;
  return vs < least ? least : vs;  // a NaN stays
}

// l 2^d: in two steps, since 2^d may be below fp32's range where the product is not.
__device__ __forceinline__ float rescaled(float l, float d) {
  const float a = mf::fast_exp2(0.5f * d);
  return l * a * a;
}

// State of 16 query rows in one wave: the lane's row is lane % 16.
template <int D>
struct Acc {
  f4 o[D / 16];  // channels 16 n + 4 (lane / 16) + i
  float m, l;    // reference; the lane's part of the sum
};

template <int D, int CODE, bool MASK>
__device__ __forceinline__ void softmax_step(Acc<D> &acc, const f4 (&s)[4], float factor, float ks, float vs,
                                             int32_t seen, h8 (&p)[2]) {
  const float c = ks * factor, lv = __builtin_amdgcn_logf(vs);
  float x[16], top = mf::kNegInf;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    x[j] = __builtin_fmaf(s[j / 4][j % 4], c, lv);
    if constexpr (MASK) x[j] = j < seen ? x[j] : mf::kNegInf;
    top = fmaxf(top, x[j]);
  }
  top = mf::max_over_slices(top);
  if (__any(top > acc.m + kRaise || (acc.m == mf::kNegInf && top > acc.m))) {
    const float m = fmaxf(acc.m, top);
    const float d = m == mf::kNegInf ? 0.0f : acc.m - m, alpha = mf::fast_exp2(d);
    acc.m = m;
    acc.l = rescaled(acc.l, d);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) acc.o[n] *= alpha;
  }
  const float m = acc.m == mf::kNegInf ? 0.0f : acc.m;
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float e = mf::fast_exp2(x[j] - m);
    sum += e;
    p[j / 8][j % 8] = mf::to_h(e);
  }
  // a lane that sees none of its keys adds nothing, whatever the block's scale holds
  acc.l += sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_rcpf(vs);
}

template <int D, int CODE, int NR>
__global__ __launch_bounds__(256, 2) void rows_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse,
                                                      float *part, float *stat) {
  constexpr int kPitch = D + 4;
  __shared__ float sh_o[4][16][kPitch];
  __shared__ float sh_m[4][16], sh_l[4][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15,
            quad = lane >> 4;
  const int32_t split = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  const Rows w = rows_of(c, q, p, unit, 16 * NR);
  const int32_t tiles = tiles_of(c, p, w), per = split_tiles_of(p, tiles);
  const int32_t begin = split * per, end = begin + per < tiles ? begin + per : tiles;
  if (begin >= end && split > 0) return;  // the first split of rows without keys writes what they get
  const int64_t sh = int64_t(w.s) * c.heads + w.h;
  const int32_t *list = p.list == nullptr ? nullptr : p.list + ((int64_t(w.s) * p.runs + w.run0 / p.run) * c.heads + w.h) * p.budget;

  h8 frag[NR][D / 32];
  float factor[NR];
  int32_t row_end[NR];
  Acc<D> acc[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int32_t r = w.r0 + 16 * n + col;
    factor[n] = load_query<D>(q, w, r, frag[n]);
    row_end[n] = visible(q, w.length, w.count, w.run0 + r / q.group);
    row_end[n] = row_end[n] < w.length ? row_end[n] : w.length;
    acc[n].m = mf::kNegInf;
    acc[n].l = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[n].o[d] = f4{0, 0, 0, 0};
  }
  const int32_t tokens = c.blocks << c.shift;
  Lane<D> l;
  l.key = (quad & 1) * 16;
  l.kcode = c.key_code + sh * tokens * D + (((col >> 2) & 1) * 16 + (col & 3)) * D + quad * 16;
  l.vcode = c.value_code + sh * tokens * D + col * c.block + l.key;
  l.kscale = c.key_scale + sh * c.blocks;
  l.vscale = c.value_scale + sh * c.blocks;

  float most = 0.0f;  // the largest value scale so far
  Raw<D> raw;
  int32_t t = begin + wave, t0 = 0, t1 = 0;
  if (t < end) {
    t0 = half_of(c, p, list, 2 * t);
    t1 = half_of(c, p, list, 2 * t + 1);
    // a tile's second half may lie behind the capacity
    if (t1 >= tokens) t1 = kNone;
    load_keys(raw, c, l, t0, t1);
    load_values(raw, c, l, t0, t1);
  }
  for (; t < end; t += 4) {
    int32_t n0 = kNone, n1 = kNone;
    const bool more = t + 4 < end;
    if (more) {
      n0 = half_of(c, p, list, 2 * (t + 4));
      n1 = half_of(c, p, list, 2 * (t + 4) + 1);
      if (n1 >= tokens) n1 = kNone;
    }
    f4 s[NR][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][j] = f4{0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        const h8 a = codes_to_h8<CODE>(raw.k[j][x].x, raw.k[j][x].y), b = codes_to_h8<CODE>(raw.k[j][x].z, raw.k[j][x].w);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          s[n][j] = mf::mfma32(a, frag[n][2 * x], s[n][j]);
          s[n][j] = mf::mfma32(b, frag[n][2 * x + 1], s[n][j]);
        }
      }
    }
    const int32_t mine = ((quad & 2) ? t1 : t0) + l.key;  // the lane's first key
    const float ks = raw.ks, vs = counted_scale(mine < w.length ? raw.vs : 1.0f, most);
    if (more) load_keys(raw, c, l, n0, n1);
    h8 pr[NR][2];
    const int32_t last = t0 > t1 ? t0 : t1;
    if (last + 32 <= w.end_first) {
#pragma unroll
      for (int n = 0; n < NR; ++n) softmax_step<D, CODE, false>(acc[n], s[n], factor[n], ks, vs, 16, pr[n]);
    } else {
#pragma unroll
      for (int n = 0; n < NR; ++n) softmax_step<D, CODE, true>(acc[n], s[n], factor[n], ks, vs, row_end[n] - mine, pr[n]);
      // codes behind the length are no values: a zero weight must not meet them
#pragma unroll
      for (int d = 0; d < D / 16; ++d) raw.v[d] = first_bytes(raw.v[d], w.length - mine);
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const h8 a = codes_to_h8<CODE>(raw.v[d].x, raw.v[d].y), b = codes_to_h8<CODE>(raw.v[d].z, raw.v[d].w);
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        acc[n].o[d] = mf::mfma32(a, pr[n][0], acc[n].o[d]);
        acc[n].o[d] = mf::mfma32(b, pr[n][1], acc[n].o[d]);
      }
    }
    if (more) load_values(raw, c, l, n0, n1);
    t0 = n0;
    t1 = n1;
  }

  // join the waves: 16 threads a row, D / 16 channels each
  constexpr int kC = D / 16;
  const int row = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * kC;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const float l_row = mf::sum_over_slices(acc[n].l);
    if (n > 0) __syncthreads();
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f4 *>(&sh_o[wave][col][16 * d + 4 * quad]) = acc[n].o[d];
    if (quad == 0) {
      sh_m[wave][col] = acc[n].m;
      sh_l[wave][col] = l_row;
    }
    __syncthreads();
    float m = mf::kNegInf;
#pragma unroll
    for (int v = 0; v < 4; ++v) m = fmaxf(m, sh_m[v][row]);
    float total = 0.0f, o[kC];
#pragma unroll
    for (int j = 0; j < kC; ++j) o[j] = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float mv = sh_m[v][row];
      const float d = mv == mf::kNegInf && !(sh_l[v][row] != 0.0f) ? mf::kNegInf : mv - m, f = mf::fast_exp2(d);
      total += rescaled(sh_l[v][row], d);
#pragma unroll
      for (int j = 0; j < kC; ++j) o[j] += f * sh_o[v][row][c0 + j];
    }
    const int32_t r = w.r0 + 16 * n + row;
    if (p.splits > 1) {
      const int64_t at = (int64_t(blockIdx.x) * (16 * NR) + 16 * n + row);
#pragma unroll
      for (int j = 0; j < kC; j += 4) {
        *reinterpret_cast<f4 *>(part + at * D + c0 + j) = f4{o[j], o[j + 1], o[j + 2], o[j + 3]};
      }
      if (c0 == 0) {
        stat[2 * at] = m;
        stat[2 * at + 1] = total;
      }
    } else if (r < w.run_rows) {
      const int32_t token = w.run0 + r / q.group, head = w.h * q.group + r % q.group;
      const bool none = token >= w.count || total == 0.0f;
      const float f = none ? 0.0f : 1.0f / total;
      uint16_t *dst = out + ((int64_t(w.s) * q.len + token) * q.heads + head) * D + c0;
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        const float v = none ? 0.0f : o[j] * f;
        dst[j] = q.fp16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v);
      }
      if (c0 == 0 && lse != nullptr) {
        lse[(int64_t(w.s) * q.heads + head) * q.len + token] =
            none ? mf::kNegInf : kLn2 * (m + __builtin_amdgcn_logf(total));
      }
    }
  }
}

// Join the splits of 16 NR rows: one wave per row.
template <int D, int NR>
__global__ __launch_bounds__(256) void join_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse,
                                                   const float *part, const float *stat) {
  constexpr int kC = D / 64;
  const int lane = threadIdx.x & 63;
  const int32_t index = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int32_t unit = index / (16 * NR), rr = index % (16 * NR);
  if (unit >= c.sequences * c.heads * p.runs * p.groups) return;
  const Rows w = rows_of(c, q, p, unit, 16 * NR);
  const int32_t r = w.r0 + rr;
  if (r >= w.run_rows) return;
  const int32_t tiles = tiles_of(c, p, w), per = split_tiles_of(p, tiles);
  const int32_t splits = tiles == 0 ? 1 : (tiles + per - 1) / per;
  const int64_t base = int64_t(unit) * p.splits * (16 * NR) + rr;
  float m = mf::kNegInf;
  for (int32_t i = lane; i < splits; i += 64) m = fmaxf(m, stat[2 * (base + int64_t(i) * (16 * NR))]);
  m = wave_max(m);
  float total = 0.0f, o[kC] = {};
  for (int32_t i = 0; i < splits; ++i) {
    const int64_t at = base + int64_t(i) * (16 * NR);
    const float mi = stat[2 * at], li = stat[2 * at + 1];
    if (mi == mf::kNegInf && !(li != 0.0f)) continue;
    const float f = mf::fast_exp2(mi - m);
    total += rescaled(li, mi - m);
#pragma unroll
    for (int j = 0; j < kC; ++j) o[j] += f * part[at * D + lane * kC + j];
  }
  const int32_t token = w.run0 + r / q.group, head = w.h * q.group + r % q.group;
  const bool none = token >= w.count || total == 0.0f;
  uint16_t *dst = out + ((int64_t(w.s) * q.len + token) * q.heads + head) * D + lane * kC;
#pragma unroll
  for (int j = 0; j < kC; ++j) {
    const float v = none ? 0.0f : o[j] / total;
    dst[j] = q.fp16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v);
  }
  if (lane == 0 && lse != nullptr) {
    lse[(int64_t(w.s) * q.heads + head) * q.len + token] = none ? mf::kNegInf : kLn2 * (m + __builtin_amdgcn_logf(total));
  }
}

int make_plan(const uc_block8_cache *cache, const uc_block8_query *query, int64_t budget, int64_t query_block,
              const char *what, Query &q, Plan &p, int &nr) {
  UC_REQUIRE(query != nullptr, "%s: query is NULL", what);
  UC_REQUIRE(half_dtype(query->dtype), "%s: queries must be bf16 or fp16", what);
  UC_REQUIRE(query->heads_q > 0 && query->heads_q % cache->heads_kv == 0,
             "%s: query heads must be a multiple of KV heads", what);
  UC_REQUIRE(query->query_len >= 0 && query->query_len < (1 << 24), "%s: bad query_len", what);
  UC_REQUIRE(query->heads_q / cache->heads_kv * query->query_len < (int64_t(1) << 30), "%s: too many query rows", what);
  UC_REQUIRE(query->max_tokens >= 0, "%s: negative max_tokens", what);
  UC_REQUIRE(budget >= 0 && budget < (1 << 24), "%s: bad budget", what);
  UC_REQUIRE(budget == 0 || query_block > 0, "%s: query_block must be positive", what);
  q = Query{static_cast<const uint16_t *>(query->query), query->q_ss, query->q_st, query->q_sh, query->query_lengths,
            static_cast<int32_t>(query->query_len), static_cast<int32_t>(query->heads_q),
            static_cast<int32_t>(query->heads_q / cache->heads_kv), query->dtype == UC_FP16, query->causal != 0, 0.0f};
  p.list = nullptr;
  p.budget = static_cast<int32_t>(budget);
  const int64_t run = budget == 0 || query_block > query->query_len ? (query->query_len > 0 ? query->query_len : 1)
                                                                     : query_block;
  p.run = static_cast<int32_t>(run);
  p.runs = static_cast<int32_t>(ceil_div(query->query_len, run));
  const int64_t rows = run * q.group;
  nr = rows > 16 ? 2 : 1;
  p.groups = static_cast<int32_t>(ceil_div(rows, 16 * nr));
  // keys that the launch expects a row to read
  const int64_t capacity = cache->blocks * cache->block_tokens;
  int64_t keys = query->max_tokens < capacity ? query->max_tokens : capacity;
  if (budget > 0) keys = budget * cache->block_tokens;
  const int64_t tiles = keys > 0 ? ceil_div(keys, kTile) : 1;
  const int64_t units = cache->sequences * cache->heads_kv * p.runs * p.groups;
  // about 1024 workgroups (four a CU), each wave with a tile at least
  int64_t splits = units > 0 ? 1024 / units : 1;
  const int64_t most = ceil_div(tiles, 4);
  splits = splits < 1 ? 1 : splits > most ? most : splits;
  p.split_tiles = static_cast<int32_t>(ceil_div(tiles, splits));
  p.splits = static_cast<int32_t>(ceil_div(tiles, p.split_tiles));
  UC_REQUIRE(units * p.splits < (int64_t(1) << 31) / (16 * nr), "%s: too many query rows", what);
  return UC_OK;
}

// Floats of the splits' partial outputs and statistics.
int64_t part_rows(const uc_block8_cache *cache, const Plan &p, int nr) {
  return p.splits > 1 ? cache->sequences * cache->heads_kv * p.runs * p.groups * p.splits * 16 * nr : 0;
}

}  // namespace
}  // namespace b8
}  // namespace uc

extern "C" int64_t uc_block8_attn_workspace_bytes(const uc_block8_cache *cache, const uc_block8_query *query,
                                                  int64_t budget, int64_t query_block) {
  using namespace uc::b8;
  Cache c;
  Query q;
  Plan p;
  int nr;
  if (check_cache(cache, "uc_block8_attn", c) ||
      make_plan(cache, query, budget, query_block, "uc_block8_attn", q, p, nr))
    return -1;
  return part_rows(cache, p, nr) * (cache->head_dim + 2) * int64_t(sizeof(float));
}

extern "C" int uc_block8_attn(const uc_block8_cache *cache, const uc_block8_query *query, const int32_t *blocks,
                              int64_t budget, int64_t query_block, float sm_scale, void *out, float *lse,
                              void *workspace, int64_t workspace_bytes, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::b8;
  Cache c;
  Query q;
  Plan p;
  int nr;
  if (int rc = check_cache(cache, "uc_block8_attn", c)) return rc;
  if (int rc = make_plan(cache, query, budget, query_block, "uc_block8_attn", q, p, nr)) return rc;
  UC_REQUIRE((blocks != nullptr) == (budget > 0), "uc_block8_attn: a block list and its budget belong together");
  UC_REQUIRE(sm_scale > 0.0f && sm_scale < __builtin_huge_valf(), "uc_block8_attn: sm_scale must be positive");
  if (q.len == 0) return UC_OK;
  UC_REQUIRE(q.p != nullptr && (reinterpret_cast<uintptr_t>(q.p) & 15) == 0 && ((q.ss | q.st | q.sh) & 7) == 0,
             "uc_block8_attn: query must be 16-byte aligned with strides that are multiples of 8");
  UC_REQUIRE(out != nullptr && (reinterpret_cast<uintptr_t>(out) & 15) == 0, "uc_block8_attn: out must be 16-byte aligned");
  const int64_t rows = part_rows(cache, p, nr);
  UC_REQUIRE(rows == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                           workspace_bytes >= rows * (cache->head_dim + 2) * int64_t(sizeof(float))),
             "uc_block8_attn: workspace too small");
  p.list = blocks;
  q.scale = sm_scale * kLog2e;
  float *part = static_cast<float *>(workspace), *stat = part + rows * cache->head_dim;
  const int64_t units = cache->sequences * cache->heads_kv * p.runs * p.groups;
  return UC_B8_DISPATCH(cache, cache->head_dim, [&] {
    auto launch = [&](auto nr_tag) {
      constexpr int NR = decltype(nr_tag)::value;
      hipLaunchKernelGGL((rows_kernel<D, CODE, NR>), dim3(static_cast<uint32_t>(units * p.splits)), dim3(256), 0,
                         as_stream(stream), c, q, p, static_cast<uint16_t *>(out), lse, part, stat);
      int rc = check_launch("uc_block8_attn");
      if (rc != UC_OK || p.splits == 1) return rc;
      hipLaunchKernelGGL((join_kernel<D, NR>), dim3(static_cast<uint32_t>(ceil_div(units * 16 * NR, 4))), dim3(256), 0,
                         as_stream(stream), c, q, p, static_cast<uint16_t *>(out), lse, part, stat);
      return check_launch("uc_block8_attn (join)");
    };
    if (nr == 1) return launch(std::integral_constant<int, 1>());
    return launch(std::integral_constant<int, 2>());
  });
}
