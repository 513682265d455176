// Attention over the 8-bit block-scaled cache for few query rows, by split keys:
// a workgroup takes up to 16 NR query rows of one KV head (its query heads x
// query tokens) and a run of 64-key tiles, its four waves alternate tiles, and what
// they hold is joined at the end; a second launch joins the workgroups' parts.
//
// Mathematics, per row r and key t of block b, in base 2:
//   x = (q_r . k_t) ks_b sm_scale log2(e) + log2(vs_b)
//   P = 2^(x - m), O = sum P v_code, l = sum P / vs_b, out = O / l, lse = ln2 (m + log2 l)
// so both scales cost nothing per key: the key's scale is the factor that the
// logit needs anyway and the value's scale is an addend of the exponent.  m is a
// running reference of x (not of the logit): P stays in fp16's range
// whatever the blocks' scales are, and its rounding (half a step, 2^-11) is
// relative to the largest contribution.  Sums, m and O are fp32.  A block whose
// value scale is less than 2^-60 of another that the row has seen (a block of zeros has
// 2^-60, another program's 0) counts as 2^-60 of that one: its weights then keep their place in l, and
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
//
// Bound by HBM: each code is read once, straight into registers, a wave's next 64 keys (16 KB at 128
// channels) on their way while it computes on the present ones, 128 KB in flight a CU.  Of 8 sequences
// of 32k tokens (28/4 heads, 269 MB) the first launch takes 42 us from back to back calls (6.4 TB/s,
// part of it from the last-level cache), both 56 over changing inputs (4.8 TB/s; a large copy
// 4.9).  Small calls are two launches: 2k tokens 7.1 + 4.8 us.
#include "uc_block8_attn.h"

#include <type_traits>

namespace uc {
namespace b8 {
namespace {

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
  float x[MASK ? 16 : 1], top = mf::kNegInf;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if constexpr (MASK) {
      x[j] = j < seen ? __builtin_fmaf(s[j / 4][j % 4], c, lv) : mf::kNegInf;
      top = fmaxf(top, x[j]);
    } else {
      top = fmaxf(top, s[j / 4][j % 4]);
    }
  }
  if constexpr (!MASK) top = __builtin_fmaf(top, c, lv);
  top = mf::max_over_slices(top);
  if (__any(top > acc.m + kRaise)) {
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
    const float e = mf::fast_exp2(MASK ? x[MASK ? j : 0] - m : __builtin_fmaf(s[j / 4][j % 4], c, lv - m));
    sum += e;
    p[j / 8][j % 8] = mf::to_h(e);
  }
  // a lane that sees none of its keys adds nothing, whatever the block's scale holds
  acc.l += sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_rcpf(vs);
}

// LDS of the waves' join; and with 32 rows of 128 channels or 48 of 64 the query fragments, which do not fit
// the registers beside the rest (they spilled: 8 x 32k tokens, 28 rows, 149 us).
template <int D, int NR>
struct Joined {
  static constexpr bool kHeld = NR * D >= 192;
  float o[4][16][D + 4];
  float m[4][16], l[4][16];
  h8 frag[kHeld ? NR * D / 32 : 1][64];
};

// Tiles begin .. end - 1 of the rows w, by a whole workgroup.  slot >= 0: the part goes there; else it
// is all there is, and the rows are finished.
template <int D, int CODE, int NR>
__device__ __forceinline__ void piece(const Cache &c, const Query &q, const Plan &p, const Rows &w, int32_t begin, int32_t end,
                                      int32_t slot, Joined<D, NR> &joined, uint16_t *out, float *lse, float *part,
                                      float *stat) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15,
            quad = lane >> 4;
  const int64_t sh = int64_t(w.s) * c.heads + w.h;
  BlockList list(c, p, w);
  auto half = [&](int32_t i) { return p.list != nullptr ? half_of<true>(c, list, i) : half_of<false>(c, list, i); };

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
    t0 = half(2 * t);
    t1 = half(2 * t + 1);
    load_keys(raw, c, l, t0, t1);
    load_values(raw, c, l, t0, t1);
  }
  h8 frag[NR][D / 32];
  float factor[NR];
  int32_t row_end[NR];
  Acc<D> acc[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int32_t r = w.r0 + 16 * n + col;
    factor[n] = load_query<D, true>(q, w, r, frag[n]);
    row_end[n] = visible(q, w.length, w.count, w.run0 + token_of(q, r));
    row_end[n] = row_end[n] < w.length ? row_end[n] : w.length;
    acc[n].m = mf::kNegInf;
    acc[n].l = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[n].o[d] = f4{0, 0, 0, 0};
  }
  if constexpr (Joined<D, NR>::kHeld) {
    __syncthreads();  // the fragments of the piece before have been read
    if (wave == 0) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k) joined.frag[n * (D / 32) + k][lane] = frag[n][k];
      }
    }
    __syncthreads();
  }
  auto step = [&](auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    int at = lane;  // opaque, so that the fragments are read in every tile and not kept
    if constexpr (Joined<D, NR>::kHeld) asm volatile("" : "+v"(at));
    auto query = [&](int n, int k) { return Joined<D, NR>::kHeld ? joined.frag[n * (D / 32) + k][at] : frag[n][k]; };
    int32_t n0 = kNone, n1 = kNone;
    const bool more = t + 4 < end;
    if (more) {
      n0 = half(2 * (t + 4));
      n1 = half(2 * (t + 4) + 1);
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
          s[n][j] = mf::mfma32(a, query(n, 2 * x), s[n][j]);
          s[n][j] = mf::mfma32(b, query(n, 2 * x + 1), s[n][j]);
        }
      }
    }
    const int32_t half0 = (quad & 2) ? t1 : t0, other0 = (quad & 2) ? t0 : t1;  // first keys of the lane's half and of the other
    const int32_t mine = half0 + l.key;                                        // the lane's first key
    const float ks = raw.ks, vs = raw.vs;
    // the scale of the other half, whose lanes share the rows' references
    float vo = vs;
    if (c.shift == 5) vo = __shfl_xor(vs, 32, kWave);
    if (more) load_keys(raw, c, l, n0, n1);
    h8 pr[NR][2];
    if constexpr (!MASK) most = larger_scale(larger_scale(most, vs), vo);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float counted = counted_scale(vs, most);
      if constexpr (MASK) {
        // blocks that the row does not see are nothing to go by (later tiles are for rows that see all of this one)
        float seen = half0 < row_end[n] ? larger_scale(most, vs) : most;
        seen = other0 < row_end[n] ? larger_scale(seen, vo) : seen;
        counted = half0 < row_end[n] ? counted_scale(vs, seen) : 1.0f;
      }
      softmax_step<D, CODE, MASK>(acc[n], s[n], factor[n], ks, counted, row_end[n] - mine, pr[n]);
    }
    if constexpr (MASK) {
      most = half0 < w.length ? larger_scale(most, vs) : most;
      most = other0 < w.length ? larger_scale(most, vo) : most;
    }
    if constexpr (MASK) {
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
    t += 4;
  };
  // tiles that every row sees come first; from the first other one on, every tile is masked
  while (t < end && (t0 > t1 ? t0 : t1) + 32 <= w.end_first) step(std::false_type());
  while (t < end) step(std::true_type());

  // join the waves: 16 threads a row, D / 16 channels each
  constexpr int kC = D / 16;
  const int row = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * kC;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const float l_row = mf::sum_over_slices(acc[n].l);
    __syncthreads();  // what was joined before has been read
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f4 *>(&joined.o[wave][col][16 * d + 4 * quad]) = acc[n].o[d];
    if (quad == 0) {
      joined.m[wave][col] = acc[n].m;
      joined.l[wave][col] = l_row;
    }
    __syncthreads();
    float m = mf::kNegInf;
#pragma unroll
    for (int v = 0; v < 4; ++v) m = fmaxf(m, joined.m[v][row]);
    float total = 0.0f, o[kC];
#pragma unroll
    for (int j = 0; j < kC; ++j) o[j] = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float mv = joined.m[v][row];
      const float d = mv == mf::kNegInf && !(joined.l[v][row] != 0.0f) ? mf::kNegInf : mv - m, f = mf::fast_exp2(d);
      total += rescaled(joined.l[v][row], d);
#pragma unroll
      for (int j = 0; j < kC; ++j) o[j] += f * joined.o[v][row][c0 + j];
    }
    const int32_t r = w.r0 + 16 * n + row;
    if (slot >= 0) {
      if (r >= w.run_rows) continue;
      const int64_t at = int64_t(slot) * (16 * NR) + 16 * n + row;
#pragma unroll
      for (int j = 0; j < kC; j += 4) {
        *reinterpret_cast<f4 *>(part + at * D + c0 + j) = f4{o[j], o[j + 1], o[j + 2], o[j + 3]};
      }
      if (c0 == 0) {
        stat[2 * at] = m;
        stat[2 * at + 1] = total;
      }
    } else if (r < w.run_rows) {
      const int32_t token = w.run0 + token_of(q, r), head = w.h * q.group + r - token_of(q, r) * q.group;
      const bool none = token >= w.count || total == 0.0f;
      const float f = none ? 0.0f : 1.0f / total;
      uint16_t *dst = out + ((int64_t(w.s) * q.len + token) * q.heads + head) * D + c0;
#pragma unroll
      for (int j = 0; j < kC; j += 2) {
        *reinterpret_cast<uint32_t *>(dst + j) = none ? 0u : pack2(o[j] * f, o[j + 1] * f, q.fp16);
      }
      if (c0 == 0 && lse != nullptr) {
        lse[(int64_t(w.s) * q.heads + head) * q.len + token] =
            none ? mf::kNegInf : kLn2 * (m + __builtin_amdgcn_logf(total));
      }
    }
  }
}

template <int D, int CODE, int NR>
__global__ __launch_bounds__(256, 2) void rows_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse,
                                                      float *part, float *stat) {
  __shared__ Joined<D, NR> joined;
  if (p.workgroups == 0) {  // one workgroup a unit
    const Rows w = rows_of(c, q, p, blockIdx.x, 16 * NR);
    piece<D, CODE, NR>(c, q, p, w, 0, tiles_of(c, p, w), -1, joined, out, lse, part, stat);
    return;
  }
  // this workgroup's steps, and the sequence, unit and step that they begin at
  const int lane = threadIdx.x & 63;
  const int32_t g = blockIdx.x, each = c.heads * p.runs;
  int32_t s0 = 0, first = 0;  // sequences s0 .. s0 + 63 are in the lanes, `first` of them is the present one
  int32_t length = 0, count = 0, steps = 0, sum = 0, total;
  auto fill = [&] {
    const int32_t i = s0 + lane;
    length = i < c.sequences ? c.length(i) : 0;
    count = i < c.sequences ? q.count(i) : 0;
    steps = i < c.sequences ? steps_of(keys_of(c, p, length, count)) : 0;
    sum = wave_prefix(steps);
  };
  fill();
  total = c.sequences <= 64 ? __builtin_amdgcn_readlane(sum, 63) : steps_before(c, q, p, 0).total;
  total *= each;
  const int32_t per = per_of(p, total);
  int32_t at = g * per;
  const int32_t stop = at + per < total ? at + per : total;
  if (at >= stop) return;
  int32_t rest = at;  // steps of the present sequence before `at`
  for (;;) {
    const uint64_t past = __ballot(sum * each > rest);
    if (past != 0) {
      first = __builtin_ctzll(past);
      break;
    }
    rest -= __builtin_amdgcn_readlane(sum, 63) * each;
    s0 += 64;
    fill();
  }
  int32_t now = __builtin_amdgcn_readlane(steps, first);  // steps of each of the sequence's units
  rest -= (__builtin_amdgcn_readlane(sum, first) - now) * each;
  int32_t n = rest / now, t = rest - n * now;  // the unit within the sequence, and its step
  while (at < stop) {
    const int32_t end = now - t < stop - at ? now : t + (stop - at), s = s0 + first;
    const int32_t h = p.runs == 1 ? n : n / p.runs, run = p.runs == 1 ? 0 : n % p.runs;
    const Rows w = rows_at(q, p, s, h, run, 0, 16 * NR, __builtin_amdgcn_readlane(length, first),
                           __builtin_amdgcn_readlane(count, first));
    // (the step's end may lie behind the last tile)
    piece<D, CODE, NR>(c, q, p, w, t, min(end, tiles_of(c, p, w)), g + s * each + n, joined, out, lse, part, stat);
    at += end - t;
    t = 0;
    if (++n == each && at < stop) {
      n = 0;
      do {
        if (++first == 64) {
          first = 0;
          s0 += 64;
          fill();
        }
        now = __builtin_amdgcn_readlane(steps, first);
      } while (now == 0);
    }
  }
}

// Where a query row's parts are: `count` slots from `first` on.
struct Parts {
  Rows w;
  int32_t r;
  int32_t first, count;
};

__device__ __forceinline__ Parts parts_of(const Cache &c, const Query &q, const Plan &p, int64_t index) {
  Parts x;
  // rows of the runs in order: (sequence, head, run, row)
  const int32_t full = p.run * q.group;
  const int64_t at = index / full;
  x.r = static_cast<int32_t>(index - at * full);
  const int32_t run = p.runs == 1 ? 0 : static_cast<int32_t>(at % p.runs);
  const int32_t sh = static_cast<int32_t>(p.runs == 1 ? at : at / p.runs), s = sh / c.heads;
  const int32_t group = p.groups == 1 ? 0 : x.r / p.rows;
  x.w = rows_at(q, p, s, sh - s * c.heads, run, group, p.rows, c.length(s), q.count(s));
  const int32_t unit = static_cast<int32_t>(at) * p.groups + group;
  if (p.workgroups == 0) {
    const int32_t tiles = tiles_of(c, p, x.w), per = split_tiles_of(p, tiles);
    x.first = unit * p.splits;
    x.count = tiles == 0 ? 1 : (tiles + per - 1) / per;
  } else {
    const Steps steps = steps_before(c, q, p, s);
    const int32_t each = c.heads * p.runs, n = unit - s * each, per = per_of(p, steps.total * each);
    const int32_t start = steps.before * each + n * steps.mine;
    x.first = steps.mine == 0 ? 0 : start / per + unit;
    x.count = steps.mine == 0 ? 0 : (start + steps.mine - 1) / per + unit - x.first + 1;
  }
  return x;
}

// Join the parts of a query row.  16 lanes take every STRIDE-th part from `begin` on, D / 16 channels each, two
// parts' loads in flight; the outcome is relative to m, the largest reference of all.
template <int D>
struct Sum {
  float o[D / 16];
  float m, l;
};

template <int D, int STRIDE>
__device__ __forceinline__ Sum<D> sum_parts(const Plan &p, const Parts &x, int32_t begin, const float *part, const float *stat) {
  constexpr int kC = D / 16;
  const int lane = threadIdx.x & 15;
  const int64_t base = int64_t(x.first) * p.rows + (x.r - x.w.r0);
  Sum<D> t;
  t.m = mf::kNegInf;
  t.l = 0.0f;
#pragma unroll
  for (int j = 0; j < kC; ++j) t.o[j] = 0.0f;
  float mi[2], li[2];
  f4 oi[2][kC / 4];
  auto load = [&](int32_t i0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int32_t i = i0 + u * STRIDE;
      const int64_t at = base + int64_t(i < x.count ? i : i0) * p.rows;
      mi[u] = stat[2 * at];
      li[u] = stat[2 * at + 1];
#pragma unroll
      for (int j = 0; j < kC / 4; ++j) oi[u][j] = *reinterpret_cast<const f4 *>(part + at * D + lane * kC + 4 * j);
    }
  };
  if (begin < x.count) load(begin);  // on their way while the largest reference is found
  for (int32_t i = lane; i < x.count; i += 16) t.m = fmaxf(t.m, stat[2 * (base + int64_t(i) * p.rows)]);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) t.m = fmaxf(t.m, __shfl_xor(t.m, o, kWave));
  for (int32_t i0 = begin; i0 < x.count;) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // a part past the end, or one whose keys the row does not see
      if (i0 + u * STRIDE >= x.count || (mi[u] == mf::kNegInf && !(li[u] != 0.0f))) continue;
      const float d = mi[u] - t.m, f = mf::fast_exp2(d);
      t.l += rescaled(li[u], d);
#pragma unroll
      for (int j = 0; j < kC; ++j) t.o[j] += f * oi[u][j / 4][j % 4];
    }
    i0 += 2 * STRIDE;
    if (i0 < x.count) load(i0);
  }
  return t;
}

template <int D>
__device__ __forceinline__ void finish_row(const Query &q, const Parts &x, const Sum<D> &t, uint16_t *out, float *lse) {
  constexpr int kC = D / 16;
  const int lane = threadIdx.x & 15;
  const int32_t g = token_of(q, x.r), token = x.w.run0 + g, head = x.w.h * q.group + x.r - g * q.group;
  const bool none = token >= x.w.count || t.l == 0.0f;
  const float f = 1.0f / t.l;
  uint32_t v[kC / 2];
#pragma unroll
  for (int j = 0; j < kC / 2; ++j) v[j] = none ? 0u : pack2(t.o[2 * j] * f, t.o[2 * j + 1] * f, q.fp16);
  uint16_t *dst = out + ((int64_t(x.w.s) * q.len + token) * q.heads + head) * D + lane * kC;
  if constexpr (kC == 8) {
    *reinterpret_cast<uint4 *>(dst) = uint4{v[0], v[1], v[2], v[3]};
  } else {
    *reinterpret_cast<uint2 *>(dst) = uint2{v[0], v[1]};
  }
  if (lane == 0 && lse != nullptr) {
    lse[(int64_t(x.w.s) * q.heads + head) * q.len + token] = none ? mf::kNegInf : kLn2 * (t.m + __builtin_amdgcn_logf(t.l));
  }
}

// Few parts a row: a wave joins four rows.
template <int D>
__global__ __launch_bounds__(256) void join_few_kernel(Cache c, Query q, Plan p, int64_t rows, uint16_t *out, float *lse,
                                                       const float *part, const float *stat) {
  const int64_t index = int64_t(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const Parts x = parts_of(c, q, p, index < rows ? index : rows - 1);  // (whole waves: they sum up lengths)
  if (index >= rows || x.r >= x.w.run_rows) return;
  finish_row<D>(q, x, sum_parts<D, 1>(p, x, 0, part, stat), out, lse);
}

// Many: a workgroup joins one row, its 16-lane groups every 16th part.
template <int D>
__global__ __launch_bounds__(256) void join_many_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse,
                                                        const float *part, const float *stat) {
  constexpr int kC = D / 16;
  __shared__ float sh_o[16][D], sh_l[16];
  const Parts x = parts_of(c, q, p, blockIdx.x);
  if (x.r >= x.w.run_rows) return;
  const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
  Sum<D> t = sum_parts<D, 16>(p, x, group, part, stat);
#pragma unroll
  for (int j = 0; j < kC; ++j) sh_o[group][lane * kC + j] = t.o[j];
  if (lane == 0) sh_l[group] = t.l;
  __syncthreads();
  if (group > 0) return;
  for (int g = 1; g < 16 && g < x.count; ++g) {
    t.l += sh_l[g];
#pragma unroll
    for (int j = 0; j < kC; ++j) t.o[j] += sh_o[g][lane * kC + j];
  }
  finish_row<D>(q, x, t, out, lse);
}

template <int D, int CODE, class... Args>
void launch_rows(int32_t rows, uint32_t workgroups, hipStream_t stream, const Args &...args) {
  if (rows == 16) {
    hipLaunchKernelGGL((rows_kernel<D, CODE, 1>), dim3(workgroups), dim3(256), 0, stream, args...);
  } else if (rows == 32) {
    hipLaunchKernelGGL((rows_kernel<D, CODE, 2>), dim3(workgroups), dim3(256), 0, stream, args...);
  } else if constexpr (D == 64) {
    hipLaunchKernelGGL((rows_kernel<D, CODE, 3>), dim3(workgroups), dim3(256), 0, stream, args...);
  }
}

// Splits of 128-row workgroups, and how many groups of four waves they have: the least time in
// tiles.  Of one group, two (head_dim 128) or three workgroups share a CU, and up to one a CU takes
// 0.65 of the time a tile; of two groups one, each with half of the tiles, joined in LDS (one
// tile).  The launch that joins splits takes two tiles and 0.006 for each part of a workgroup.  Measured, one split -> the chosen: 112 units of 64 tiles 110 -> 56 us (4 splits), 28 of 256
// 412 -> 59 (18), 572 of 64 247 -> 213 (4), 376 of 128 at head_dim 64 196 -> 151 (2); 512 of 64 stay at
// one (206; two would take 224), as do 440 of 31 (66; 89).
void split_tiles(int64_t units, int64_t tiles, int64_t head_dim, bool listed, Plan &p) {
  const int64_t slots = head_dim == 128 ? 512 : 768;
  int64_t best = 1;
  double least = 1e300;
  const int64_t most = ceil_div(tiles, 4) < 64 ? ceil_div(tiles, 4) : 64;
  for (int64_t k = 1; k <= most; ++k) {
    const double join = k > 1 ? 2.0 + 0.006 * static_cast<double>(units * k) : 0.0;
    const double rounds = units * k <= slots / 2 ? 0.65 : static_cast<double>(ceil_div(units * k, slots));
    const double one = rounds * static_cast<double>(ceil_div(tiles, k)) + join;
    const double two = static_cast<double>(ceil_div(units * k, 256) * ceil_div(tiles, 2 * k)) + 1.0 + join;
    if (one < least) {
      least = one;
      best = k;
      p.key_groups = 1;
    }
    if (two < least && !listed) {
      least = two;
      best = k;
      p.key_groups = 2;
    }
  }
  p.split_tiles = static_cast<int32_t>(ceil_div(tiles, best));
  p.splits = static_cast<int32_t>(ceil_div(tiles, p.split_tiles));
}

constexpr int64_t kShare = 512;  // workgroups that share the tiles of few rows: two a CU

int make_plan(const uc_block8_cache *cache, const uc_block8_query *query, int64_t budget, int64_t query_block,
              const char *what, Query &q, Plan &p) {
  UC_REQUIRE(query != nullptr, "%s: query is NULL", what);
  UC_REQUIRE(half_dtype(query->dtype), "%s: queries must be bf16 or fp16", what);
  UC_REQUIRE(query->heads_q > 0 && query->heads_q % cache->heads_kv == 0,
             "%s: query heads must be a multiple of KV heads", what);
  UC_REQUIRE(query->query_len >= 0 && query->query_len < (1 << 24), "%s: bad query_len", what);
  UC_REQUIRE(query->heads_q < (1 << 24), "%s: too many query heads", what);  // (the products below stay in 64 bits)
  UC_REQUIRE(query->heads_q / cache->heads_kv * query->query_len < (int64_t(1) << 30), "%s: too many query rows", what);
  UC_REQUIRE(query->max_tokens >= 0, "%s: negative max_tokens", what);
  UC_REQUIRE(budget >= 0 && budget <= (1 << 30) / cache->block_tokens, "%s: bad budget", what);
  UC_REQUIRE(budget == 0 || query_block > 0, "%s: query_block must be positive", what);
  q = Query{static_cast<const uint16_t *>(query->query), query->q_ss, query->q_st, query->q_sh, query->query_lengths,
            static_cast<int32_t>(query->query_len), static_cast<int32_t>(query->heads_q),
            static_cast<int32_t>(query->heads_q / cache->heads_kv), query->dtype == UC_FP16, query->causal != 0, 0.0f,
            make_fastdiv(static_cast<uint32_t>(query->heads_q / cache->heads_kv))};
  p.list = nullptr;
  p.budget = static_cast<int32_t>(budget);
  const int64_t run = budget == 0 || query_block > query->query_len ? (query->query_len > 0 ? query->query_len : 1)
                                                                     : query_block;
  p.run = static_cast<int32_t>(run);
  p.runs = static_cast<int32_t>(ceil_div(query->query_len, run));
  const int64_t rows = run * q.group;
  p.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 48 && cache->head_dim == 64 ? 48 : kTileRows;
  p.groups = static_cast<int32_t>(ceil_div(rows, int64_t(p.rows)));
  // keys that the launch expects a row to read
  const int64_t capacity = cache->blocks * cache->block_tokens;
  int64_t keys = query->max_tokens < capacity ? query->max_tokens : capacity;
  if (budget > 0) keys = budget * cache->block_tokens;
  const int64_t tiles = keys > 0 ? ceil_div(keys, kTile) : 1;
  const int64_t units = cache->sequences * cache->heads_kv * p.runs * p.groups;
  p.workgroups = 0;
  p.key_groups = 1;
  if (p.rows == kTileRows) {
    split_tiles(units, tiles, cache->head_dim, budget > 0, p);
  } else {
    p.splits = 1;
    p.split_tiles = 0;
    // lists are of one length, so many of them load the CUs alike
    if (budget == 0 || units < 1024) {
      const int64_t most = ceil_div(tiles, 4) * units;
      p.workgroups = static_cast<int32_t>(most < kShare ? (most > 0 ? most : 1) : kShare);
    }
  }
  // a launch has less than 2^32 threads, and 32-bit counts of tiles
  const bool joins = p.splits > 1 || p.workgroups > 0;
  UC_REQUIRE(units * p.splits < (1 << 24) &&
                 (!joins || cache->sequences * cache->heads_kv * p.runs * p.run * q.group < (1 << 28)),
             "%s: too many query rows", what);
  const int64_t longest = budget > 0 ? keys : capacity;
  UC_REQUIRE(p.workgroups == 0 || units * ceil_div(longest, 4 * kTile) < (1 << 28), "%s: too many keys in all", what);
  return UC_OK;
}

// Floats of the splits' partial outputs and statistics.
int64_t part_rows(const uc_block8_cache *cache, const Plan &p) {
  const int64_t units = cache->sequences * cache->heads_kv * p.runs * p.groups;
  return p.workgroups > 0 ? (units + p.workgroups) * p.rows : p.splits > 1 ? units * p.splits * p.rows : 0;
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
  if (check_cache(cache, "uc_block8_attn", c) ||
      make_plan(cache, query, budget, query_block, "uc_block8_attn", q, p))
    return -1;
  return part_rows(cache, p) * (cache->head_dim + 2) * int64_t(sizeof(float));
}

extern "C" int uc_block8_attn(const uc_block8_cache *cache, const uc_block8_query *query, const int32_t *blocks,
                              int64_t budget, int64_t query_block, float sm_scale, void *out, float *lse,
                              void *workspace, int64_t workspace_bytes, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::b8;
  Cache c;
  Query q;
  Plan p;
  if (int rc = check_cache(cache, "uc_block8_attn", c)) return rc;
  if (int rc = make_plan(cache, query, budget, query_block, "uc_block8_attn", q, p)) return rc;
  // (times log2(e) it stays in fp32's range)
  UC_REQUIRE(sm_scale > 0.0f && sm_scale <= 0x1p127f, "uc_block8_attn: sm_scale must be positive, and 2^127 at most");
  if (q.len == 0) return UC_OK;
  UC_REQUIRE((blocks != nullptr) == (budget > 0), "uc_block8_attn: a block list and its budget belong together");
  UC_REQUIRE(q.p != nullptr && (reinterpret_cast<uintptr_t>(q.p) & 15) == 0 && ((q.ss | q.st | q.sh) & 7) == 0,
             "uc_block8_attn: query must be 16-byte aligned with strides that are multiples of 8");
  UC_REQUIRE(out != nullptr && (reinterpret_cast<uintptr_t>(out) & 15) == 0, "uc_block8_attn: out must be 16-byte aligned");
  const int64_t rows = part_rows(cache, p);
  UC_REQUIRE(rows == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                           workspace_bytes >= rows * (cache->head_dim + 2) * int64_t(sizeof(float))),
             "uc_block8_attn: workspace too small");
  p.list = blocks;
  q.scale = sm_scale * kLog2e;
  float *part = static_cast<float *>(workspace), *stat = part + rows * cache->head_dim;
  const int64_t units = cache->sequences * cache->heads_kv * p.runs * p.groups;
  const uint32_t workgroups = static_cast<uint32_t>(p.workgroups > 0 ? p.workgroups : units * p.splits);
  int rc;
  if (p.rows == kTileRows) {
    rc = launch_tiles(cache, c, q, p, static_cast<uint16_t *>(out), lse, part, stat, as_stream(stream));
  } else {
    rc = UC_B8_DISPATCH(cache, cache->head_dim, [&] {
      launch_rows<D, CODE>(p.rows, workgroups, as_stream(stream), c, q, p, static_cast<uint16_t *>(out), lse, part, stat);
      return check_launch("uc_block8_attn");
    });
  }
  if (rc != UC_OK || (p.splits == 1 && p.workgroups == 0)) return rc;
  const int64_t q_rows = cache->sequences * cache->heads_kv * p.runs * p.run * q.group;
  // parts of a row, if all sequences were of the expected length
  const bool few = (p.workgroups > 0 ? ceil_div(p.workgroups, units) : p.splits) <= 8;
  auto join = [&](auto d_tag) {
    constexpr int D = decltype(d_tag)::value;
    if (few) {
      hipLaunchKernelGGL((join_few_kernel<D>), dim3(static_cast<uint32_t>(ceil_div(q_rows, 16))), dim3(256), 0,
                         as_stream(stream), c, q, p, q_rows, static_cast<uint16_t *>(out), lse, part, stat);
    } else {
      hipLaunchKernelGGL((join_many_kernel<D>), dim3(static_cast<uint32_t>(q_rows)), dim3(256), 0, as_stream(stream), c,
                         q, p, static_cast<uint16_t *>(out), lse, part, stat);
    }
    return check_launch("uc_block8_attn (join)");
  };
  return cache->head_dim == 128 ? join(std::integral_constant<int, 128>()) : join(std::integral_constant<int, 64>());
}
