// Attention over the paged 16-bit cache, by split keys.
//
// Mathematics, per row r and key t, in base 2:
//   x = (q_r . k_t) sm_scale log2(e), P = 2^(x - m), O = sum P v, l = sum P, out = O / l, lse = ln2 (m + log2 l)
// m is a running reference of the row, 2^6 below its largest weight when it was last raised; it is raised
// when a weight passes 2^14, so that most tiles leave O alone, and fp16 weights keep their bits
// down to 2^-24.  Sums, m and O are fp32.  A weight goes into the matrix products as two 16-bit numbers,
// its rounding and what that leaves, so that the products lose 2^-16 of it and not 2^-8 (fp16: 2^-22 and not 2^-11): the
// cores have the time beside the loads.
//
// Layout: S^T = K Q^T on 16x16x32 MFMAs.  Row r of key tile a is key 8 (r / 4) + 4 a + r % 4 of a wave's 32,
// so that a lane's eight logits are eight consecutive keys of one query row: the operand that
// O^T = V^T P^T takes, with no exchange between lanes.  Its other operand, eight keys of one channel, comes from
// rows of the page as they are: a lane loads 16 (D = 64: 8) bytes of each of its eight keys, and one
// byte permutation per pair of keys and channel turns them round.  Fragment n then holds
// channels D/16 r + n, and a lane ends with consecutive channels of its query row.
//
// Bound by HBM: each row is read once, straight into registers, a wave's next 32 keys (16 KB at 128
// channels) on their way while it computes on the present ones.  Of 8 sequences of 32k tokens (28/4 heads, 537 MB) both
// launches take 98.6 us (5.4 TB/s; a large copy 5.0), of 64 ragged ones up to 8k in pages of 16 194 (5.5).
// Small calls are two launches: 2k tokens 6.0 + 4.5 us, 16 x 5 tokens (40 rows) 16.3 + 4.7.  What they wait for
// first are the lengths, then the table, then the rows; queries ride along.
#include "uc_paged_attn.h"

#include <type_traits>

namespace uc {
namespace pg {
namespace {

// Rows of one tile as they come from memory.
template <int D>
struct Raw {
  u4 k[2][D / 32];
  uint32_t v[8][D / 32];
};

template <int D>
struct Lane {
  const uint16_t *key, *value;  // of the head in page 0, at the lane's offset in a half tile
};

template <int D>
__device__ __forceinline__ void load_keys(Raw<D> &raw, const Lane<D> &l, int64_t a, int64_t b) {
  const int64_t at = (threadIdx.x & 8) ? b : a;
  const uint16_t *p = l.key + (at < 0 ? 0 : at);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int k = 0; k < D / 32; ++k) raw.k[t][k] = *reinterpret_cast<const u4 *>(p + t * 4 * D + k * 32);
  }
}

template <int D>
__device__ __forceinline__ void load_values(Raw<D> &raw, const Lane<D> &l, int64_t a, int64_t b) {
  const int64_t at = (threadIdx.x & 32) ? b : a;
  const uint16_t *p = l.value + (at < 0 ? 0 : at);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (D == 128) {
      const u4 v = *reinterpret_cast<const u4 *>(p + j * D);
#pragma unroll
      for (int i = 0; i < 4; ++i) raw.v[j][i] = v[i];
    } else {
      const u2 v = *reinterpret_cast<const u2 *>(p + j * D);
#pragma unroll
      for (int i = 0; i < 2; ++i) raw.v[j][i] = v[i];
    }
  }
}

// Fragment n of the values: channel n of each lane's, its eight keys.
template <int D, int DT>
__device__ __forceinline__ typename Half<DT>::V8 value_fragment(const Raw<D> &raw, int n) {
  uint32_t w[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    w[t] = n % 2 ? halves_of<true>(raw.v[2 * t][n / 2], raw.v[2 * t + 1][n / 2])
                 : halves_of<false>(raw.v[2 * t][n / 2], raw.v[2 * t + 1][n / 2]);
  }
  return __builtin_bit_cast(typename Half<DT>::V8, u4{w[0], w[1], w[2], w[3]});
}

// State of 16 query rows in one wave: the lane's row is lane % 16, its channels of o[n][i] are
// D/4 (lane / 16) + D/16 i + n.
template <int D>
struct Acc {
  f4 o[D / 16];
  float m, l;  // reference; the lane's part of the sum
};

template <int D, int DT, bool MASK>
__device__ __forceinline__ void softmax_step(Acc<D> &acc, f4 (&s)[2], float factor, int32_t seen, bool again,
                                             typename Half<DT>::V8 &high, typename Half<DT>::V8 &low) {
  typedef typename Half<DT>::T T;
  float top = mf::kNegInf;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (MASK) s[j / 4][j % 4] = j >= seen ? mf::kNegInf : s[j / 4][j % 4];  // (its weight is 0 then)
    top = fmaxf(top, s[j / 4][j % 4]);
  }
  top = mf::max_over_slices(top * factor);
  if (__any(top - acc.m > kRaise)) {
    // (of the rows that ask for it: no row's last bits hang on what only another one sees)
    const float m = top - acc.m > kRaise ? top - kHead : acc.m;
    const float alpha = acc.m == mf::kNegInf ? 0.0f : mf::fast_exp2(acc.m - m);
    acc.m = m;
    acc.l *= alpha;
#pragma unroll
    for (int n = 0; n < D / 16; ++n) acc.o[n] *= alpha;
  }
  float m = acc.m == mf::kNegInf ? 0.0f : acc.m;
  if (MASK && __builtin_expect(again, false)) round_far(s, factor, m);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = __builtin_fmaf(s[j / 4][j % 4], factor, -m);
    const float e = mf::fast_exp2(x);
    acc.l += e;
    high[j] = static_cast<T>(e);
    low[j] = static_cast<T>(e - static_cast<float>(high[j]));
  }
}

// LDS of the waves' join; and of more than 16 rows the query fragments, which need not fit the registers.
template <int D, int DT, int NR>
struct Joined {
  static constexpr bool kHeld = NR * D >= 192;
  float o[4][16][D + 4];  // (a wave's part holds a tile's values, 8 D / 32 dwords a lane)
  float m[4][16], l[4][16];
  uint32_t bad;  // whether a second pass is asked for
  typename Half<DT>::V8 frag[kHeld ? NR * D / 32 : 1][64];
};

// Steps begin .. end - 1 of the rows w, by a whole workgroup.  slot >= 0: the part goes there; else it
// is all there is, and the rows are finished.  Returns whether values that are not finite went into sums, or a reference lies far off:
// then once more with `search`.
template <int D, int DT, int NR>
__device__ __forceinline__ bool piece(const Cache &c, const Query &q, const Rows &w, int32_t begin, int32_t end, int32_t slot,
                                      bool search, Joined<D, DT, NR> &joined, uint16_t *out, float *lse, float *part,
                                      float *stat) {
  typedef Half<DT> H;
  typedef typename H::V8 V8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15,
            quad = lane >> 4;
  Pages pages(c, w.s);
  Lane<D> l;
  const int64_t head = int64_t(w.h << c.shift) * D;
  l.key = c.key + head + (8 * ((col >> 2) & 1) + (col & 3)) * D + quad * 8;
  l.value = c.value + head + 8 * (quad & 1) * D + col * (D / 16);

  V8 frag[NR][D / 32];
  int32_t row_end[NR];
  Acc<D> acc[NR];
  Infinite infinite[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int32_t r = w.r0 + 16 * n + col;
    const bool there = r < w.rows;
    // (rows past the last are the first's again, and nobody's)
    const int32_t at = there ? r : w.r0, token = token_of(q, at);
    row_end[n] = there ? visible(q, w.length, w.count, token) : 0;
    const uint16_t *p = q.p + w.s * q.ss + token * q.st + (w.h * q.group + at - token * q.group) * q.sh + quad * 8;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) frag[n][k] = *reinterpret_cast<const V8 *>(p + k * 32);
    acc[n].m = mf::kNegInf;
    acc[n].l = 0.0f;
    infinite[n] = Infinite{0, 0};
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[n].o[d] = f4{0, 0, 0, 0};
  }
  const int32_t stop = end * kStep < w.end_last ? end * kStep : w.end_last;
  int32_t t = begin * kStep + wave * kTile;
  Raw<D> raw;
  // where a tile's halves begin (16 keys lie in one page), and the entries of the next one
  int64_t first_a = -1, first_b = -1;
  int32_t entry_a = 0, entry_b = 0;
  if (t < stop) {
    entry_a = pages.of(t);
    entry_b = pages.of(t + 16);
    first_a = place_of(c, entry_a, t, D);
    first_b = place_of(c, entry_b, t + 16, D);
    load_keys(raw, l, first_a, first_b);
    load_values(raw, l, first_a, first_b);
    entry_a = pages.of(t + kStep);
    entry_b = pages.of(t + kStep + 16);
  }
  typedef Joined<D, DT, NR> J;
  if constexpr (J::kHeld) {
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
    if constexpr (J::kHeld) asm volatile("" : "+v"(at));
    auto query = [&](int n, int k) { return J::kHeld ? joined.frag[n * (D / 32) + k][at] : frag[n][k]; };
    const bool more = t + kStep < stop;
    const int64_t next_a = place_of(c, entry_a, t + kStep, D), next_b = place_of(c, entry_b, t + kStep + 16, D);
    f4 s[NR][2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][a] = f4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const V8 rows = __builtin_bit_cast(V8, raw.k[a][k]);
#pragma unroll
        for (int n = 0; n < NR; ++n) s[n][a] = H::mfma(rows, query(n, k), s[n][a]);
      }
    }
    if (more) load_keys(raw, l, next_a, next_b);
    // (asked for here: LDS reads and scalar loads are waited for together, and none of the former follows for a while)
    __builtin_amdgcn_sched_barrier(0);
    entry_a = pages.of(t + 2 * kStep);
    entry_b = pages.of(t + 2 * kStep + 16);
    __builtin_amdgcn_sched_barrier(0);
    const int32_t mine = t + 8 * quad;                              // the lane's first key
    const bool there = ((quad & 2) ? first_b : first_a) >= 0;              // and its page
    V8 high[NR], low[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      softmax_step<D, DT, MASK>(acc[n], s[n], q.scale, there ? row_end[n] - mine : 0, search, high[n], low[n]);
    }
    if constexpr (MASK) {
      // what no row sees is no value
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool held = there && mine + j < w.end_last;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) raw.v[j][i] = held ? raw.v[j][i] : 0u;
      }
      if (search || w.end_first != w.end_last) {  // some rows see more than others
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) bad |= infinite_bits<DT>(raw.v[j][i]);
        }
        if (__builtin_expect(__any(bad != 0), false)) {
// (a loop over the fragments, through the wave's part of the LDS that the join takes: it is rare, and written
          // out it takes the registers that the other tiles need)
          uint32_t *held = reinterpret_cast<uint32_t *>(joined.o[wave]) + lane;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) held[(j * (D / 32) + i) * 64] = raw.v[j][i];
          }
#pragma unroll 1
          for (int d = 0; d < D / 16; ++d) {
            u4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t a = held[(2 * j * (D / 32) + d / 2) * 64], b = held[((2 * j + 1) * (D / 32) + d / 2) * 64];
              v[j] = d % 2 ? halves_of<true>(a, b) : halves_of<false>(a, b);
            }
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              note_infinite<DT>(__builtin_bit_cast(V8, v), there ? row_end[n] - mine : 0, d, infinite[n]);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) raw.v[j][i] = finite_half<DT>(raw.v[j][i]);
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const V8 v = value_fragment<D, DT>(raw, d);
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        acc[n].o[d] = H::mfma(v, high[n], acc[n].o[d]);
        acc[n].o[d] = H::mfma(v, low[n], acc[n].o[d]);
      }
    }
    if (more) load_values(raw, l, next_a, next_b);
    first_a = next_a;
    first_b = next_b;
    t += kStep;
  };
  // tiles that every row sees come first; from the first other one on, every tile is masked
  while (!search && t < stop && t + kTile <= w.end_first && first_a >= 0 && first_b >= 0) step(std::false_type());
  while (t < stop) step(std::true_type());

  // join the waves: 16 threads a row, D / 16 channels each
  constexpr int kC = D / 16;
  const int row = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * kC;
  const float least = search ? 0x1p-149f : 0.0f;  // (infinities stay, however small the factor)
  bool bad = false;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const float l_row = mf::sum_over_slices(acc[n].l);
    bad |= is_far(acc[n].m);
    add_infinite(acc[n].o, infinite[n]);
    __syncthreads();  // what was joined before, and its flag, have been read
    if (n == 0 && threadIdx.x == 0) joined.bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int d = 0; d < kC; d += 4) {
        *reinterpret_cast<f4 *>(&joined.o[wave][col][(D / 4) * quad + kC * i + d]) =
            f4{acc[n].o[d][i], acc[n].o[d + 1][i], acc[n].o[d + 2][i], acc[n].o[d + 3][i]};
      }
    }
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
      // a wave without keys of this row has nothing to add, unless what it has is not a number
      if (joined.m[v][row] == mf::kNegInf && joined.l[v][row] == 0.0f) continue;
      const float f = fmaxf(mf::fast_exp2(joined.m[v][row] - m), least);
      total += f * joined.l[v][row];
#pragma unroll
      for (int j = 0; j < kC; ++j) o[j] += f * joined.o[v][row][c0 + j];
    }
    const int32_t r = w.r0 + 16 * n + row;
    if (r >= w.rows) continue;
    if (total == 0.0f && m == mf::kNegInf) {
      const int32_t mine = visible(q, w.length, w.count, token_of(q, r));
      m = no_reference(c, w.s, begin * kStep, mine < stop ? mine : stop);
    }
    bad |= spoiled<kC>([&](int j) { return o[j]; }, total);
    if (slot >= 0) {
      const int64_t at = int64_t(slot) * (16 * NR) + 16 * n + row;
#pragma unroll
      for (int j = 0; j < kC; j += 4) {
        *reinterpret_cast<f4 *>(part + at * D + c0 + j) = f4{o[j], o[j + 1], o[j + 2], o[j + 3]};
      }
      if (c0 == 0) {
        stat[2 * at] = m;
        stat[2 * at + 1] = total;
      }
    } else {
      store_row<D, DT>(q, w, r, c0, o, m, total, out, lse);
    }
  }
  if (__any(bad)) joined.bad = 1;  // (barriers lie between this, the first write and the read)
  __syncthreads();  // the next piece may write what has been read here
  return __builtin_expect(__builtin_amdgcn_readfirstlane(joined.bad) != 0, false);
}

// The steps of all units ((sequence, head) in order) are cut into runs of equal length for the
// workgroups, so that sequences of any lengths load them alike.  A unit's part in workgroup g is in slot
// g + unit: of two parts in order one of the two is larger.
__device__ __forceinline__ int32_t steps_of(int32_t length, int32_t count) {
  return count > 0 ? (length + kStep - 1) / kStep : 0;
}

__device__ __forceinline__ int32_t per_of(const Plan &p, int32_t total) { return (total + p.workgroups - 1) / p.workgroups; }

template <int D, int DT, int NR>
__global__ __launch_bounds__(256, D == 128 && NR > 2 ? 1 : 2) void rows_kernel(Cache c, Query q, Plan p, uint16_t *out,
                                                                             float *lse, float *part, float *stat) {
  __shared__ Joined<D, DT, NR> joined;
  const int lane = threadIdx.x & 63;
  const int32_t g = blockIdx.x, each = c.heads;  // (a unit holds all rows of a head)
  int32_t s0 = 0, first = 0;  // sequences s0 .. s0 + 63 are in the lanes, `first` of them is the present one
  int32_t length = 0, count = 0, steps = 0, sum = 0, total = 0;
  auto fill = [&] {
    const int32_t i = s0 + lane;
    length = count = 0;
    if (i < c.sequences) sizes_of(c, q, i, length, count);
    steps = steps_of(length, count);
    sum = wave_prefix(steps);
  };
  for (s0 = 0; s0 < c.sequences; s0 += 64) {
    fill();
    total += __builtin_amdgcn_readlane(sum, 63);
  }
  if (c.sequences > 64) {
    s0 = 0;
    fill();
  }
  s0 = 0;
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
  bool search = false;
  while (at < stop) {
    const int32_t end = now - t < stop - at ? now : t + (stop - at), s = s0 + first;
    // Where registers are short the row's number is opaque, so that what it gives is worked out for each piece: held across
    // pieces the tiles spill for it (8 x 4 tokens of 16k at 128 channels 52.6 us, 51.2 so; at 64, 16 x 8 of 4k 28.7 and 26.7,
    // 16 x 5 21.9 and 21.7).
    int32_t only = 0;
    if constexpr (Joined<D, DT, NR>::kHeld) asm volatile("" : "+s"(only));
    const Rows w = rows_at(q, s, n, only, 16 * NR, __builtin_amdgcn_readlane(length, first),
                           __builtin_amdgcn_readlane(count, first));
    const int32_t slot = end - t == now ? -1 : g + s * each + n;
    search = piece<D, DT, NR>(c, q, w, t, end, slot, search, joined, out, lse, part, stat) && !search;
    if (search) continue;
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

__device__ __forceinline__ Parts parts_of(const Cache &c, const Query &q, const Plan &p, int32_t index) {
  Parts x;
  const int32_t full = q.len * q.group, sh = index / full, s = sh / c.heads;
  x.r = index - sh * full;
  const int32_t each = c.heads;
  int32_t total = 0, before = 0, mine = 0, my_length = 0, my_count = 0;
  for (int32_t s0 = 0; s0 < c.sequences; s0 += 64) {
    const int32_t i = s0 + (threadIdx.x & 63);
    int32_t length = 0, count = 0;
    if (i < c.sequences) sizes_of(c, q, i, length, count);
    const int32_t n = steps_of(length, count);
    const int32_t sum = wave_prefix(n);
    const int32_t m = __shfl(n, s - s0, kWave), b = __shfl(sum, s - s0, kWave);
    const int32_t ml = __shfl(length, s - s0, kWave), mc = __shfl(count, s - s0, kWave);
    if (s >= s0 && s < s0 + 64) {
      mine = m;
      before = total + b - m;
      my_length = ml;
      my_count = mc;
    }
    total += __builtin_amdgcn_readlane(sum, 63);
  }
  x.w = rows_at(q, s, sh - s * c.heads, 0, p.rows, my_length, my_count);
  const int32_t per = per_of(p, total * each);
  const int32_t start = before * each + (sh - s * each) * mine;
  x.first = mine == 0 ? 0 : start / per + sh;
  x.count = mine == 0 ? 0 : (start + mine - 1) / per + sh - x.first + 1;
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
      if (i0 + u * STRIDE >= x.count || (mi[u] == mf::kNegInf && li[u] == 0.0f)) continue;
      const float f = mf::fast_exp2(mi[u] - t.m);
      t.l += f * li[u];
#pragma unroll
      for (int j = 0; j < kC; ++j) t.o[j] += joining(f, oi[u][j / 4][j % 4]);
    }
    i0 += 2 * STRIDE;
    if (i0 < x.count) load(i0);
  }
  return t;
}

// Few parts a row: a wave joins four rows.  (Rows of one part are finished already.)
template <int D, int DT>
__global__ __launch_bounds__(256) void join_few_kernel(Cache c, Query q, Plan p, int32_t rows, uint16_t *out, float *lse,
                                                       const float *part, const float *stat) {
  const int32_t index = blockIdx.x * 16 + (threadIdx.x >> 4), last = rows - 1;
  const Parts x = parts_of(c, q, p, index < rows ? index : last);  // (whole waves: they sum up the lengths)
  if (index >= rows || x.count == 1) return;
  const Sum<D> t = sum_parts<D, 1>(p, x, 0, part, stat);
  store_row<D, DT>(q, x.w, x.r, (threadIdx.x & 15) * (D / 16), t.o, t.m, t.l, out, lse);
}

// Many: a workgroup joins one row, its 16-lane groups every 16th part.
template <int D, int DT>
__global__ __launch_bounds__(256) void join_many_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse,
                                                        const float *part, const float *stat) {
  constexpr int kC = D / 16;
  __shared__ float sh_o[16][D], sh_l[16];
  const Parts x = parts_of(c, q, p, blockIdx.x);
  if (x.count == 1) return;
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
  store_row<D, DT>(q, x.w, x.r, lane * kC, t.o, t.m, t.l, out, lse);
}

constexpr int64_t kShare = 512;  // workgroups that share the steps: two a CU

int make_plan(const uc_paged_cache *cache, const Cache &c, const uc_block8_query *query, const char *what, Query &q, Plan &p) {
  UC_REQUIRE(query != nullptr, "%s: query is NULL", what);
  UC_REQUIRE(query->dtype == cache->dtype, "%s: queries must have the cache's dtype", what);
  UC_REQUIRE(query->heads_q > 0 && query->heads_q < (1 << 24) && query->heads_q % cache->heads_kv == 0,
             "%s: query heads must be a multiple of KV heads", what);
  UC_REQUIRE(query->query_len >= 0 && query->query_len < (1 << 24), "%s: bad query_len", what);
  UC_REQUIRE(query->max_tokens >= 0, "%s: negative max_tokens", what);
  const int64_t group = query->heads_q / cache->heads_kv, rows = group * query->query_len;
  q = Query{static_cast<const uint16_t *>(query->query), query->q_ss, query->q_st, query->q_sh, query->query_lengths,
            static_cast<int32_t>(query->query_len), static_cast<int32_t>(query->heads_q), static_cast<int32_t>(group),
            query->causal != 0, 0.0f, 0.0f, make_fastdiv(static_cast<uint32_t>(group))};
  p.rows = rows <= 64 ? static_cast<int32_t>(ceil_div(rows, int64_t(16))) * 16 : kTileRows;
  if (p.rows == 0) p.rows = 16;
  p.groups = static_cast<int32_t>(ceil_div(rows, int64_t(p.rows)));
  const int64_t capacity = c.capacity(), keys = query->max_tokens < capacity ? query->max_tokens : capacity;
  // a launch has less than 2^32 threads, and 32-bit counts of rows and steps (few rows are joined by up to a workgroup each)
  UC_REQUIRE(cache->sequences * cache->heads_kv < (1 << 28) && rows < (1 << 28) &&
                 cache->sequences * cache->heads_kv * rows < (p.rows >= kTileRows ? 1 << 27 : 1 << 24),
             "%s: too many query rows", what);
  const int64_t units = cache->sequences * cache->heads_kv * p.groups;
  UC_REQUIRE(units * ceil_div(capacity, int64_t(kStep)) < (1 << 30), "%s: too many keys in all", what);
  if (p.rows == kTileRows) {
    // Two workgroups a CU at most, as many on each XCD, of four tiles at least; two where that leaves a unit in 16 parts at
    // most (50 queries of 500 tokens 20.5 -> 16.4 us; 20 of 10,000 33 with four, 39 with two).
    const int64_t each = keys > 0 ? ceil_div(keys, int64_t(kKeys)) : 1, least = each <= 32 ? 2 : 4, tiles = units * each;
    p.workgroups = 0;
    if (cache->sequences * p.groups <= kMostShared && units * ceil_div(capacity, int64_t(kKeys)) < (1 << 30)) {
      p.workgroups = static_cast<int32_t>(tiles < least * kShare ? ceil_div(tiles, 8 * least) * 8 : kShare);
    }
    UC_REQUIRE(units < (1 << 21), "%s: too many query rows", what);
    return UC_OK;
  }
  const int64_t steps = units * ceil_div(keys, int64_t(kStep));
  p.workgroups = static_cast<int32_t>(steps < kShare ? (steps > 0 ? steps : 1) : kShare);
  return UC_OK;
}

int64_t part_rows(const uc_paged_cache *cache, const Plan &p) {
  // (of many rows, a workgroup's first and last unit may be parts)
  if (p.rows == kTileRows) return int64_t(2) * p.workgroups * p.rows;
  return (cache->sequences * cache->heads_kv * p.groups + p.workgroups) * p.rows;
}

}  // namespace
}  // namespace pg
}  // namespace uc

extern "C" int64_t uc_paged_attn_workspace_bytes(const uc_paged_cache *cache, const uc_block8_query *query) {
  using namespace uc::pg;
  Cache c;
  Query q;
  Plan p;
  if (check_cache(cache, 0, "uc_paged_attn", c) || make_plan(cache, c, query, "uc_paged_attn", q, p)) return -1;
  return q.len == 0 ? 0 : part_rows(cache, p) * (cache->head_dim + 2) * int64_t(sizeof(float));
}

extern "C" int uc_paged_attn(const uc_paged_cache *cache, int64_t layer, const uc_block8_query *query, float sm_scale,
                             void *out, float *lse, void *workspace, int64_t workspace_bytes, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::pg;
  const char *what = "uc_paged_attn";
  Cache c;
  Query q;
  Plan p;
  if (int rc = check_cache(cache, layer, what, c)) return rc;
  if (int rc = make_plan(cache, c, query, what, q, p)) return rc;
  // (times log2(e) it stays in fp32's range, and a normal number: the kernels flush others to 0)
  UC_REQUIRE(sm_scale >= 0x1p-126f && sm_scale <= 0x1p127f, "%s: sm_scale must be 2^-126 at least, and 2^127 at most", what);
  if (q.len == 0) return UC_OK;
  UC_REQUIRE(q.p != nullptr && (reinterpret_cast<uintptr_t>(q.p) & 15) == 0 && ((q.ss | q.st | q.sh) & 7) == 0,
             "%s: query must be 16-byte aligned with strides that are multiples of 8", what);
  UC_REQUIRE(out != nullptr && (reinterpret_cast<uintptr_t>(out) & 15) == 0, "%s: out must be 16-byte aligned", what);
  const int64_t rows = part_rows(cache, p);
  UC_REQUIRE(rows == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                           workspace_bytes >= rows * (cache->head_dim + 2) * int64_t(sizeof(float))),
             "%s: workspace too small", what);
  q.scale = sm_scale * kLog2e;
  q.unit = static_cast<float>(static_cast<double>(sm_scale) / static_cast<double>(q.scale) - static_cast<double>(kLn2));
  float *part = static_cast<float *>(workspace), *stat = part + rows * cache->head_dim;
  const int64_t units = cache->sequences * cache->heads_kv * p.groups;
  const int32_t q_rows = static_cast<int32_t>(cache->sequences * cache->heads_kv * q.len * q.group);
  // parts of a row, if all sequences were of the expected length
  const bool few = ceil_div(p.workgroups, units) <= 8;
  auto run = [&](auto d_tag, auto dt_tag) {
    constexpr int D = decltype(d_tag)::value, DT = decltype(dt_tag)::value;
    auto rows_launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(p.workgroups)), dim3(256), 0, as_stream(stream), c, q, p,
                         static_cast<uint16_t *>(out), lse, part, stat);
    };
    if (p.rows == kTileRows) {
      return launch_tiles(what, DT, D, c, q, p, static_cast<uint16_t *>(out), lse, part, stat, as_stream(stream));
    } else if (p.rows == 16) {
      rows_launch(rows_kernel<D, DT, 1>);
    } else if (p.rows == 32) {
      rows_launch(rows_kernel<D, DT, 2>);
    } else if (p.rows == 48) {
      rows_launch(rows_kernel<D, DT, 3>);
    } else {
      rows_launch(rows_kernel<D, DT, 4>);
    }
    if (int rc = check_launch(what)) return rc;
    if (few) {
      hipLaunchKernelGGL((join_few_kernel<D, DT>), dim3(static_cast<uint32_t>(ceil_div(q_rows, 16))), dim3(256), 0,
                         as_stream(stream), c, q, p, q_rows, static_cast<uint16_t *>(out), lse, part, stat);
    } else {
      hipLaunchKernelGGL((join_many_kernel<D, DT>), dim3(static_cast<uint32_t>(q_rows)), dim3(256), 0, as_stream(stream), c,
                         q, p, static_cast<uint16_t *>(out), lse, part, stat);
    }
    return check_launch(what);
  };
  auto by_type = [&](auto d_tag) {
    return cache->dtype == UC_FP16 ? run(d_tag, std::integral_constant<int, UC_FP16>())
                                   : run(d_tag, std::integral_constant<int, UC_BF16>());
  };
  return cache->head_dim == 128 ? by_type(std::integral_constant<int, 128>()) : by_type(std::integral_constant<int, 64>());
}
