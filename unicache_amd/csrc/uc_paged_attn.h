// What the attention kernels of the paged cache share: queries, rows, pages and the 16-bit operands.
#pragma once
#include "uc_mfma.h"
#include "uc_paged.h"

namespace uc {
namespace pg {

using mf::f4;

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;                 // keys of a wave's tile
constexpr int kStep = 4 * kTile;          // keys of a workgroup's step
constexpr float kHead = 6.0f;             // a raised reference lies 2^6 below the largest weight
constexpr float kRaise = 14.0f;           // and is raised where a weight passes 2^14: fp16 holds 2^-24 .. 2^15

struct Query {
  const uint16_t *p;
  int64_t ss, st, sh;
  const int32_t *lens;
  int32_t len, heads, group;
  int32_t causal;
  float scale;  // sm_scale * log2(e)
  float unit;   // sm_scale / scale - ln2: what rounding made of a unit of the scaled products in natural logarithms
  FastDiv by_group;

  __device__ __forceinline__ int32_t count(int32_t s) const { return lens == nullptr ? len : clamped(lens[s]); }
  __device__ __forceinline__ int32_t clamped(int32_t n) const { return n < 0 ? 0 : n > len ? len : n; }
};

// A sequence's length and number of queries, both on their way at once.
__device__ __forceinline__ void sizes_of(const Cache &c, const Query &q, int32_t s, int32_t &length, int32_t &count) {
  const int32_t n = c.lengths[s], m = (q.lens != nullptr ? q.lens : c.lengths)[s];
  length = c.clamped(n);
  count = q.lens != nullptr ? q.clamped(m) : q.len;
}

constexpr int kTileRows = 128;            // rows of a unit of many (uc_paged_tiles.hip)

struct Plan {
  int32_t rows, groups;  // rows of a unit, and units of a (sequence, KV head): one, of all its rows, up to 64
  int32_t workgroups;    // that share all steps; 0 (many rows): one a unit
};

// The rows of a unit: row r is query token r / group of head h * group + r % group.
struct Rows {
  int32_t s, h, length, count;
  int32_t rows, r0;            // of the (sequence, head); first row of the unit
  int32_t end_first, end_last; // keys that the first and the last row that counts see
};

__device__ __forceinline__ int32_t token_of(const Query &q, int32_t r) { return static_cast<int32_t>(fast_div(r, q.by_group)); }

__device__ __forceinline__ int32_t visible(const Query &q, int32_t length, int32_t count, int32_t token) {
  if (token >= count) return 0;
  if (!q.causal) return length;
  const int32_t e = length - count + token + 1;
  return e < 0 ? 0 : e;
}

__device__ __forceinline__ Rows rows_at(const Query &q, int32_t s, int32_t h, int32_t group, int32_t rows, int32_t length,
                                        int32_t count) {
  Rows w;
  w.s = s;
  w.h = h;
  w.length = length;
  w.count = count;
  w.rows = q.len * q.group;
  w.r0 = group * rows;
  const int32_t t0 = token_of(q, w.r0);
  int32_t t1 = token_of(q, (w.r0 + rows < w.rows ? w.r0 + rows : w.rows) - 1);
  t1 = t1 < count ? t1 : count - 1;
  const bool none = w.r0 >= w.rows || t0 >= count;
  w.end_first = none ? 0 : visible(q, length, count, t0);
  w.end_last = none ? 0 : visible(q, length, count, t1);
  return w;
}

// A sequence's row of the table, read by scalar loads: an entry that is asked for a tile ahead of its use
// costs no wave a wait, and what follows from it stays in scalar registers.
struct Pages {
  typedef const __attribute__((address_space(4))) int32_t *Scalars;
  Scalars row;
  int32_t last, shift;

  __device__ __forceinline__ Pages(const Cache &c, int32_t s)
      : row((Scalars)(c.table + int64_t(s) * c.width)), last(c.width - 1), shift(c.shift) {}

  // The entry of token t, which is the same in the whole wave; past the table the last one (no row sees such tokens).
  __device__ __forceinline__ int32_t of(int32_t t) const {
    const int32_t e = __builtin_amdgcn_readfirstlane(t >> shift);
    return row[e < last ? e : last];
  }
};

// The first row of a head's tokens t .. in their page, in elements from its first in page 0; -1 where there is no page.
__device__ __forceinline__ int64_t place_of(const Cache &c, int32_t entry, int32_t t, int32_t d) {
  const bool is = c.is_page(entry);
  const int64_t at = int64_t(is ? entry : 0) * c.page_elems + (t & (c.page - 1)) * d;
  return is ? at : -1;
}

// 16-bit operands.
template <int DT>
struct Half;
template <>
struct Half<UC_FP16> {
  typedef _Float16 T;
  typedef T V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f4 mfma(V8 a, V8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Half<UC_BF16> {
  typedef __bf16 T;
  typedef T V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f4 mfma(V8 a, V8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef typename Half<DT>::T T;
  typedef T V2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, V2{static_cast<T>(a), static_cast<T>(b)});
}

// Values that are not finite.  In tiles that not every row sees whole a hidden key's weight is 0, and 0 times them is NaN; where a
// row sees them its weight may have been rounded to 0, or be two numbers of which one is 0 or negative.  So where there are
// any the products take 0 in their place, and others count, for each row, the keys that it does see of each kind; one is
// enough to make the sum what it is.  Tiles that some rows see in part are searched for them; the others only when a sum is no number
// at the end, in a second pass over all tiles, each searched.
template <int DT>
constexpr uint32_t kInfinity = DT == UC_FP16 ? 0x7c00u : 0x7f80u;

// Not 0 where a half of w is not finite: its exponent and 1 overflow into the sign.
template <int DT>
__device__ __forceinline__ uint32_t infinite_bits(uint32_t w) {
  constexpr uint32_t e = kInfinity<DT>, one = DT == UC_FP16 ? 0x0400u : 0x0080u;
  return ((w & (e | e << 16)) + (one | one << 16)) & 0x80008000u;
}

// w with zeros in the place of halves that are not finite.
template <int DT>
__device__ __forceinline__ uint32_t finite_half(uint32_t w) {
  const uint32_t b = infinite_bits<DT>(w);
  return w & ~((b >> 15) * 0xffffu);
}

// A bit for each of a lane's outputs, 4 d + i: the row sees an infinity (or a negative one) there; both for NaN.
struct Infinite {
  uint32_t up, down;
};

// What fragment v, of the outputs' fragment d, holds of them for rows that see the first `seen` of a lane's eight keys.
template <int DT>
__device__ __forceinline__ void note_infinite(typename Half<DT>::V8 v, int32_t seen, int d, Infinite &x) {
  typedef typename Half<DT>::T T;
  typedef typename Half<DT>::V8 V8;
  constexpr uint32_t e = kInfinity<DT>;
  const u4 u = __builtin_bit_cast(u4, v);
  V8 sees, up, down;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t h = j % 2 ? u[j / 2] >> 16 : u[j / 2] & 0xffffu, size = h & 0x7fffu;
    sees[j] = static_cast<T>(j < seen ? 1.0f : 0.0f);
    up[j] = static_cast<T>(size > e || h == e ? 1.0f : 0.0f);
    down[j] = static_cast<T>(size > e || h == (e | 0x8000u) ? 1.0f : 0.0f);
  }
  const f4 a = Half<DT>::mfma(up, sees, f4{0, 0, 0, 0}), b = Half<DT>::mfma(down, sees, f4{0, 0, 0, 0});
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.up |= (a[i] > 0.0f ? 1u : 0u) << (4 * d + i);
    x.down |= (b[i] > 0.0f ? 1u : 0u) << (4 * d + i);
  }
}

// And to the sums of finite values.
template <int N>
__device__ __forceinline__ void add_infinite(f4 (&o)[N], const Infinite &x) {
  if (__builtin_expect(!__any((x.up | x.down) != 0), true)) return;
#pragma unroll
  for (int d = 0; d < N; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bit = 1u << (4 * d + i);
      o[d][i] += (x.up & bit) != 0 ? __builtin_huge_valf() : 0.0f;
      o[d][i] -= (x.down & bit) != 0 ? __builtin_huge_valf() : 0.0f;
    }
  }
}

// Whether a row's N sums, beside that of its weights, show that such values went into them.
template <int N, class At>
__device__ __forceinline__ bool spoiled(At at, float l) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = __builtin_elementwise_maximum(top, __builtin_fabsf(at(j)));  // (passes NaN on)
  return !(top < __builtin_huge_valf()) && l < __builtin_huge_valf();
}

// Logits in base 2 are products s factor, fused with the reference m taken off: s factor is not rounded, while m was made of the
// largest one rounded.  So x of the largest is off by half a step of either, one at most up to kFar; beyond, weights
// would leave what 16 bits hold.  Where a reference lies there, all is done in a second pass too, in which
// such rows' products are rounded first: they are replaced by x.
constexpr float kFar = 0x1p24f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > kFar && fabsf(m) < __builtin_huge_valf(); }
template <int N>
__device__ __forceinline__ void round_far(f4 (&s)[N], float &factor, float &m) {
  const bool far = is_far(m);
#pragma unroll
  for (int j = 0; j < N; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float product = s[j][i] * factor;
      s[j][i] = far ? product - m : s[j][i];
    }
  }
  factor = far ? 1.0f : factor;
  m = far ? 0.0f : m;
}

// A part's sum as it joins others: where it is not finite it stays so, however small the factor.
__device__ __forceinline__ float joining(float f, float o) {
  const float x = f * o;
  return x == x ? x : o;  // (a factor that is no number makes the sum of the weights NaN, and so the row)
}

// The lower or the upper halves of two dwords as one.
template <bool UPPER>
__device__ __forceinline__ uint32_t halves_of(uint32_t first, uint32_t second) {
  return __builtin_amdgcn_perm(second, first, UPPER ? 0x07060302u : 0x05040100u);
}

// The reference of a row that has none after tokens first .. end - 1: -inf where there is no key among them, else its logits all lie
// below fp32's range, and with the lowest finite one it ends as 0 / 0 = NaN, unless another part has weights.
__device__ __forceinline__ float no_reference(const Cache &c, int32_t s, int32_t first, int32_t end) {
  for (int32_t t = first; t < end; t = (t | (c.page - 1)) + 1) {
    if (c.is_page(c.table[int64_t(s) * c.width + (t >> c.shift)])) return -0x1.fffffep127f;
  }
  return mf::kNegInf;
}

// The log-sum-exp of a row that sees keys (a sum of 0 is of logits below fp32's range), rounded once: the scale's own rounding and
// that of a sum with m would each be as much again.
__device__ __forceinline__ float lse_of(const Query &q, float m, float l) {
  const float rest = __builtin_fmaf(m, q.unit, kLn2 * __builtin_amdgcn_logf(l));
  return l == 0.0f ? __builtin_nanf("") : __builtin_fmaf(m, kLn2, rest);
}

// D / 16 channels of a finished row.
template <int D, int DT>
__device__ __forceinline__ void store_row(const Query &q, const Rows &w, int32_t r, int32_t c0, const float *o, float m,
                                          float l, uint16_t *out, float *lse) {
  constexpr int kC = D / 16;
  const int32_t t = token_of(q, r), head = w.h * q.group + r - t * q.group;
  const bool none = t >= w.count || (l == 0.0f && m == mf::kNegInf);
  const float f = none ? 0.0f : 1.0f / l;
  uint32_t v[kC / 2];
#pragma unroll
  for (int j = 0; j < kC / 2; ++j) v[j] = none ? 0u : pack2<DT>(o[2 * j] * f, o[2 * j + 1] * f);
  uint16_t *dst = out + ((int64_t(w.s) * q.len + t) * q.heads + head) * D + c0;
  if constexpr (kC == 8) {
    *reinterpret_cast<uint4 *>(dst) = uint4{v[0], v[1], v[2], v[3]};
  } else {
    *reinterpret_cast<uint2 *>(dst) = uint2{v[0], v[1]};
  }
  if (c0 == 0 && lse != nullptr) {
    lse[(int64_t(w.s) * q.heads + head) * q.len + t] = none ? mf::kNegInf : lse_of(q, m, l);
  }
}

// uc_paged_tiles.hip: many query rows.
constexpr int kKeys = 64;                 // keys of a tile
constexpr int64_t kMostShared = 4096;     // row groups of all sequences that a wave adds up
int launch_tiles(const char *what, int dtype, int64_t head_dim, const Cache &c, const Query &q, const Plan &p, uint16_t *out,
                 float *lse, float *part, float *stat, hipStream_t stream);

}  // namespace pg
}  // namespace uc
