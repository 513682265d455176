// What the attention kernels of the paged cache share: queries, rows, pages and the 16-bit operands.
#pragma once
#include "uc_mfma.h"
#include "uc_paged.h"

namespace uc {
namespace pg {

using mf::f4;

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
  FastDiv by_group;

  __device__ __forceinline__ int32_t count(int32_t s) const {
    if (lens == nullptr) return len;
    const int32_t n = lens[s];
    return n < 0 ? 0 : n > len ? len : n;
  }
};

constexpr int kTileRows = 128;            // rows of a unit of many (uc_paged_tiles.hip)

struct Plan {
  int32_t rows, groups;         // rows of a unit, and units of a (sequence, KV head)
  int32_t workgroups;           // few rows: workgroups that share all steps; 0: many rows
  int32_t splits, split_tiles;  // many rows: splits of a unit's keys, and the 64-key tiles of one
};

// Tiles of one split: the host's figure, or more where a sequence is longer than it expected.
__device__ __forceinline__ int32_t split_tiles_of(const Plan &p, int32_t tiles) {
  const int32_t least = (tiles + p.splits - 1) / p.splits;
  return least > p.split_tiles ? least : p.split_tiles;
}

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

// A sequence's pages, 64 entries at a time in a wave's lanes, so that a tile's page is no load that its
// rows' loads would wait for.  What is no page reads as -1.
struct Pages {
  const int32_t *row;
  int32_t width, pages, chunk, held;

  __device__ __forceinline__ Pages(const Cache &c, int32_t s)
      : row(c.table + int64_t(s) * c.width), width(c.width), pages(c.pages), chunk(-1), held(-1) {}

  __device__ __forceinline__ int32_t entry(int32_t e) {
    if (e >= width) return -1;
    if ((e >> 6) != chunk) {
      chunk = e >> 6;
      const int32_t i = chunk * 64 + (threadIdx.x & 63), p = i < width ? row[i] : -1;
      held = static_cast<uint32_t>(p) < static_cast<uint32_t>(pages) ? p : -1;
    }
    return __builtin_amdgcn_readlane(held, e & 63);
  }
};

// Where 32 keys lie: each half's first row, in elements from a head's first in page 0; -1 where there is no page.
struct Place {
  int32_t t;
  int64_t a, b;
};

__device__ __forceinline__ Place place_of(const Cache &c, Pages &pages, int32_t t, int32_t d) {
  Place x;
  x.t = t;
  const int32_t p = pages.entry(t >> c.shift);
  x.a = p < 0 ? -1 : int64_t(p) * c.page_elems + (t & (c.page - 1)) * d;
  if (c.shift >= 5) {
    x.b = p < 0 ? -1 : x.a + 16 * d;
  } else {
    const int32_t n = pages.entry((t >> c.shift) + 1);
    x.b = n < 0 ? -1 : int64_t(n) * c.page_elems;
  }
  return x;
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

// Bits of the halves of w that are no finite numbers.
template <int DT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t e = DT == UC_FP16 ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0xffffu : 0u) | ((w & (e << 16)) == e << 16 ? 0xffff0000u : 0u);
}

// The lower or the upper halves of two dwords as one.
template <bool UPPER>
__device__ __forceinline__ uint32_t halves_of(uint32_t first, uint32_t second) {
  return __builtin_amdgcn_perm(second, first, UPPER ? 0x07060302u : 0x05040100u);
}

// uc_paged_tiles.hip: many query rows.
int64_t tile_workgroups(int64_t lists, int64_t groups);
int launch_tiles(const char *what, int dtype, int64_t head_dim, const Cache &c, const Query &q, const Plan &p, uint16_t *out,
                 float *lse, float *part, float *stat, hipStream_t stream);

}  // namespace pg
}  // namespace uc
