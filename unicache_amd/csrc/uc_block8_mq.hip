// Attention over the 8-bit block-scaled cache for many query rows: prompts,
// image edits, selected blocks of a prompt's chunk.  The mathematics is that of
// uc_block8_attn.hip.
//
// A workgroup owns 128 query rows of one KV head, 32 per wave, and walks 64-key
// tiles.  Its 256 threads read the next tile's codes into registers (16 bytes
// each, 16 in all at D = 128) while the present one is computed, turn them into
// fp16 once for all rows, and write the other of two LDS buffers: one barrier a
// tile.  The scales of a tile are two scalars (its halves may lie in two
// blocks), so the codes are never multiplied.
//
// LDS rows (a key's channels, a channel's keys) hold 16-byte chunks in swizzled
// order, so that the fragments' 16-byte reads meet no bank twice.  Key tile j's row r is key
// 32 (j / 2) + 8 (r / 4) + 4 (j % 2) + r % 4, so that a lane's logits of two tiles are
// eight consecutive keys of its query row: the operand of O^T = V^T P^T.
#include "uc_block8_attn.h"

namespace uc {
namespace b8 {
namespace {

typedef uint32_t u4v __attribute__((ext_vector_type(4)));

template <int D>
struct Tile {
  static constexpr int kKeyRow = D * 2, kValueRow = kTile * 2;      // bytes
  static constexpr int kKeyBytes = kTile * kKeyRow, kValueBytes = D * kValueRow;
  static constexpr int kBytes = kKeyBytes + kValueBytes;            // of one buffer
  static constexpr int kLoads = kTile * D / 16 / 256;               // 16-byte loads per thread, keys and values each
};

// A tile's codes on their way to LDS, and its scales.
template <int D>
struct Staged {
  uint4 k[Tile<D>::kLoads], v[Tile<D>::kLoads];
  float ks[2], vs[2];
  int32_t t[2];  // first keys of the halves
};

template <int D>
__device__ __forceinline__ void fetch(Staged<D> &st, const Cache &c, int64_t sh, const uint8_t *kbase,
                                      const uint8_t *vbase, int32_t t0, int32_t t1) {
  constexpr int kPerKey = D / 16;
  st.t[0] = t0;
  st.t[1] = t1;
  const int32_t a0 = t0 == kNone ? 0 : t0, a1 = t1 == kNone ? 0 : t1;
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    const int key = threadIdx.x / kPerKey + i * (256 / kPerKey);
    const int32_t t = (key < 32 ? a0 : a1 - 32) + key;
    st.k[i] = *reinterpret_cast<const uint4 *>(kbase + int64_t(t) * D + threadIdx.x % kPerKey * 16);
    const int channel = threadIdx.x / 4 + i * 64, k16 = threadIdx.x % 4;
    const int32_t u = (k16 < 2 ? a0 : a1) + (k16 & 1) * 16;
    st.v[i] = *reinterpret_cast<const uint4 *>(vbase + (int64_t(u >> c.shift) << c.shift) * D + channel * c.block +
                                               (u & (c.block - 1)));
  }
  const int64_t b = sh * c.blocks;
  st.ks[0] = c.key_scale[b + (a0 >> c.shift)];
  st.ks[1] = c.key_scale[b + (a1 >> c.shift)];
  st.vs[0] = c.value_scale[b + (a0 >> c.shift)];
  st.vs[1] = c.value_scale[b + (a1 >> c.shift)];
}

// The order of a key's chunks in LDS.
__device__ __forceinline__ int key_swizzle(int key) { return (key & 3) | ((key >> 3) & 3) << 2; }

template <int D, int CODE>
__device__ __forceinline__ void store(Staged<D> &st, char *buf, int32_t length) {
  constexpr int kPerKey = D / 16, kChunks = D / 8;
  if (st.t[0] + 32 > length || st.t[1] + 32 > length) {  // codes behind the length are no values
    const int32_t k16 = threadIdx.x % 4;
    const int32_t u = (k16 < 2 ? st.t[0] : st.t[1]) + (k16 & 1) * 16;
#pragma unroll
    for (int i = 0; i < Tile<D>::kLoads; ++i) st.v[i] = first_bytes(st.v[i], length - u);
  }
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    const int key = threadIdx.x / kPerKey + i * (256 / kPerKey), c16 = threadIdx.x % kPerKey;
    char *row = buf + key * Tile<D>::kKeyRow;
    const int sw = key_swizzle(key) & (kChunks - 1);
    // eight lanes hold one key at D = 128: half of them write their second chunk first
    const int odd = D == 128 ? (c16 >> 2) & 1 : 0;
    const uint32_t x0 = odd ? st.k[i].z : st.k[i].x, y0 = odd ? st.k[i].w : st.k[i].y;
    const uint32_t x1 = odd ? st.k[i].x : st.k[i].z, y1 = odd ? st.k[i].y : st.k[i].w;
    *reinterpret_cast<h8 *>(row + 16 * ((2 * c16 + odd) ^ sw)) = codes_to_h8<CODE>(x0, y0);
    *reinterpret_cast<h8 *>(row + 16 * ((2 * c16 + (odd ^ 1)) ^ sw)) = codes_to_h8<CODE>(x1, y1);
    const int channel = threadIdx.x / 4 + i * 64, k16 = threadIdx.x % 4;
    char *vrow = buf + Tile<D>::kKeyBytes + channel * Tile<D>::kValueRow;
    *reinterpret_cast<h8 *>(vrow + 16 * ((2 * k16) ^ (channel & 7))) = codes_to_h8<CODE>(st.v[i].x, st.v[i].y);
    *reinterpret_cast<h8 *>(vrow + 16 * ((2 * k16 + 1) ^ (channel & 7))) = codes_to_h8<CODE>(st.v[i].z, st.v[i].w);
  }
}

// Sixteen query rows of a wave: the lane's row is lane % 16.
template <int D>
struct Acc16 {
  f4 o[D / 16];
  float m, l;
};

// Weights of one tile for 16 rows; ends[h]: keys of half h that the lane's row sees, from its own first key on.
template <int D, bool MASK>
__device__ __forceinline__ void weights(Acc16<D> &acc, const f4 (&s)[4], const float (&c)[2], const float (&lv)[2],
                                        const float (&inv)[2], const int32_t (&ends)[2], h8 (&p)[2]) {
  float x[MASK ? 16 : 1];
  float top = mf::kNegInf;
  if constexpr (MASK) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int h = j / 8;
      x[j] = j % 8 < ends[h] ? __builtin_fmaf(s[j / 4][j % 4], c[h], lv[h]) : mf::kNegInf;
      top = fmaxf(top, x[j]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float t = s[2 * h][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) t = fmaxf(t, s[2 * h + j / 4][j % 4]);
      top = fmaxf(top, __builtin_fmaf(t, c[h], lv[h]));
    }
  }
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
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float sum = 0.0f;
    const float shift = lv[h] - m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = mf::fast_exp2(MASK ? x[MASK ? 8 * h + j : 0] - m : __builtin_fmaf(s[2 * h + j / 4][j % 4], c[h], shift));
      sum += e;
      p[h][j] = mf::to_h(e);
    }
    if constexpr (MASK) {
      acc.l += sum == 0.0f ? 0.0f : sum * inv[h];
    } else {
      acc.l = __builtin_fmaf(sum, inv[h], acc.l);
    }
  }
}

template <int D, int CODE>
__global__ __launch_bounds__(256, 2) void tile_kernel(Cache c, Query q, Plan p, uint32_t units, uint16_t *out, float *lse,
                                                      float *part, float *stat) {
  typedef Tile<D> T;
  __shared__ __attribute__((aligned(16))) char lds[2 * T::kBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int32_t split = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  const Rows w = rows_of(c, q, p, unit, kTileRows);
  const int32_t tiles = tiles_of(c, p, w), per = split_tiles_of(p, tiles);
  const int32_t begin = split * per, end = begin + per < tiles ? begin + per : tiles;
  if (begin >= end && split > 0) return;
  const int64_t sh = int64_t(w.s) * c.heads + w.h;
  const int32_t *list =
      p.list == nullptr ? nullptr : p.list + ((int64_t(w.s) * p.runs + w.run0 / p.run) * c.heads + w.h) * p.budget;
  const int32_t tokens = c.blocks << c.shift;
  const uint8_t *kbase = c.key_code + sh * tokens * D, *vbase = c.value_code + sh * tokens * D;

  h8 frag[2][D / 32];
  float factor[2];
  int32_t row_end[2];
  Acc16<D> acc[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int32_t r = w.r0 + wave * 32 + n * 16 + col;
    factor[n] = load_query<D, false>(q, w, r, frag[n]);
    const int32_t e = visible(q, w.length, w.count, w.run0 + token_of(q, r));
    row_end[n] = e < w.length ? e : w.length;
    acc[n].m = mf::kNegInf;
    acc[n].l = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[n].o[d] = f4{0, 0, 0, 0};
  }
  // LDS offsets of the fragments: key tile j adds (32 (j / 2) + 4 (j % 2)) rows, channel tile n 16 rows
  const int krow = (col >> 2) * 8 + (col & 3);
  int ka[D / 32], va[2];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) ka[k] = krow * T::kKeyRow + 16 * ((4 * k + quad) ^ (key_swizzle(krow) & (D / 8 - 1)));
#pragma unroll
  for (int h = 0; h < 2; ++h) va[h] = T::kKeyBytes + col * T::kValueRow + 16 * ((4 * h + quad) ^ (col & 7));

  float most = 0.0f;
  Staged<D> st;
  auto get = [&](int32_t t) {
    int32_t t0 = half_of(c, p, list, 2 * t), t1 = half_of(c, p, list, 2 * t + 1);
    if (t1 >= tokens) t1 = kNone;
    fetch<D>(st, c, sh, kbase, vbase, t0, t1);
  };
  if (begin < end) {
    get(begin);
    store<D, CODE>(st, lds, w.length);
  }
  __syncthreads();
  for (int32_t t = begin; t < end; ++t) {
    const char *buf = lds + ((t - begin) & 1) * T::kBytes;
    char *other = lds + ((t - begin + 1) & 1) * T::kBytes;
    const int32_t t0 = st.t[0], t1 = st.t[1];
    float ks[2], vs[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      ks[h] = st.ks[h];
      vs[h] = counted_scale(st.t[h] < w.length ? st.vs[h] : 1.0f, most);
    }
    const bool more = t + 1 < end;
    if (more) get(t + 1);

    f4 s[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[0][j] = s[1][j] = f4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const h8 a = *reinterpret_cast<const h8 *>(buf + ka[k] + (32 * (j / 2) + 4 * (j % 2)) * T::kKeyRow);
        s[0][j] = mf::mfma32(a, frag[0][k], s[0][j]);
        s[1][j] = mf::mfma32(a, frag[1][k], s[1][j]);
      }
    }
    h8 pr[2][2];
    const float lv[2] = {__builtin_amdgcn_logf(vs[0]), __builtin_amdgcn_logf(vs[1])};
    const float inv[2] = {__builtin_amdgcn_rcpf(vs[0]), __builtin_amdgcn_rcpf(vs[1])};
    const bool whole = (t0 > t1 ? t0 : t1) + 32 <= w.end_first;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const float cc[2] = {ks[0] * factor[n], ks[1] * factor[n]};
      const int32_t ends[2] = {row_end[n] - t0 - 8 * quad, row_end[n] - t1 - 8 * quad};
      if (whole) {
        weights<D, false>(acc[n], s[n], cc, lv, inv, ends, pr[n]);
      } else {
        weights<D, true>(acc[n], s[n], cc, lv, inv, ends, pr[n]);
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const h8 a = *reinterpret_cast<const h8 *>(buf + va[h] + d * 16 * T::kValueRow);
        acc[0].o[d] = mf::mfma32(a, pr[0][h], acc[0].o[d]);
        acc[1].o[d] = mf::mfma32(a, pr[1][h], acc[1].o[d]);
      }
    }
    if (more) store<D, CODE>(st, other, w.length);
    __syncthreads();
  }

#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int32_t rr = wave * 32 + n * 16 + col, r = w.r0 + rr;
    const float total = mf::sum_over_slices(acc[n].l);
    if (p.splits > 1) {
      const int64_t at = int64_t(blockIdx.x) * kTileRows + rr;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f4 *>(part + at * D + 16 * d + 4 * quad) = acc[n].o[d];
      if (quad == 0) {
        stat[2 * at] = acc[n].m;
        stat[2 * at + 1] = total;
      }
    } else if (r < w.run_rows) {
      const int32_t token = w.run0 + token_of(q, r), head = w.h * q.group + r - token_of(q, r) * q.group;
      const bool none = token >= w.count || total == 0.0f;
      const float f = none ? 0.0f : 1.0f / total;
      uint16_t *dst = out + ((int64_t(w.s) * q.len + token) * q.heads + head) * D + 4 * quad;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint16_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = none ? 0.0f : acc[n].o[d][i] * f;
          v[i] = q.fp16 ? f32_to_f16_bits(x) : f32_to_bf16_bits(x);
        }
        *reinterpret_cast<uint2 *>(dst + 16 * d) = uint2{v[0] | (uint32_t(v[1]) << 16), v[2] | (uint32_t(v[3]) << 16)};
      }
      if (quad == 0 && lse != nullptr) {
        lse[(int64_t(w.s) * q.heads + head) * q.len + token] =
            none ? mf::kNegInf : kLn2 * (acc[n].m + __builtin_amdgcn_logf(total));
      }
    }
  }
}

}  // namespace

int launch_tiles(const uc_block8_cache *cache, const Cache &c, const Query &q, const Plan &p, uint32_t workgroups,
                 uint16_t *out, float *lse, float *part, float *stat, hipStream_t stream) {
  return UC_B8_DISPATCH(cache, cache->head_dim, [&] {
    hipLaunchKernelGGL((tile_kernel<D, CODE>), dim3(workgroups), dim3(256), 0, stream, c, q, p, workgroups / p.splits, out,
                       lse, part, stat);
    return check_launch("uc_block8_attn");
  });
}

}  // namespace b8
}  // namespace uc
