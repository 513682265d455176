// Attention over the 8-bit block-scaled cache for many query rows: prompts,
// image edits, selected blocks of a prompt's chunk.  The mathematics is that of
// uc_block8_attn.hip.
//
// A workgroup owns 128 query rows of one KV head, 32 per wave, and walks 64-key
// tiles.  Its 256 threads read the next tile's codes into registers (16 bytes
// each, 16 in all at D = 128) while the present one is computed, turn them into
// fp16 once for all rows, and write the other of two LDS buffers: one barrier a
// tile.  The scales of a tile are two scalars (its halves may lie in two
// blocks), so the codes are never multiplied; only in masked tiles of two blocks each row has value scales
// of its own (3 x 777 padded prompts 47.9 us without that, which lost keys beside very large values, and 48.9).
// At D = 64 a tile has half the MFMAs and the same weights: 8.8 other vector instructions a MFMA, 3.7 at 128.
//
// LDS rows (a key's channels, a channel's keys) hold 16-byte chunks in swizzled
// order, so that the fragments' 16-byte reads meet no bank twice.  Key tile j's row r is key
// 32 (j / 2) + 8 (r / 4) + 4 (j % 2) + r % 4, so that a lane's logits of two tiles are
// eight consecutive keys of its query row: the operand of O^T = V^T P^T.
//
// Bound by the vector instructions beside the matrix cores: at D = 128 a wave's tile is 64 MFMAs
// (1,024 cycles) and about 235 other vector instructions (the exponentials and what leads to
// them, the maxima, the casts, the next tile's conversion).  The cores are busy about 47 % of the
// time, the LDS 35 %, without a bank conflict.  4096 causal queries behind 12k tokens of 32/8 heads:
// 859 to 908 us by card, 1,060 to 1,120 TFLOP/s; a large library product reaches 1,355.  64 rows a wave would halve the
// LDS reads but need twice the accumulators.  The matrix phases run at raised priority, so that
// the wave that is in one keeps the cores fed.  Codes converted a tile earlier, beside the Q K
// products, were 7 % slower.
#include "uc_block8_attn.h"

#include <type_traits>

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

// What a thread loads.  A load's 256 threads take one half tile (at D = 64: the first two waves one
// half, the last two the other), so its address is a scalar and a constant of the lane.
template <int D>
struct Loader {
  int key, c16;       // keys: the key in its half, 16 channels
  int channel, k16;   // values: the channel, 16 keys of its half
  uint32_t koff, voff;

  __device__ __forceinline__ explicit Loader(int32_t block) {
    const int tid = threadIdx.x & 255;
    if constexpr (D == 128) {
      // eight lanes write two keys' chunks to LDS, so that they meet no bank twice
      c16 = (tid & 3) | ((tid >> 3) & 1) << 2;
      key = ((tid >> 2) & 1) | (tid >> 4) << 1;
    } else {
      c16 = tid & 3;
      key = (tid >> 2) & 31;
    }
    channel = (tid >> 1) & (D - 1);
    k16 = tid & 1;
    koff = key * D + c16 * 16;
    voff = channel * block + k16 * 16;
  }
  // The half of load i: the same for a wave.
  __device__ __forceinline__ int half(int i) const { return D == 128 ? i : __builtin_amdgcn_readfirstlane((threadIdx.x >> 7) & 1); }
};

template <int D>
__device__ __forceinline__ void fetch(Staged<D> &st, const Cache &c, int64_t sh, const uint8_t *kbase,
                                      const uint8_t *vbase, const Loader<D> &ld, int32_t t0, int32_t t1) {
  st.t[0] = t0;
  st.t[1] = t1;
  const int32_t a[2] = {t0 == kNone ? 0 : t0, t1 == kNone ? 0 : t1};
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    const int32_t t = ld.half(i) ? a[1] : a[0];
    st.k[i] = *reinterpret_cast<const uint4 *>(kbase + int64_t(t) * D + ld.koff);
    st.v[i] = *reinterpret_cast<const uint4 *>(vbase + ((int64_t(t >> c.shift) << c.shift) * D + (t & (c.block - 1))) + ld.voff);
  }
  const int64_t b = sh * c.blocks;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    st.ks[h] = c.key_scale[b + (a[h] >> c.shift)];
    st.vs[h] = c.value_scale[b + (a[h] >> c.shift)];
  }
}

// The orders of a key's and of a channel's chunks in LDS.
__device__ __forceinline__ int key_swizzle(int key) { return (key & 3) | ((key >> 3) & 3) << 2; }
__device__ __forceinline__ int value_swizzle(int channel) {
  return (channel & 1) | ((channel >> 2) & 1) << 1 | ((channel >> 1) & 1) << 2;
}

// Codes behind the length are no values.
template <int D>
__device__ __forceinline__ void clear(Staged<D> &st, const Loader<D> &ld, int32_t length) {
  if (st.t[0] + 32 > length || st.t[1] + 32 > length) {
#pragma unroll
    for (int i = 0; i < Tile<D>::kLoads; ++i) {
      st.v[i] = first_bytes(st.v[i], length - (ld.half(i) ? st.t[1] : st.t[0]) - ld.k16 * 16);
    }
  }
}

template <int D, int CODE>
__device__ __forceinline__ void store_keys(const Staged<D> &st, char *buf, const Loader<D> &ld) {
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    char *row = buf + (ld.key + 32 * ld.half(i)) * Tile<D>::kKeyRow;
    const int sw = key_swizzle(ld.key) & (D / 8 - 1);
    *reinterpret_cast<h8 *>(row + 16 * ((2 * ld.c16) ^ sw)) = codes_to_h8<CODE>(st.k[i].x, st.k[i].y);
    *reinterpret_cast<h8 *>(row + 16 * ((2 * ld.c16 + 1) ^ sw)) = codes_to_h8<CODE>(st.k[i].z, st.k[i].w);
  }
}

template <int D, int CODE>
__device__ __forceinline__ void store_values(const Staged<D> &st, char *buf, const Loader<D> &ld) {
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    char *row = buf + Tile<D>::kKeyBytes + ld.channel * Tile<D>::kValueRow;
    const int chunk = 4 * ld.half(i) + 2 * ld.k16, sw = value_swizzle(ld.channel);
    *reinterpret_cast<h8 *>(row + 16 * (chunk ^ sw)) = codes_to_h8<CODE>(st.v[i].x, st.v[i].y);
    *reinterpret_cast<h8 *>(row + 16 * ((chunk + 1) ^ sw)) = codes_to_h8<CODE>(st.v[i].z, st.v[i].w);
  }
}

// Sixteen query rows of a wave: the lane's row is lane % 16.
template <int D>
struct Acc16 {
  f4 o[D / 16];
  float m, l;
};

// A logit of one row, as the exponent of its weight.
template <bool MASK>
__device__ __forceinline__ float exponent(float s, float c, float shift, bool seen) {
  const float x = __builtin_fmaf(s, c, shift);
  return MASK && !seen ? mf::kNegInf : x;
}

// The reference of 16 rows' weights, raised where one of the tile's logits asks for it.  N == 2: its halves are
// in two blocks; else one scale of each kind is the tile's.  ends[h]: keys of half h that the lane's
// row sees, from its own first key on.
template <int D, bool MASK, int N>
__device__ __forceinline__ float reference(Acc16<D> &acc, const f4 (&s)[4], const float (&c)[N], const float (&lv)[N],
                                           const int32_t (&ends)[2]) {
  constexpr int kK = 16 / N;  // logits of a lane per scale
  float top = mf::kNegInf;
  if constexpr (MASK) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      top = fmaxf(top, exponent<true>(s[j / 4][j % 4], c[j / kK], lv[j / kK], j % 8 < ends[j / 8]));
    }
  } else {
#pragma unroll
    for (int h = 0; h < N; ++h) {
      float t = mf::kNegInf;
#pragma unroll
      for (int j = h * kK; j < (h + 1) * kK; ++j) t = fmaxf(t, s[j / 4][j % 4]);
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
  return acc.m == mf::kNegInf ? 0.0f : acc.m;
}

// The weights of half a tile, and their sum.
template <bool MASK>
__device__ __forceinline__ float weights(const f4 (&s)[4], int half, float c, float lv, float inv, float m,
                                         int32_t end, float l, h8 &p) {
  float sum = 0.0f;
  const float shift = lv - m;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float e = mf::fast_exp2(exponent<MASK>(s[2 * half + j / 4][j % 4], c, shift, j < end));
    sum = j == 0 ? e : sum + e;
    p[j] = mf::to_h(e);
  }
  if constexpr (MASK) return l + (sum == 0.0f ? 0.0f : sum * inv);
  return __builtin_fmaf(sum, inv, l);
}

// The second group's rows join the first's, lane by lane, through LDS (which nobody reads any more).
template <int D>
__device__ __forceinline__ void join_groups(Acc16<D> (&acc)[2], f4 *sh, int part_of, int wave) {
  constexpr int kO = D / 16;
  const int lane = threadIdx.x & 63;
  f4 *at = sh + wave * 2 * (kO + 1) * 64 + lane;
  if (part_of == 1) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int d = 0; d < kO; ++d) at[(n * (kO + 1) + d) * 64] = acc[n].o[d];
      at[(n * (kO + 1) + kO) * 64] = f4{acc[n].m, acc[n].l, 0, 0};
    }
  }
  __syncthreads();
  if (part_of == 1) return;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const f4 s = at[(n * (kO + 1) + kO) * 64];
    const float m = fmaxf(acc[n].m, s[0]);
    const float d0 = m == mf::kNegInf ? 0.0f : acc[n].m - m, d1 = m == mf::kNegInf ? 0.0f : s[0] - m;
    const float f0 = mf::fast_exp2(d0), f1 = mf::fast_exp2(d1);
    acc[n].m = m;
    acc[n].l = rescaled(acc[n].l, d0) + rescaled(s[1], d1);
#pragma unroll
    for (int d = 0; d < kO; ++d) {
      const f4 o = at[(n * (kO + 1) + d) * 64];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n].o[d][i] = acc[n].o[d][i] * f0 + o[i] * f1;
    }
  }
}

template <int D, int CODE, int N, bool LISTED, int G>
__global__ __launch_bounds__(256 * G, 2) void tile_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse,
                                                      float *part, float *stat) {
  typedef Tile<D> T;
  __shared__ __attribute__((aligned(16))) char lds_all[2 * G * T::kBytes];
  // G == 2: two groups of four waves hold the same rows and take half of the tiles each
  const int part_of = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  char *const lds = lds_all + part_of * 2 * T::kBytes;
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & 3, col = lane & 15, quad = lane >> 4;
  // Two waves share a SIMD: of two groups, or in slots of the SIMD that differ in their last bit (HW_ID's first four bits).
  // One goes before the other in its vector phases, so that they do not reach the matrix cores
  // together (without: prefill 4k 914 us, edit 50.6; with: 894, 48.5).
  const bool before = (G == 2 ? part_of : __builtin_amdgcn_s_getreg((3 << 11) | 4) & 1) != 0;
  auto vector_phase = [&] {
    if (before) {
      __builtin_amdgcn_s_setprio(1);
    } else {
      __builtin_amdgcn_s_setprio(0);
    }
  };
  // Workgroups go to the 8 XCDs in turn.  A list is one split of the keys of one (sequence, head, run);
  // its row groups are dealt into `deal` hands so that 8 divides the number of hands, and an XCD plays whole hands:
  // its L2 then holds the keys of few lists (8 heads of 16k tokens: 1011 -> 908 us).
  const int32_t lists = c.sequences * c.heads * p.runs * p.splits, deal = 8 / (lists & 7 ? lists & -lists : 8);
  const int32_t slots = (p.groups + deal - 1) / deal, x = blockIdx.x & 7, at = blockIdx.x >> 3, turn = at / slots;
  const int32_t hand = x + 8 * turn, list_index = hand % lists, group = (at - turn * slots) * deal + hand / lists;
  if (group >= p.groups) return;
  const int32_t split = list_index % p.splits;
  // the later rows of a causal run see more keys: the longest first
  const int32_t unit = list_index / p.splits * p.groups + (q.causal ? p.groups - 1 - group : group);
  const Rows w = rows_of(c, q, p, unit, kTileRows);
  const int32_t tiles = tiles_of(c, p, w), per = split_tiles_of(p, tiles);
  const int32_t begin0 = split * per, end0 = begin0 + per < tiles ? begin0 + per : tiles;
  if (begin0 >= end0 && split > 0) return;
  const int32_t steps = end0 > begin0 ? (end0 - begin0 + G - 1) / G : 0;  // of a group; the second may have one less
  const int32_t begin = begin0 + part_of * steps, end = begin + steps < end0 ? begin + steps : end0;
  const int64_t sh = int64_t(w.s) * c.heads + w.h;
  BlockList list(c, p, w);
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
  for (int h = 0; h < 2; ++h) va[h] = T::kKeyBytes + col * T::kValueRow + 16 * ((4 * h + quad) ^ value_swizzle(col));

  float most = 0.0f;  // the largest value scale so far
  Staged<D> st;
  const Loader<D> ld(c.block);
  auto get = [&](int32_t t) {
    const int32_t t0 = half_of<LISTED>(c, list, 2 * t), t1 = half_of<LISTED>(c, list, 2 * t + 1);
    fetch<D>(st, c, sh, kbase, vbase, ld, t0, t1);
  };
  // whether every row sees all keys of the staged tile
  auto whole = [&] { return (st.t[0] > st.t[1] ? st.t[0] : st.t[1]) + 32 <= w.end_first; };
  int32_t t = begin;
  int present = 0;  // LDS offset of the tile's buffer
  auto step = [&](auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const char *buf = lds + present;
    const int32_t t0 = st.t[0], t1 = st.t[1];
    // (one block: the halves' scales are the same, and the first is there if any is)
    // Masked halves of two blocks: a row goes by the scales that it sees, so they count for each row by itself.
    constexpr int R = MASK && N == 2 ? 2 : 1;
    float ks[N], lv[R][N], inv[R][N];
#pragma unroll
    for (int h = 0; h < N; ++h) ks[h] = st.ks[h];
    const float before = most;
#pragma unroll
    for (int h = 0; h < N; ++h) most = !MASK || st.t[h] < w.length ? larger_scale(most, st.vs[h]) : most;
#pragma unroll
    for (int n = 0; n < R; ++n) {
      float seen = most;
      if constexpr (R == 2) {
        seen = t0 < row_end[n] ? larger_scale(before, st.vs[0]) : before;
        seen = t1 < row_end[n] ? larger_scale(seen, st.vs[N - 1]) : seen;
      }
#pragma unroll
      for (int h = 0; h < N; ++h) {
        const bool there = !MASK || st.t[h] < (R == 2 ? row_end[n] : w.length);
        const float vs = there ? counted_scale(st.vs[h], seen) : 1.0f;
        lv[n][h] = __builtin_amdgcn_logf(vs);
        inv[n][h] = __builtin_amdgcn_rcpf(vs);
      }
    }
    const bool more = t + 1 < end;
    if (more) get(t + 1);

    __builtin_amdgcn_s_setprio(3);
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
    vector_phase();
    h8 pr[2][2];
    float cc[2][N], m[2];
    int32_t ends[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int h = 0; h < N; ++h) cc[n][h] = ks[h] * factor[n];
      ends[n][0] = row_end[n] - t0 - 8 * quad;
      ends[n][1] = row_end[n] - t1 - 8 * quad;
      m[n] = reference<D, MASK, N>(acc[n], s[n], cc[n], lv[n % R], ends[n]);
    }
    auto weigh = [&](int h) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int b = h * (N - 1);
        acc[n].l = weights<MASK>(s[n], h, cc[n][b], lv[n % R][b], inv[n % R][b], m[n], ends[n][h], acc[n].l, pr[n][h]);
      }
    };
    weigh(0);
    // The second half's weights take their turns beside the first's P V products, and the next tile's
    // codes become fp16 beside the second's (after the last tile the present one's again, into the
    // buffer that nobody reads): prefill 4k 859 us, 898 with the weights before the products and codes beside
    // both.  Lists and 64 channels, whose workgroups are few or have half the products, do better the
    // second way (sparse prefill 164, 167; 3 x 777 tokens 48.9, 49.6).
    constexpr bool kEarly = D == 64 || LISTED;
    if constexpr (kEarly) weigh(1);
    clear<D>(st, ld, w.length);
    present ^= T::kBytes;
    __builtin_amdgcn_s_setprio(3);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      h8 a[D / 16];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) a[d] = *reinterpret_cast<const h8 *>(buf + va[h] + d * 16 * T::kValueRow);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        acc[0].o[d] = mf::mfma32(a[d], pr[0][h], acc[0].o[d]);
        acc[1].o[d] = mf::mfma32(a[d], pr[1][h], acc[1].o[d]);
      }
      if (!kEarly && h == 0) {
        weigh(1);
        if constexpr (!MASK) {  // (masked tiles have more vector instructions than this order provides for)
          __builtin_amdgcn_sched_group_barrier(0x100, D / 16, 0);  // the values
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);    // a product,
            __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);  // an exponential
            __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);    // and other vector instructions
          }
        }
      }
      if (kEarly ? h == 0 : h == 1) store_keys<D, CODE>(st, lds + present, ld);
      if (h == 1) store_values<D, CODE>(st, lds + present, ld);
    }
    vector_phase();
    __syncthreads();
    ++t;
  };
  if (begin < end) {
    get(begin);
    clear<D>(st, ld, w.length);
    store_keys<D, CODE>(st, lds, ld);
    store_values<D, CODE>(st, lds, ld);
  }
  __syncthreads();
  // tiles that every row sees come first; from the first other one on, every tile is masked
  while (t < end && whole()) step(std::false_type());
  while (t < end) step(std::true_type());
  if constexpr (G == 2) {
    if (end - begin < steps) __syncthreads();  // the other group's last tile
    join_groups<D>(acc, reinterpret_cast<f4 *>(lds_all), part_of, wave);
    if (part_of == 1) return;
  }

#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int32_t rr = wave * 32 + n * 16 + col, r = w.r0 + rr;
    const float total = mf::sum_over_slices(acc[n].l);
    if (p.splits > 1) {
      if (r >= w.run_rows) continue;
      const int64_t at = (int64_t(unit) * p.splits + split) * kTileRows + rr;
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
        const f4 x = none ? f4{0, 0, 0, 0} : acc[n].o[d] * f;
        *reinterpret_cast<uint2 *>(dst + 16 * d) = uint2{pack2(x[0], x[1], q.fp16), pack2(x[2], x[3], q.fp16)};
      }
      if (quad == 0 && lse != nullptr) {
        lse[(int64_t(w.s) * q.heads + head) * q.len + token] =
            none ? mf::kNegInf : kLn2 * (acc[n].m + __builtin_amdgcn_logf(total));
      }
    }
  }
}

template <int D, int CODE, int N, class... Args>
void launch_tile(bool listed, int groups, uint32_t workgroups, hipStream_t stream, const Args &...args) {
  if (listed) {
    hipLaunchKernelGGL((tile_kernel<D, CODE, N, true, 1>), dim3(workgroups), dim3(256), 0, stream, args...);
  } else if (groups == 2) {
    hipLaunchKernelGGL((tile_kernel<D, CODE, N, false, 2>), dim3(workgroups), dim3(512), 0, stream, args...);
  } else {
    hipLaunchKernelGGL((tile_kernel<D, CODE, N, false, 1>), dim3(workgroups), dim3(256), 0, stream, args...);
  }
}

}  // namespace

int launch_tiles(const uc_block8_cache *cache, const Cache &c, const Query &q, const Plan &p, uint16_t *out, float *lse,
                 float *part, float *stat, hipStream_t stream) {
  // (the hands may be one row group longer than they need to be)
  const int64_t lists = int64_t(c.sequences) * c.heads * p.runs * p.splits, deal = 8 / (lists & 7 ? lists & -lists : 8);
  UC_REQUIRE(lists * deal * ceil_div(p.groups, deal) < (1 << 24) / p.key_groups, "uc_block8_attn: too many query rows");
  const uint32_t workgroups = static_cast<uint32_t>(lists * deal * ceil_div(p.groups, deal));
  return UC_B8_DISPATCH(cache, cache->head_dim, [&] {
    if (c.block == 32) {
      launch_tile<D, CODE, 2>(p.list != nullptr, p.key_groups, workgroups, stream, c, q, p, out, lse, part, stat);
    } else {
      launch_tile<D, CODE, 1>(p.list != nullptr, p.key_groups, workgroups, stream, c, q, p, out, lse, part, stat);
    }
    return check_launch("uc_block8_attn");
  });
}

}  // namespace b8
}  // namespace uc
