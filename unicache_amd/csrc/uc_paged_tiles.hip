// Attention over the paged 16-bit cache for many query rows: a prompt's chunk, an image's queries.
// The mathematics is that of uc_paged_attn.hip, but for the weights, which go into the products as one 16-bit number
// (half a step, 2^-8 in bf16, 2^-11 in fp16, of each at most; over 13k keys outputs lie 2.3e-3 from 64-bit arithmetic,
// 1.7e-3 of it their own rounding): the matrix cores, not the loads, are what such calls wait for.
//
// A workgroup owns 128 query rows of one KV head, 32 per wave, and walks 64-key tiles.  Its 256 threads
// read the next tile into registers while the present one is computed, and write the other of two LDS
// buffers: one barrier a tile.  Keys lie there as rows, values channel by channel, as the products read them: a
// thread takes D/32 channels of eight keys and turns them round with one byte permutation per pair of keys
// and channel.  16 keys lie in one page, so each load of a wave has its page in scalar registers.
//
// LDS rows (a key's channels, a channel's keys) hold 16-byte chunks in swizzled order, so that the fragments'
// 16-byte reads meet no bank twice.  Key tile j's row r is key 32 (j / 2) + 8 (r / 4) + 4 (j % 2) + r % 4, so that a lane's
// logits of two tiles are eight consecutive keys of its query row: the operand of O^T = V^T P^T.
//
// Bound by phases that overlap in part: at D = 128 a wave's tile is 64 MFMAs (1,024 cycles), about 190 other vector
// instructions (32 exponentials among them) and 32 KB of LDS reads, each about 40 % of what two waves a SIMD could
// have.  2 x 2k causal queries (32/8 heads) behind 11k tokens: 705 to 760 us by box, up to 930
// TFLOP/s; 4096 of 16k not causal 1,058 to 1,105 us, 995 to 1,039; a large library product reaches 1,413.
#include "uc_paged_attn.h"

#include <type_traits>

namespace uc {
namespace pg {
namespace {

template <int D>
struct Tile {
  static constexpr int kKeyRow = D * 2, kValueRow = kKeys * 2;      // bytes
  static constexpr int kKeyBytes = kKeys * kKeyRow, kValueBytes = D * kValueRow;
  static constexpr int kBytes = kKeyBytes + kValueBytes;            // of one buffer
  static constexpr int kLoads = kKeys * D / 8 / 256;                // 16-byte loads of keys per thread
  static constexpr int kChannels = D / 32;                          // of a thread's values
};

// A tile on its way to LDS.
template <int D>
struct Staged {
  u4 k[Tile<D>::kLoads];
  uint32_t v[8][D / 64];
  int32_t t;        // its first key
  uint32_t absent;  // bit i: its keys 16 i .. 16 i + 15 have no page
};

// Table entries of a tile to come.  WHOLE: pages of 64 tokens or more, one entry a tile; else those of each 16 keys, and
// of a wave's loads.
template <int D, bool WHOLE>
struct Entries {
  int32_t quarter[WHOLE ? 1 : 4], key[WHOLE ? 1 : Tile<D>::kLoads], value;
};

// What a thread loads: a chunk of keys (16 lanes, at D = 64 eight, a key), and channels of eight keys.
template <int D>
struct Loader {
  int key, chunk, group, channel, wave;
  uint32_t koff, voff;

  __device__ __forceinline__ Loader() {
    const int tid = threadIdx.x;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    chunk = tid & (D / 8 - 1);
    key = tid / (D / 8);
    group = tid >> 5;
    channel = (tid & 31) * Tile<D>::kChannels;
    koff = (key & 15) * D + chunk * 8;
    voff = (group & 1) * 8 * D + channel;
  }
  // The quarter of key load i: the same for a wave.
  __device__ __forceinline__ int32_t quarter(int i) const { return D == 128 ? i : 2 * i + (wave >> 1); }
};

template <int D, bool WHOLE>
__device__ __forceinline__ void ask(Entries<D, WHOLE> &e, const Pages &pages, const Loader<D> &ld, int32_t t) {
#pragma unroll
  for (int i = 0; i < (WHOLE ? 1 : 4); ++i) e.quarter[i] = pages.of(t + 16 * i);
  if constexpr (!WHOLE) {
#pragma unroll
    for (int i = 0; i < Tile<D>::kLoads; ++i) e.key[i] = D == 128 ? e.quarter[i] : pages.of(t + 16 * ld.quarter(i));
    e.value = pages.of(t + 16 * ld.wave);
  }
}

template <int D, bool WHOLE>
__device__ __forceinline__ void fetch(Staged<D> &st, const Cache &c, const Entries<D, WHOLE> &e, const uint16_t *key,
                                      const uint16_t *value, const Loader<D> &ld, int32_t t) {
  st.t = t;
  st.absent = 0;
#pragma unroll
  for (int i = 0; i < (WHOLE ? 1 : 4); ++i) st.absent |= c.is_page(e.quarter[i]) ? 0u : WHOLE ? 15u : 1u << i;
  // (what has no page is read from the first)
  auto place = [&](int32_t entry, int32_t at) {
    return (c.is_page(entry) ? int64_t(entry) * c.page_elems : 0) + (at & (c.page - 1)) * D;
  };
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    const uint16_t *k = key + place(WHOLE ? e.quarter[0] : e.key[i], t + 16 * ld.quarter(i));
    st.k[i] = *reinterpret_cast<const u4 *>(k + ld.koff);
  }
  const uint16_t *v = value + place(WHOLE ? e.quarter[0] : e.value, t + 16 * ld.wave) + ld.voff;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (D == 128) {
      const u2 x = *reinterpret_cast<const u2 *>(v + j * D);
      st.v[j][0] = x[0];
      st.v[j][D / 64 - 1] = x[1];
    } else {
      st.v[j][0] = *reinterpret_cast<const uint32_t *>(v + j * D);
    }
  }
}

// The orders of a key's and of a channel's chunks in LDS.
template <int D>
__device__ __forceinline__ int key_swizzle(int key) {
  return ((key & 3) | ((key >> 3) & 3) << 2) & (D / 8 - 1);
}
template <int D>
__device__ __forceinline__ int value_swizzle(int channel) {
  return D == 128 ? ((channel >> 2) & 7) ^ ((channel & 3) << 1) : ((channel >> 1) & 7) ^ ((channel & 1) << 2);
}

template <int D>
__device__ __forceinline__ void store_keys(const Staged<D> &st, char *buf, const Loader<D> &ld) {
#pragma unroll
  for (int i = 0; i < Tile<D>::kLoads; ++i) {
    const int key = ld.key + i * (2048 / D);
    *reinterpret_cast<u4 *>(buf + key * Tile<D>::kKeyRow + 16 * (ld.chunk ^ key_swizzle<D>(key))) = st.k[i];
  }
}

// What lies behind the length is no value.
template <int D>
__device__ __forceinline__ void clear_values(Staged<D> &st, const Loader<D> &ld, int32_t length) {
  const bool there = ((st.absent >> ld.wave) & 1) == 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool held = there && st.t + 8 * ld.group + j < length;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) st.v[j][i] = held ? st.v[j][i] : 0u;
  }
}

template <int D>
__device__ __forceinline__ void store_values(const Staged<D> &st, char *buf, const Loader<D> &ld) {
#pragma unroll
  for (int c = 0; c < Tile<D>::kChannels; ++c) {
    const int channel = ld.channel + c;
    uint32_t w[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      w[p] = c % 2 ? halves_of<true>(st.v[2 * p][c / 2], st.v[2 * p + 1][c / 2])
                   : halves_of<false>(st.v[2 * p][c / 2], st.v[2 * p + 1][c / 2]);
    }
    *reinterpret_cast<u4 *>(buf + Tile<D>::kKeyBytes + channel * Tile<D>::kValueRow +
                               16 * (ld.group ^ value_swizzle<D>(channel))) = u4{w[0], w[1], w[2], w[3]};
  }
}

// Sixteen query rows of a wave: the lane's row is lane % 16, its channels 16 n + 4 (lane / 16) + i.
template <int D>
struct Acc16 {
  f4 o[D / 16];
  float m, l;
};

// The reference of 16 rows' weights, raised where one of the tile's logits asks for it.  seen[h]: keys of half h that the
// lane's row sees, from the lane's own first on.
template <int D, bool MASK>
__device__ __forceinline__ float reference(Acc16<D> &acc, f4 (&s)[4], float factor, const int32_t (&seen)[2]) {
  float top = mf::kNegInf;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if (MASK) s[j / 4][j % 4] = j % 8 >= seen[j / 8] ? mf::kNegInf : s[j / 4][j % 4];  // (its weight is 0 then)
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
  return acc.m == mf::kNegInf ? 0.0f : acc.m;
}

// The weights of half a tile, and the sum of all.
template <int DT>
__device__ __forceinline__ float weights(const f4 (&s)[4], int half, float factor, float m, float l,
                                         typename Half<DT>::V8 &p) {
  typedef typename Half<DT>::T T;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float e = mf::fast_exp2(__builtin_fmaf(s[2 * half + j / 4][j % 4], factor, -m));
    l += e;
    p[j] = static_cast<T>(e);
  }
  return l;
}

// Products of N fragments read from LDS, with the reads kAhead fragments ahead of their use, in just this order.  (Left to itself
// the compiler, short of registers, reads each one right before its use and waits for it: 2 x 2k of 13k 803 us, 755 so; two more
// ahead 760.)
template <int N, class Load, class Use>
__device__ __forceinline__ void products(Load load, Use use) {
  constexpr int kAhead = 4;
  decltype(load(0)) a[N];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) a[i] = load(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + kAhead < N) a[i + kAhead] = load(i + kAhead);
    __builtin_amdgcn_sched_barrier(0);
    use(i, a[i]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The tiles of all units, ordered by KV head, sequence and row group, are cut into runs of equal length for the
// workgroups: calls of any lengths and any number of units load them alike, and only a run's first and last
// unit may be parts, joined by a second launch.  (Causal rows see fewer keys the earlier they are, so units differ.)
// `flat` counts the row groups of all sequences.
__device__ __forceinline__ int32_t tiles_of(const Cache &c, const Query &q, const Plan &p, int32_t flat) {
  if (flat >= c.sequences * p.groups) return 0;
  const int32_t s = flat / p.groups;
  int32_t length, count;
  sizes_of(c, q, s, length, count);
  return (rows_at(q, s, 0, flat - s * p.groups, kTileRows, length, count).end_last + kKeys - 1) / kKeys;
}

// For a whole wave: tiles of a head, of its units before `flat`, and of that.
struct Sums {
  int32_t total, before, mine;

  __device__ __forceinline__ Sums(const Cache &c, const Query &q, const Plan &p, int32_t flat) : total(0), before(0), mine(0) {
    for (int32_t f0 = 0; f0 < c.sequences * p.groups; f0 += 64) {
      const int32_t n = tiles_of(c, q, p, f0 + (threadIdx.x & 63)), sum = wave_prefix(n);
      if (flat >= f0 && flat < f0 + 64) {
        mine = __builtin_amdgcn_readlane(n, flat - f0);
        before = total + __builtin_amdgcn_readlane(sum, flat - f0) - mine;
      }
      total += __builtin_amdgcn_readlane(sum, 63);
    }
  }
  __device__ __forceinline__ int32_t per(const Cache &c, const Plan &p) const {
    const int32_t n = (total * c.heads + p.workgroups - 1) / p.workgroups;
    return n > 0 ? n : 1;
  }
};

// Where a workgroup leaves a part: that of its first unit, or that of its last.
__device__ __forceinline__ int32_t slot_of(int32_t run, bool first) { return 2 * run + (first ? 0 : 1); }

// A workgroup's way through its run.
struct Walk {
  int32_t h, flat, tiles;       // the unit, and its tiles
  int32_t begin, end;           // those of them that are the workgroup's
  int32_t left;                 // tiles of the run from `begin` on
  bool first;

  __device__ __forceinline__ Walk(const Cache &c, const Query &q, const Plan &p, int32_t run) : begin(0), first(true) {
    if (p.workgroups == 0) {  // a unit
      const int32_t flats = c.sequences * p.groups;
      h = run / flats;
      flat = run - h * flats;
      tiles = end = left = __builtin_amdgcn_readfirstlane(tiles_of(c, q, p, flat));
      if (left == 0) left = 1;  // (rows without keys are finished too)
      return;
    }
    const Sums sums(c, q, p, 0);
    const int32_t per = sums.per(c, p), all = sums.total * c.heads, at = run * per;
    left = at + per < all ? per : all - at;
    if (left <= 0) return;
    h = at / sums.total;
    int32_t rest = at - h * sums.total;
    for (flat = 0;; flat += 64) {
      const int32_t n = tiles_of(c, q, p, flat + (threadIdx.x & 63)), sum = wave_prefix(n);
      const uint64_t past = __ballot(sum > rest);
      if (past != 0) {
        const int32_t i = __builtin_ctzll(past);
        tiles = __builtin_amdgcn_readlane(n, i);
        begin = rest - (__builtin_amdgcn_readlane(sum, i) - tiles);
        flat += i;
        break;
      }
      rest -= __builtin_amdgcn_readlane(sum, 63);
    }
    end = tiles - begin < left ? tiles : begin + left;
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next(const Cache &c, const Query &q, const Plan &p) {
    left -= p.workgroups == 0 ? left : end - begin;
    if (left <= 0) return;
    do {
      if (++flat == c.sequences * p.groups) {
        flat = 0;
        ++h;
      }
      tiles = __builtin_amdgcn_readfirstlane(tiles_of(c, q, p, flat));
    } while (tiles == 0);  // (there are `left` more)
    begin = 0;
    end = tiles < left ? tiles : left;
    first = false;
  }
  __device__ __forceinline__ Rows rows(const Cache &c, const Query &q, const Plan &p) const {
    const int32_t s = flat / p.groups;
    int32_t length, count;
    sizes_of(c, q, s, length, count);
    return rows_at(q, s, h, flat - s * p.groups, kTileRows, length, count);
  }
  __device__ __forceinline__ bool part() const { return end - begin != tiles; }
  __device__ __forceinline__ int32_t slot(int32_t run) const { return slot_of(run, first); }
};

template <int D, int DT, bool WHOLE>
__global__ __launch_bounds__(256, 2) void tile_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse, float *part,
                                                      float *stat) {
  typedef Tile<D> T;
  typedef Half<DT> H;
  typedef typename H::V8 V8;
  __shared__ __attribute__((aligned(16))) char lds[2 * T::kBytes];
  __shared__ uint32_t bad;  // whether a second pass over the unit's tiles is asked for
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quad = lane >> 4;
  // Two waves share a SIMD, in slots that differ in their last bit (HW_ID's first four bits).
  // One goes before the other in its vector phases, so that they do not reach the matrix cores together.
  const bool before = (__builtin_amdgcn_s_getreg((3 << 11) | 4) & 1) != 0;
  auto vector_phase = [&] {
    if (before) {
      __builtin_amdgcn_s_setprio(1);
    } else {
      __builtin_amdgcn_s_setprio(0);
    }
  };
  // Workgroups go to the 8 XCDs in turn; an XCD takes runs that follow each other, so that its L2 holds the keys of few heads.
  const int32_t run = p.workgroups == 0 ? blockIdx.x : (blockIdx.x & 7) * (p.workgroups / 8) + (blockIdx.x >> 3);
  Walk walk(c, q, p, run);
  const Loader<D> ld;
  const int krow = (col >> 2) * 8 + (col & 3);
  bool search = false;
  while (walk.more()) {
  const Rows w = walk.rows(c, q, p);
  const int32_t begin = walk.begin, end = walk.end;
  Pages pages(c, w.s);
  const int64_t head = int64_t(w.h << c.shift) * D;
  const uint16_t *keys = c.key + head, *values = c.value + head;

  V8 frag[2][D / 32];
  int32_t row_end[2];
  Acc16<D> acc[2];
  Infinite infinite[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    infinite[n] = Infinite{0, 0};
    const int32_t r = w.r0 + wave * 32 + n * 16 + col;
    const bool there = r < w.rows;
    // (rows past the last are the first's again, and nobody's)
    const int32_t at = there ? r : w.r0, token = token_of(q, at);
    row_end[n] = there ? visible(q, w.length, w.count, token) : 0;
    const uint16_t *row = q.p + w.s * q.ss + token * q.st + (w.h * q.group + at - token * q.group) * q.sh + quad * 8;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) frag[n][k] = *reinterpret_cast<const V8 *>(row + k * 32);
    acc[n].m = mf::kNegInf;
    acc[n].l = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[n].o[d] = f4{0, 0, 0, 0};
  }
  // LDS offsets of the fragments: key tile j adds (32 (j / 2) + 4 (j % 2)) rows, channel tile n 16 rows
  int ka[D / 32], va[2];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) ka[k] = krow * T::kKeyRow + 16 * ((4 * k + quad) ^ key_swizzle<D>(krow));
#pragma unroll
  for (int h = 0; h < 2; ++h) va[h] = T::kKeyBytes + col * T::kValueRow + 16 * ((4 * h + quad) ^ value_swizzle<D>(col));

  Staged<D> st;
  Entries<D, WHOLE> entries;  // of the tile after the staged one
  // whether every row sees all keys of the staged tile
  auto whole = [&] {
    return st.t + kKeys <= w.end_first && st.absent == 0;
  };
  int32_t t = begin;
  int present = 0;  // the tile's buffer
  auto step = [&](auto mask_tag) {
    constexpr bool MASK = decltype(mask_tag)::value;
    const char *buf = lds + present * T::kBytes;
    const int32_t t0 = st.t;
    auto value = [&](int h, int d) {
      // (at 128 channels the chunks' order of channels 16 on is the first's with 4 changed)
      return *reinterpret_cast<const V8 *>(buf + ((D == 128 ? h ^ (d & 1) : h) ? va[1] : va[0]) + d * 16 * T::kValueRow);
    };
    const uint32_t absent = st.absent;
    const bool more = t + 1 < end;
    if (more) fetch<D, WHOLE>(st, c, entries, keys, values, ld, (t + 1) * kKeys);

    __builtin_amdgcn_s_setprio(3);
    f4 s[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[0][j] = s[1][j] = f4{0, 0, 0, 0};
    products<D / 8>(
        [&](int i) {
          const int j = i / (D / 32), k = i % (D / 32);
          return *reinterpret_cast<const V8 *>(buf + ka[k] + (32 * (j / 2) + 4 * (j % 2)) * T::kKeyRow);
        },
        [&](int i, V8 a) {
          const int j = i / (D / 32), k = i % (D / 32);
          s[0][j] = H::mfma(a, frag[0][k], s[0][j]);
          s[1][j] = H::mfma(a, frag[1][k], s[1][j]);
        });
    vector_phase();
    // (asked for here: LDS reads and scalar loads are waited for together, and none of the former follows for a while)
    __builtin_amdgcn_sched_barrier(0);
    ask(entries, pages, ld, (t + 2) * kKeys);
    __builtin_amdgcn_sched_barrier(0);
    V8 pr[2][2];
    float m[2], factor[2] = {q.scale, q.scale};
    int32_t seen[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        seen[n][h] = row_end[n] - t0 - 32 * h - 8 * quad;
        if (MASK && ((absent >> (2 * h + (quad >> 1))) & 1) != 0) seen[n][h] = 0;
      }
      m[n] = reference<D, MASK>(acc[n], s[n], q.scale, seen[n]);
      if (MASK && __builtin_expect(search, false)) round_far(s[n], factor[n], m[n]);
    }
    auto weigh = [&](int h) {
#pragma unroll
      for (int n = 0; n < 2; ++n) acc[n].l = weights<DT>(s[n], h, factor[n], m[n], acc[n].l, pr[n][h]);
    };
    weigh(0);
    weigh(1);
    present ^= 1;
    // (some rows see less than there is; those of one causal token, 128 query heads or more of a KV head, all do)
    if (MASK && (search || w.end_first < w.length)) {
      u4 *held = reinterpret_cast<u4 *>(lds + (present ^ 1) * T::kBytes + T::kKeyBytes);
      uint32_t bad = 0;
      for (int i = lane; i < T::kValueBytes / 16; i += 64) {
        const u4 v = held[i];
        bad |= infinite_bits<DT>(v[0]) | infinite_bits<DT>(v[1]) | infinite_bits<DT>(v[2]) | infinite_bits<DT>(v[3]);
      }
      if (__builtin_expect(__any(bad != 0), false)) {  // (the same in every wave)
#pragma unroll 1
        for (int i = 0; i < D / 8; ++i) {
          const int d = i >> 1, h = i & 1;
          const V8 v = value(h, d);
          note_infinite<DT>(v, h ? seen[0][1] : seen[0][0], d, infinite[0]);
          note_infinite<DT>(v, h ? seen[1][1] : seen[1][0], d, infinite[1]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < T::kValueBytes / 16; i += 256) {
          u4 v = held[i];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = finite_half<DT>(v[k]);
          held[i] = v;
        }
        __syncthreads();
      }
    }
    if (more && !whole()) clear_values<D>(st, ld, w.length);
    __builtin_amdgcn_s_setprio(3);
    products<D / 8>([&](int i) { return value(i / (D / 16), i % (D / 16)); },
                    [&](int i, V8 a) {
                      const int h = i / (D / 16), d = i % (D / 16);
                      acc[0].o[d] = H::mfma(a, pr[0][h], acc[0].o[d]);
                      acc[1].o[d] = H::mfma(a, pr[1][h], acc[1].o[d]);
                    });
    // (after the last tile the present one's again, into the buffer that nobody reads)
    store_keys<D>(st, lds + present * T::kBytes, ld);
    store_values<D>(st, lds + present * T::kBytes, ld);
    vector_phase();
    __syncthreads();
    ++t;
  };
  st.t = 0;
  st.absent = 0;
  if (begin < end) {
    ask(entries, pages, ld, begin * kKeys);
    fetch<D, WHOLE>(st, c, entries, keys, values, ld, begin * kKeys);
    if (!whole()) clear_values<D>(st, ld, w.length);
    ask(entries, pages, ld, (begin + 1) * kKeys);
    store_keys<D>(st, lds, ld);
    store_values<D>(st, lds, ld);
  }
  // (The queries are here now: else the first products of every tile would wait for whatever was asked for last, which
  // is the next tile: 2 x 2k of 13k 755 us, 733 so; 4 x 1k of 4k at 64 channels 64.5, 61.0 so.)
#pragma unroll
  for (int n = 0; n < 2; ++n) {
#pragma unroll
    for (int k = 0; k < D / 32; ++k) asm volatile("" : "+v"(frag[n][k]));
  }
  __syncthreads();
  if (threadIdx.x == 0) bad = 0;  // (the last unit's has been read; a barrier a tile lies before this one's is written)
  // tiles that every row sees come first; from the first other one on, every tile is masked
  while (!search && t < end && whole()) step(std::false_type());
  while (t < end) step(std::true_type());

#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int32_t rr = wave * 32 + n * 16 + col, r = w.r0 + rr;
    const float total = mf::sum_over_slices(acc[n].l);
    add_infinite(acc[n].o, infinite[n]);
    if (r >= w.rows) continue;
    if (total == 0.0f && acc[n].m == mf::kNegInf) {
      acc[n].m = no_reference(c, w.s, begin * kKeys, row_end[n] < end * kKeys ? row_end[n] : end * kKeys);
    }
    if (row_end[n] > 0 && (is_far(acc[n].m) || spoiled<D / 4>([&](int j) { return acc[n].o[j / 4][j % 4]; }, total))) bad = 1;
    if (walk.part()) {
      const int64_t slot = int64_t(walk.slot(run)) * kTileRows + rr;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f4 *>(part + slot * D + 16 * d + 4 * quad) = acc[n].o[d];
      if (quad == 0) {
        stat[2 * slot] = acc[n].m;
        stat[2 * slot + 1] = total;
      }
    } else {
      const int32_t token = token_of(q, r), h = w.h * q.group + r - token * q.group;
      const bool none = token >= w.count || (total == 0.0f && acc[n].m == mf::kNegInf);
      const float f = none ? 0.0f : 1.0f / total;
      uint16_t *dst = out + ((int64_t(w.s) * q.len + token) * q.heads + h) * D + 4 * quad;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const f4 y = none ? f4{0, 0, 0, 0} : acc[n].o[d] * f;
        *reinterpret_cast<uint2 *>(dst + 16 * d) = uint2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
      }
      if (quad == 0 && lse != nullptr) {
        lse[(int64_t(w.s) * q.heads + h) * q.len + token] = none ? mf::kNegInf : lse_of(q, acc[n].m, total);
      }
    }
  }
  __syncthreads();
  search = __builtin_amdgcn_readfirstlane(bad) != 0 && !search;
  if (!search) walk.next(c, q, p);
  }
}

// Units in parts are joined, and those without keys finished: a workgroup takes 16 rows of a unit, 16 lanes each.
template <int D, int DT>
__global__ __launch_bounds__(256) void tile_join_kernel(Cache c, Query q, Plan p, uint16_t *out, float *lse,
                                                        const float *part, const float *stat) {
  constexpr int kC = D / 16, kAhead = 4;  // parts on their way
  const int32_t unit = blockIdx.x, flats = c.sequences * p.groups, h = unit / flats, flat = unit - h * flats;
  const Sums sums(c, q, p, flat);
  const int32_t per = sums.per(c, p), start = h * sums.total + sums.before, stop = start + sums.mine;
  const int32_t w0 = start / per, w1 = sums.mine == 0 ? w0 - 1 : (stop - 1) / per;
  if (w1 == w0) return;
  const int32_t s = flat / p.groups, lane = threadIdx.x & 15, rr = blockIdx.y * 16 + (threadIdx.x >> 4);
  const Rows w = rows_at(q, s, h, flat - s * p.groups, kTileRows, c.length(s), q.count(s));
  if (w.r0 + rr >= w.rows) return;
  auto slot = [&](int32_t i) { return int64_t(slot_of(i, i > w0 || start == w0 * per)) * kTileRows + rr; };
  float m = mf::kNegInf, l = 0.0f, o[kC];
#pragma unroll
  for (int j = 0; j < kC; ++j) o[j] = 0.0f;
  for (int32_t i = w0 + lane; i <= w1; i += 16) m = fmaxf(m, stat[2 * slot(i)]);
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, kWave));
  for (int32_t i0 = w0; i0 <= w1; i0 += kAhead) {
    float mi[kAhead], li[kAhead];
    f4 x[kAhead][kC / 4];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t at = slot(i0 + u <= w1 ? i0 + u : w1);
      mi[u] = stat[2 * at];
      li[u] = stat[2 * at + 1];
#pragma unroll
      for (int j = 0; j < kC / 4; ++j) x[u][j] = *reinterpret_cast<const f4 *>(part + at * D + lane * kC + 4 * j);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u > w1 || (mi[u] == mf::kNegInf && li[u] == 0.0f)) continue;
      const float f = mf::fast_exp2(mi[u] - m);
      l += li[u] * f;
#pragma unroll
      for (int j = 0; j < kC; ++j) o[j] += joining(f, x[u][j / 4][j % 4]);
    }
  }
  store_row<D, DT>(q, w, w.r0 + rr, lane * kC, o, m, l, out, lse);
}

}  // namespace

int launch_tiles(const char *what, int dtype, int64_t head_dim, const Cache &c, const Query &q, const Plan &p, uint16_t *out,
                 float *lse, float *part, float *stat, hipStream_t stream) {
  const int32_t units = c.sequences * c.heads * p.groups;
  const dim3 grid(static_cast<uint32_t>(p.workgroups > 0 ? p.workgroups : units));
  auto go = [&](auto kernel, dim3 workgroups) {
    hipLaunchKernelGGL(kernel, workgroups, dim3(256), 0, stream, c, q, p, out, lse, part, stat);
    return check_launch(what);
  };
  auto run = [&](auto d_tag, auto dt_tag) {
    constexpr int D = decltype(d_tag)::value, DT = decltype(dt_tag)::value;
    const int rc = c.page >= kKeys ? go(tile_kernel<D, DT, true>, grid) : go(tile_kernel<D, DT, false>, grid);
    return rc != UC_OK || p.workgroups == 0 ? rc : go(tile_join_kernel<D, DT>, dim3(units, kTileRows / 16));
  };
  auto by_type = [&](auto d_tag) {
    return dtype == UC_FP16 ? run(d_tag, std::integral_constant<int, UC_FP16>()) : run(d_tag, std::integral_constant<int, UC_BF16>());
  };
  return head_dim == 128 ? by_type(std::integral_constant<int, 128>()) : by_type(std::integral_constant<int, 64>());
}

}  // namespace pg
}  // namespace uc
