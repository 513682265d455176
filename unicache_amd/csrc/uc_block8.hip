// The 8-bit block-scaled KV cache: quantizing dense rows into blocks (pack,
// append) and restoring them.
//
// A block is B tokens of one KV head.  With a = max(max|x|, 2^-60 L), L the
// largest code (127 or 448), scale = a (1/L) and code = round(x (L/a)); the
// key's bounds are the per-channel extremes of its codes in steps of a/127,
// rounded outwards.  All of it is one pass over the rows: HBM-bound byte work,
// 2 + 1 bytes per element.  Measured: 55,707 tokens of 8 heads (4 ragged sequences of up to
// 16k, 228 MB of rows) 92 us packing, 66 us restoring into 268 MB; 4.6 - 5.0 TB/s both together, a
// large copy 4.9.
//
// One workgroup owns one block.  A thread takes four consecutive tokens of
// eight channels (four 16-byte loads each of keys and values, whole 256-byte
// rows per 16 lanes at D = 128), so the values' token-minor codes
// [D][B] are 4x4 byte transposes in registers and dword writes to LDS, from
// which they leave in 16-byte stores.
#include "uc_block8.h"

#include <algorithm>

namespace uc {
namespace b8 {

int check_cache(const uc_block8_cache *c, const char *what, Cache &out) {
  UC_REQUIRE(c != nullptr, "%s: cache is NULL", what);
  UC_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim must be 64 or 128", what);
  UC_REQUIRE(c->block_tokens == 32 || c->block_tokens == 64 || c->block_tokens == 128,
             "%s: block_tokens must be 32, 64 or 128", what);
  UC_REQUIRE(c->code_dtype == UC_INT8 || c->code_dtype == UC_E4M3, "%s: codes must be int8 or e4m3", what);
  UC_REQUIRE(c->sequences > 0 && c->heads_kv > 0 && c->blocks > 0, "%s: empty cache", what);
  // token indexes are int32; scales and blocks are addressed in 64 bits
  UC_REQUIRE(c->sequences < (1 << 24) && c->heads_kv < (1 << 16) && c->blocks <= ((1u << 31) - 1) / c->block_tokens / 2,
             "%s: cache too large", what);
  UC_REQUIRE(c->sequences * c->heads_kv <= (1 << 24), "%s: too many sequences x heads", what);
  UC_REQUIRE(c->key_code && c->value_code && c->key_scale && c->value_scale && c->key_bounds && c->lengths,
             "%s: the cache has a NULL tensor", what);
  UC_REQUIRE(((reinterpret_cast<uintptr_t>(c->key_code) | reinterpret_cast<uintptr_t>(c->value_code) |
               reinterpret_cast<uintptr_t>(c->key_bounds)) & 15) == 0 &&
                 ((reinterpret_cast<uintptr_t>(c->key_scale) | reinterpret_cast<uintptr_t>(c->value_scale) |
                   reinterpret_cast<uintptr_t>(c->lengths)) & 3) == 0,
             "%s: codes and bounds must be 16-byte aligned, scales and lengths 4-byte", what);
  out.key_code = static_cast<uint8_t *>(c->key_code);
  out.value_code = static_cast<uint8_t *>(c->value_code);
  out.key_scale = c->key_scale;
  out.value_scale = c->value_scale;
  out.bounds = c->key_bounds;
  out.lengths = c->lengths;
  out.sequences = static_cast<int32_t>(c->sequences);
  out.heads = static_cast<int32_t>(c->heads_kv);
  out.blocks = static_cast<int32_t>(c->blocks);
  out.block = c->block_tokens;
  out.shift = c->block_tokens == 32 ? 5 : c->block_tokens == 64 ? 6 : 7;
  return UC_OK;
}

namespace {

typedef unsigned short us2 __attribute__((ext_vector_type(2)));

// Work of a thread: units of four tokens x eight channels.
template <int D, int B>
struct Shape {
  static constexpr int kChunks = D / 8;
  static constexpr int kUnits = B / 4 * kChunks;
  static constexpr int kThreads = kUnits < 256 ? kUnits : 256;
  static constexpr int kPer = kUnits / kThreads;
  static constexpr int kPitch = B + 4;  // bytes of a channel's row in LDS: an odd number of dwords
  static constexpr int kWaves = kThreads / kWave;
};

template <int D, int B>
struct Shared {
  uint8_t codes[D * Shape<D, B>::kPitch];
  uint32_t amax[2][4];
  float hi[4][D], lo[4][D];
};

__device__ __forceinline__ uint32_t max_u16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}

// Largest magnitude (16-bit pattern; a NaN is above infinity) of four rows.
__device__ __forceinline__ uint32_t abs_max(const uint4 (&x)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m = max_u16(m, max_u16(max_u16(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                           max_u16(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
  }
  m = max_u16(m, m >> 16);
  return m & 0xffffu;
}

// Eight 16-bit values times `inv`, as codes (two dwords) and, for the bounds, as values.
template <int CODE, int IN, bool VALUES>
__device__ __forceinline__ uint2 quantize8(uint4 raw, float inv, float *val) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t out[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = w[2 * j + i / 2];
      y[i] = mul_rn(half_bits_to_f32<IN>(i % 2 ? bits >> 16 : bits), inv);
      y[i] = __builtin_amdgcn_fmed3f(y[i], -kLimit<CODE>, kLimit<CODE>);
    }
    if constexpr (CODE == UC_INT8) {
      uint32_t p = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = rintf(y[i]);
        p |= (static_cast<uint32_t>(static_cast<int>(y[i])) & 0xffu) << (8 * i);
      }
      out[j] = p;
    } else {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
      out[j] = static_cast<uint32_t>(p);
      if constexpr (VALUES) codes_to_f4<CODE>(out[j], y);
    }
    if constexpr (VALUES) {
#pragma unroll
      for (int i = 0; i < 4; ++i) val[4 * j + i] = y[i];
    }
  }
  return uint2{out[0], out[1]};
}

// The byte transpose of four rows of four codes.
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&out)[4]) {
  const uint32_t t0 = __builtin_amdgcn_perm(b, a, 0x05010400u), t1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t u0 = __builtin_amdgcn_perm(d, c, 0x05010400u), u1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  out[0] = __builtin_amdgcn_perm(u0, t0, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(u0, t0, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(u1, t1, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(u1, t1, 0x07060302u);
}

// A bound in steps of a/127: int8 codes are such steps; an e4m3 code c is
// 127 c / 448 of them.  c is a multiple of 2^-9, so a quotient that is no whole
// number is farther than 2^-18 from one, more than half an ulp below 128: the
// rounded division has the floor and ceiling of the exact one.
template <int CODE>
__device__ __forceinline__ int32_t bound(float v, bool high) {
  if constexpr (CODE == UC_INT8) return static_cast<int32_t>(v);
  const float q = div_rn(mul_rn(v, 127.0f), 448.0f);
  return static_cast<int32_t>(high ? ceilf(q) : floorf(q));
}

// Quantize one block by a whole workgroup: x[u] / y[u] are the thread's rows
// of keys and values (zero where a row does not count), `rows` of the block
// count.
template <int D, int B, int CODE, int IN>
__device__ void quantize_block(const uint4 (&x)[Shape<D, B>::kPer][4], const uint4 (&y)[Shape<D, B>::kPer][4], int rows,
                               const Cache &cache, int64_t block_index, Shared<D, B> &sh) {
  typedef Shape<D, B> S;
  constexpr float kL = kLimit<CODE>;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int u = 0; u < S::kPer; ++u) {
    mk = max(mk, abs_max(x[u]));
    mv = max(mv, abs_max(y[u]));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mk = max(mk, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mk), o, kWave)));
    mv = max(mv, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mv), o, kWave)));
  }
  __syncthreads();  // the previous block's reads of `sh` are over
  if (lane == 0) {
    sh.amax[0][wave] = mk;
    sh.amax[1][wave] = mv;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < S::kWaves; ++w) {
    mk = max(mk, sh.amax[0][w]);
    mv = max(mv, sh.amax[1][w]);
  }
  // a block holding an infinity or a NaN: that is its scale, its codes are 0
  const float fk = half_bits_to_f32<IN>(mk), fv = half_bits_to_f32<IN>(mv);
  const bool badk = !(fk < __builtin_huge_valf()), badv = !(fv < __builtin_huge_valf());
  const float ak = badk ? fk : fmaxf(fk, kL * kTiny), av = badv ? fv : fmaxf(fv, kL * kTiny);
  const float ik = badk ? 0.0f : div_rn(kL, ak), iv = badv ? 0.0f : div_rn(kL, av);

  float hi[8], lo[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hi[j] = -512.0f;
    lo[j] = 512.0f;
  }
#pragma unroll
  for (int u = 0; u < S::kPer; ++u) {
    const int unit = tid + u * S::kThreads, c = unit % S::kChunks, g = unit / S::kChunks;
    uint8_t *kout = cache.key_code + (block_index * B + 4 * g) * D + 8 * c;
    uint2 vc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float val[8];
      uint2 kc = quantize8<CODE, IN, true>(x[u][i], ik, val);
      vc[i] = quantize8<CODE, IN, false>(y[u][i], iv, nullptr);
      if (badk) kc = uint2{0, 0};
      if (badv) vc[i] = uint2{0, 0};
      *reinterpret_cast<uint2 *>(kout + i * D) = kc;
      const bool counts = 4 * g + i < rows;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        hi[j] = counts ? fmaxf(hi[j], badk ? 0.0f : val[j]) : hi[j];
        lo[j] = counts ? fminf(lo[j], badk ? 0.0f : val[j]) : lo[j];
      }
    }
    uint32_t t[4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == 0) {
        transpose4(vc[0].x, vc[1].x, vc[2].x, vc[3].x, t);
      } else {
        transpose4(vc[0].y, vc[1].y, vc[2].y, vc[3].y, t);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<uint32_t *>(sh.codes + (8 * c + 4 * half + j) * S::kPitch + 4 * g) = t[j];
      }
    }
  }
  // the bounds: over the wave's lanes of one chunk, then over the waves
#pragma unroll
  for (int o = 32; o >= S::kChunks; o >>= 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      hi[j] = fmaxf(hi[j], __shfl_xor(hi[j], o, kWave));
      lo[j] = fminf(lo[j], __shfl_xor(lo[j], o, kWave));
    }
  }
  if (lane < S::kChunks) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sh.hi[wave][8 * lane + j] = hi[j];
      sh.lo[wave][8 * lane + j] = lo[j];
    }
  }
  __syncthreads();
  for (int d = tid; d < D; d += S::kThreads) {
    float h = sh.hi[0][d], l = sh.lo[0][d];
#pragma unroll
    for (int w = 1; w < S::kWaves; ++w) {
      h = fmaxf(h, sh.hi[w][d]);
      l = fminf(l, sh.lo[w][d]);
    }
    int8_t *b = cache.bounds + block_index * 2 * D;
    b[d] = static_cast<int8_t>(rows > 0 ? bound<CODE>(h, true) : 0);
    b[D + d] = static_cast<int8_t>(rows > 0 ? bound<CODE>(l, false) : 0);
  }
  if (tid == 0) {
    cache.key_scale[block_index] = mul_rn(ak, 1.0f / kL);
    cache.value_scale[block_index] = mul_rn(av, 1.0f / kL);
  }
  uint8_t *vout = cache.value_code + block_index * B * D;
  for (int i = tid; i < D * B / 16; i += S::kThreads) {
    const int d = i / (B / 16), t = i % (B / 16) * 16;
    const uint32_t *src = reinterpret_cast<const uint32_t *>(sh.codes + d * S::kPitch + t);
    *reinterpret_cast<uint4 *>(vout + 16 * i) = uint4{src[0], src[1], src[2], src[3]};
  }
}

// Dense rows: element (s, t, h, d) at s*ss + t*st + h*sh + d (elements of 2 bytes).
struct Dense {
  const uint16_t *p;
  int64_t ss, st, sh;
  __device__ __forceinline__ const uint16_t *row(int64_t s, int64_t t, int64_t h) const {
    return p + s * ss + t * st + h * sh;
  }
};

// A workgroup per block of every (sequence, head): blocks along x, these pairs along y and, past the most
// that y holds, z.
constexpr int64_t kGridY = 65535;

dim3 block_grid(const Cache &c, int64_t blocks) {
  const int64_t pairs = int64_t(c.sequences) * c.heads, y = pairs < kGridY ? pairs : kGridY;
  return dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(y), static_cast<uint32_t>(ceil_div(pairs, y)));
}

__device__ __forceinline__ int32_t pair_of_grid() { return blockIdx.z * gridDim.y + blockIdx.y; }

template <int D, int B, int CODE, int IN>
__global__ __launch_bounds__((Shape<D, B>::kThreads)) void pack_kernel(Cache cache, Dense key, Dense value,
                                                                       int32_t tokens, const int32_t *row_counts,
                                                                       int32_t *lengths, uint16_t *tail) {
  typedef Shape<D, B> S;
  __shared__ Shared<D, B> sh;
  const int32_t b = blockIdx.x, pair = pair_of_grid(), sequence = pair / cache.heads, h = pair % cache.heads;
  if (sequence >= cache.sequences) return;
  int32_t length = row_counts != nullptr ? row_counts[sequence] : tokens;
  length = length < 0 ? 0 : length > tokens ? tokens : length;
  if (b == 0 && h == 0 && threadIdx.x == 0) lengths[sequence] = length;
  int rows = length - b * B;
  rows = rows < 0 ? 0 : rows > B ? B : rows;
  uint4 x[S::kPer][4], y[S::kPer][4];
#pragma unroll
  for (int u = 0; u < S::kPer; ++u) {
    const int unit = threadIdx.x + u * S::kThreads, c = unit % S::kChunks, g = unit / S::kChunks;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * g + i;
      x[u][i] = y[u][i] = uint4{0, 0, 0, 0};
      if (r < rows) {
        x[u][i] = *reinterpret_cast<const uint4 *>(key.row(sequence, int64_t(b) * B + r, h) + 8 * c);
        y[u][i] = *reinterpret_cast<const uint4 *>(value.row(sequence, int64_t(b) * B + r, h) + 8 * c);
      }
    }
  }
  quantize_block<D, B, CODE, IN>(x, y, rows, cache, int64_t(pair) * cache.blocks + b, sh);
  // the open block's rows, for append
  if (tail != nullptr && rows > 0 && rows < B) {
    uint16_t *t = tail + int64_t(pair) * 2 * B * D;
#pragma unroll
    for (int u = 0; u < S::kPer; ++u) {
      const int unit = threadIdx.x + u * S::kThreads, c = unit % S::kChunks, g = unit / S::kChunks;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * g + i;
        if (r < rows) {
          *reinterpret_cast<uint4 *>(t + r * D + 8 * c) = x[u][i];
          *reinterpret_cast<uint4 *>(t + (B + r) * D + 8 * c) = y[u][i];
        }
      }
    }
  }
}

// Rows that sequence s takes of an append call.
__device__ __forceinline__ int32_t appended(const Cache &cache, const int32_t *counts, int32_t s, int32_t tokens,
                                            int32_t length) {
  int32_t n = counts != nullptr ? counts[s] : tokens;
  n = n < 0 ? 0 : n > tokens ? tokens : n;
  const int32_t room = (cache.blocks << cache.shift) - length;
  return n < room ? n : room;
}

// One workgroup per (sequence, KV head) and block that the new rows may touch, `most` of them (one
// after the other, 4096 tokens of 8 heads took 210 us; so, 19).  The first block may hold rows of `tail`; its
// workgroup leaves the last block's rows there too, once it has read what was there: a
// thread reads and writes the same tail elements, so no barrier orders them.
template <int D, int B, int CODE, int IN>
__global__ __launch_bounds__((Shape<D, B>::kThreads)) void append_kernel(Cache cache, Dense key, Dense value,
                                                                         int32_t tokens, const int32_t *counts,
                                                                         uint16_t *tail, int32_t most) {
  typedef Shape<D, B> S;
  __shared__ Shared<D, B> sh;
  const int32_t unit = blockIdx.x / most, index = blockIdx.x % most;
  const int32_t sequence = unit / cache.heads, h = unit % cache.heads;
  const int32_t length = cache.length(sequence);
  const int32_t n = appended(cache, counts, sequence, tokens, length);
  const int32_t end = length + n, b = length / B + index;
  if (n <= 0 || b * B >= end) return;
  const int32_t last = (end - 1) / B;
  uint16_t *t = tail + int64_t(unit) * 2 * B * D;
  const int rows = end - b * B < B ? end - b * B : B;
  uint4 x[S::kPer][4], y[S::kPer][4];
#pragma unroll
  for (int u = 0; u < S::kPer; ++u) {
    const int at = threadIdx.x + u * S::kThreads, c = at % S::kChunks, g = at / S::kChunks;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * g + i;
      const int32_t token = b * B + r;
      x[u][i] = y[u][i] = uint4{0, 0, 0, 0};
      if (token < length) {
        x[u][i] = *reinterpret_cast<const uint4 *>(t + r * D + 8 * c);
        y[u][i] = *reinterpret_cast<const uint4 *>(t + (B + r) * D + 8 * c);
      } else if (token < end) {
        x[u][i] = *reinterpret_cast<const uint4 *>(key.row(sequence, token - length, h) + 8 * c);
        y[u][i] = *reinterpret_cast<const uint4 *>(value.row(sequence, token - length, h) + 8 * c);
      }
    }
  }
  // the rows of the block that stays open
  if (index == 0 && end % B != 0) {
#pragma unroll
    for (int u = 0; u < S::kPer; ++u) {
      const int at = threadIdx.x + u * S::kThreads, c = at % S::kChunks, g = at / S::kChunks;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * g + i;
        const int32_t token = last * B + r;
        if (token < length || token >= end) continue;
        uint4 kr = x[u][i], vr = y[u][i];
        if (last != b) {
          kr = *reinterpret_cast<const uint4 *>(key.row(sequence, token - length, h) + 8 * c);
          vr = *reinterpret_cast<const uint4 *>(value.row(sequence, token - length, h) + 8 * c);
        }
        *reinterpret_cast<uint4 *>(t + r * D + 8 * c) = kr;
        *reinterpret_cast<uint4 *>(t + (B + r) * D + 8 * c) = vr;
      }
    }
  }
  quantize_block<D, B, CODE, IN>(x, y, rows, cache, int64_t(unit) * cache.blocks + b, sh);
}

__global__ void advance_kernel(Cache cache, int32_t *lengths, int32_t tokens, const int32_t *counts) {
  const int32_t s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s >= cache.sequences) return;
  const int32_t length = cache.length(s);
  lengths[s] = length + appended(cache, counts, s, tokens, length);
}

// One workgroup restores one block of keys and values; the values' codes turn
// through LDS.
template <int D, int B, int CODE, int OUT>
__global__ __launch_bounds__((Shape<D, B>::kThreads)) void dequant_kernel(Cache cache, uint16_t *key, uint16_t *value,
                                                                          int32_t tokens) {
  typedef Shape<D, B> S;
  __shared__ uint8_t codes[D * S::kPitch];
  const int32_t b = blockIdx.x, pair = pair_of_grid(), sequence = pair / cache.heads, h = pair % cache.heads;
  if (sequence >= cache.sequences) return;
  const int64_t block_index = int64_t(pair) * cache.blocks + b;
  const int32_t length = cache.length(sequence);
  const bool any = b * B < length;
  const float ks = any ? cache.key_scale[block_index] : 0.0f, vs = any ? cache.value_scale[block_index] : 0.0f;
  if (any) {
    const uint8_t *vin = cache.value_code + block_index * B * D;
    for (int i = threadIdx.x; i < D * B / 16; i += S::kThreads) {
      const int d = i / (B / 16), t = i % (B / 16) * 16;
      const uint4 w = *reinterpret_cast<const uint4 *>(vin + 16 * i);
      uint32_t *dst = reinterpret_cast<uint32_t *>(codes + d * S::kPitch + t);
      dst[0] = w.x;
      dst[1] = w.y;
      dst[2] = w.z;
      dst[3] = w.w;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < S::kPer; ++u) {
    const int unit = threadIdx.x + u * S::kThreads, c = unit % S::kChunks, g = unit / S::kChunks;
    uint32_t vt[2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = any ? *reinterpret_cast<const uint32_t *>(codes + (8 * c + 4 * half + j) * S::kPitch + 4 * g) : 0;
      }
      transpose4(w[0], w[1], w[2], w[3], vt[half]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t t = b * B + 4 * g + i;
      if (t >= tokens) continue;
      const bool live = t < length;
      uint2 kc = uint2{0, 0};
      if (live) kc = *reinterpret_cast<const uint2 *>(cache.key_code + (block_index * B + 4 * g + i) * D + 8 * c);
      const uint2 vc = uint2{vt[0][i], vt[1][i]};
      uint32_t ko[4], vo[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float a[4], e[4];
        codes_to_f4<CODE>(j ? kc.y : kc.x, a);
        codes_to_f4<CODE>(j ? vc.y : vc.x, e);
        uint16_t ka[4], va[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          float kv = live ? mul_rn(a[m], ks) : 0.0f, vv = live ? mul_rn(e[m], vs) : 0.0f;
          // keeps product and cast apart: fused to one mixed-precision FMA they would round once
          if constexpr (OUT == UC_FP16) asm("" : "+v"(kv), "+v"(vv));
          ka[m] = OUT == UC_BF16 ? f32_to_bf16_bits(kv) : f32_to_f16_bits(kv);
          va[m] = OUT == UC_BF16 ? f32_to_bf16_bits(vv) : f32_to_f16_bits(vv);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          ko[2 * j + m] = ka[2 * m] | (uint32_t(ka[2 * m + 1]) << 16);
          vo[2 * j + m] = va[2 * m] | (uint32_t(va[2 * m + 1]) << 16);
        }
      }
      const int64_t at = ((int64_t(sequence) * tokens + t) * cache.heads + h) * D + 8 * c;
      *reinterpret_cast<uint4 *>(key + at) = uint4{ko[0], ko[1], ko[2], ko[3]};
      *reinterpret_cast<uint4 *>(value + at) = uint4{vo[0], vo[1], vo[2], vo[3]};
    }
  }
}

#define UC_B8_DISPATCH_BLOCK(cache, ...)                                         \
  [&] {                                                                          \
    switch ((cache)->block_tokens) {                                             \
      case 32: { constexpr int B = 32; return __VA_ARGS__(); }                   \
      case 64: { constexpr int B = 64; return __VA_ARGS__(); }                   \
      default: { constexpr int B = 128; return __VA_ARGS__(); }                  \
    }                                                                            \
  }()

#define UC_B8_DISPATCH_HALF(code, NAME, ...)                                     \
  [&] {                                                                          \
    if ((code) == UC_BF16) { constexpr int NAME = UC_BF16; return __VA_ARGS__(); } \
    else { constexpr int NAME = UC_FP16; return __VA_ARGS__(); }                 \
  }()

int check_dense(const char *what, const void *p, int64_t ss, int64_t st, int64_t sh, const char *name) {
  UC_REQUIRE(p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ((ss | st | sh) & 7) == 0,
             "%s: %s must be 16-byte aligned with strides that are multiples of 8", what, name);
  return UC_OK;
}

}  // namespace
}  // namespace b8
}  // namespace uc

extern "C" int uc_block8_pack(const uc_block8_cache *cache, const void *key, int64_t k_ss, int64_t k_st, int64_t k_sh,
                              const void *value, int64_t v_ss, int64_t v_st, int64_t v_sh, int in_dtype,
                              int64_t tokens, const int32_t *row_counts, void *tail, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::b8;
  Cache c;
  if (int rc = check_cache(cache, "uc_block8_pack", c)) return rc;
  UC_REQUIRE(half_dtype(in_dtype), "uc_block8_pack: keys and values must be bf16 or fp16");
  UC_REQUIRE(tokens >= 0 && tokens <= cache->blocks * cache->block_tokens, "uc_block8_pack: tokens exceed the capacity");
  if (tokens == 0) return UC_OK;
  if (int rc = check_dense("uc_block8_pack", key, k_ss, k_st, k_sh, "key")) return rc;
  if (int rc = check_dense("uc_block8_pack", value, v_ss, v_st, v_sh, "value")) return rc;
  UC_REQUIRE((reinterpret_cast<uintptr_t>(tail) & 15) == 0, "uc_block8_pack: tail must be 16-byte aligned");
  const Dense k{static_cast<const uint16_t *>(key), k_ss, k_st, k_sh};
  const Dense v{static_cast<const uint16_t *>(value), v_ss, v_st, v_sh};
  return UC_B8_DISPATCH(cache, cache->head_dim, [&] {
    return UC_B8_DISPATCH_BLOCK(cache, [&] {
      return UC_B8_DISPATCH_HALF(in_dtype, IN, [&] {
        const dim3 grid = block_grid(c, ceil_div(tokens, int64_t(B)));
        hipLaunchKernelGGL((pack_kernel<D, B, CODE, IN>), grid, dim3(Shape<D, B>::kThreads), 0, as_stream(stream), c, k,
                           v, static_cast<int32_t>(tokens), row_counts, cache->lengths, static_cast<uint16_t *>(tail));
        return check_launch("uc_block8_pack");
      });
    });
  });
}

extern "C" int uc_block8_append(const uc_block8_cache *cache, void *tail, const void *key, int64_t k_ss, int64_t k_st,
                                int64_t k_sh, const void *value, int64_t v_ss, int64_t v_st, int64_t v_sh,
                                int in_dtype, int64_t tokens, const int32_t *counts, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::b8;
  Cache c;
  if (int rc = check_cache(cache, "uc_block8_append", c)) return rc;
  UC_REQUIRE(half_dtype(in_dtype), "uc_block8_append: keys and values must be bf16 or fp16");
  UC_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 30), "uc_block8_append: bad number of tokens");
  UC_REQUIRE(tail != nullptr && (reinterpret_cast<uintptr_t>(tail) & 15) == 0,
             "uc_block8_append: tail must be given and 16-byte aligned");
  if (tokens == 0) return UC_OK;
  if (int rc = check_dense("uc_block8_append", key, k_ss, k_st, k_sh, "key")) return rc;
  if (int rc = check_dense("uc_block8_append", value, v_ss, v_st, v_sh, "value")) return rc;
  const Dense k{static_cast<const uint16_t *>(key), k_ss, k_st, k_sh};
  const Dense v{static_cast<const uint16_t *>(value), v_ss, v_st, v_sh};
  // blocks that the rows may touch
  const int64_t most = std::min<int64_t>(ceil_div(tokens - 1, int64_t(c.block)) + 1, c.blocks);
  UC_REQUIRE(int64_t(c.sequences) * c.heads * most < (1 << 24), "uc_block8_append: too many rows");
  const int rc = UC_B8_DISPATCH(cache, cache->head_dim, [&] {
    return UC_B8_DISPATCH_BLOCK(cache, [&] {
      return UC_B8_DISPATCH_HALF(in_dtype, IN, [&] {
        hipLaunchKernelGGL((append_kernel<D, B, CODE, IN>), dim3(static_cast<uint32_t>(c.sequences * c.heads * most)),
                           dim3(Shape<D, B>::kThreads), 0, as_stream(stream), c, k, v, static_cast<int32_t>(tokens),
                           counts, static_cast<uint16_t *>(tail), static_cast<int32_t>(most));
        return check_launch("uc_block8_append");
      });
    });
  });
  if (rc != UC_OK) return rc;
  // after every head has read the lengths
  hipLaunchKernelGGL(advance_kernel, dim3(static_cast<uint32_t>(ceil_div(c.sequences, 256))), dim3(256), 0,
                     as_stream(stream), c, cache->lengths, static_cast<int32_t>(tokens), counts);
  return check_launch("uc_block8_append");
}

extern "C" int uc_block8_dequant(const uc_block8_cache *cache, void *out_key, void *out_value, int out_dtype,
                                 int64_t tokens, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::b8;
  Cache c;
  if (int rc = check_cache(cache, "uc_block8_dequant", c)) return rc;
  UC_REQUIRE(half_dtype(out_dtype), "uc_block8_dequant: outputs must be bf16 or fp16");
  UC_REQUIRE(tokens >= 0 && tokens <= cache->blocks * cache->block_tokens,
             "uc_block8_dequant: tokens exceed the capacity");
  if (tokens == 0) return UC_OK;
  UC_REQUIRE(out_key && out_value &&
                 ((reinterpret_cast<uintptr_t>(out_key) | reinterpret_cast<uintptr_t>(out_value)) & 15) == 0,
             "uc_block8_dequant: outputs must be 16-byte aligned");
  return UC_B8_DISPATCH(cache, cache->head_dim, [&] {
    return UC_B8_DISPATCH_BLOCK(cache, [&] {
      return UC_B8_DISPATCH_HALF(out_dtype, OUT, [&] {
        const dim3 grid = block_grid(c, ceil_div(tokens, int64_t(B)));
        hipLaunchKernelGGL((dequant_kernel<D, B, CODE, OUT>), grid, dim3(Shape<D, B>::kThreads), 0, as_stream(stream),
                           c, static_cast<uint16_t *>(out_key), static_cast<uint16_t *>(out_value),
                           static_cast<int32_t>(tokens));
        return check_launch("uc_block8_dequant");
      });
    });
  });
}
