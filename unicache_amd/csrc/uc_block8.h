// Geometry and code conversion of the 8-bit block-scaled KV cache, shared by
// its kernels (uc_block8.hip, uc_block8_attn.hip, uc_block8_select.hip).
#pragma once
#include "uc_common.h"
#include "uc_mfma.h"

namespace uc {
namespace b8 {

using mf::f4;
using mf::h2;
using mf::h8;

constexpr float kTiny = 0x1p-60f;  // the smallest scale of a block

// Largest magnitude of a code's value.
template <int CODE>
constexpr float kLimit = CODE == UC_INT8 ? 127.0f : 448.0f;

// The cache as the kernels take it (by value).
struct Cache {
  uint8_t *key_code, *value_code;
  float *key_scale, *value_scale;
  int8_t *bounds;
  const int32_t *lengths;
  int32_t sequences, heads, blocks;  // blocks: capacity per sequence
  int32_t block, shift;              // tokens of a block, its log2

  // Tokens of sequence s; a length outside [0, capacity] reads as the nearer end.
  __device__ __forceinline__ int32_t length(int32_t s) const {
    const int32_t n = lengths[s], most = blocks << shift;
    return n < 0 ? 0 : n > most ? most : n;
  }
};

// Checks a uc_block8_cache and fills `out`; UC_OK or UC_EINVAL with the error set.
int check_cache(const uc_block8_cache *c, const char *what, Cache &out);

// Four codes of one dword as fp16 (both formats are exact in fp16).
template <int CODE>
__device__ __forceinline__ void codes_to_h4(uint32_t w, h2 &a, h2 &b) {
  if constexpr (CODE == UC_INT8) {
    // code + 128 in the mantissa of 1024, then 1152 is subtracted exactly
    const uint32_t u = w ^ 0x80808080u;
    const h2 base{mf::to_h(1152.0f), mf::to_h(1152.0f)};
    a = mf::as_h2(__builtin_amdgcn_perm(u, 0x64646464u, 0x00050004u)) - base;
    b = mf::as_h2(__builtin_amdgcn_perm(u, 0x64646464u, 0x00070006u)) - base;
  } else {
    a = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    b = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  }
}

// Eight codes (two dwords) as an MFMA operand fragment.
template <int CODE>
__device__ __forceinline__ h8 codes_to_h8(uint32_t w0, uint32_t w1) {
  h2 a, b, c, d;
  codes_to_h4<CODE>(w0, a, b);
  codes_to_h4<CODE>(w1, c, d);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four codes of one dword as fp32.
template <int CODE>
__device__ __forceinline__ void codes_to_f4(uint32_t w, float *out) {
  h2 a, b;
  codes_to_h4<CODE>(w, a, b);
  out[0] = static_cast<float>(a[0]);
  out[1] = static_cast<float>(a[1]);
  out[2] = static_cast<float>(b[0]);
  out[3] = static_cast<float>(b[1]);
}

#define UC_B8_DISPATCH(cache, head_dim, ...)                                             \
  [&] {                                                                                  \
    if ((cache)->code_dtype == UC_INT8) {                                                \
      constexpr int CODE = UC_INT8;                                                      \
      if ((head_dim) == 128) { constexpr int D = 128; return __VA_ARGS__(); }            \
      else { constexpr int D = 64; return __VA_ARGS__(); }                               \
    } else {                                                                             \
      constexpr int CODE = UC_E4M3;                                                      \
      if ((head_dim) == 128) { constexpr int D = 128; return __VA_ARGS__(); }            \
      else { constexpr int D = 64; return __VA_ARGS__(); }                               \
    }                                                                                    \
  }()

}  // namespace b8
}  // namespace uc
