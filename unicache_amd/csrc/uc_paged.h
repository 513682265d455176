// The paged KV cache as its kernels take it (uc_paged.hip, uc_paged_attn.hip, uc_rotary.hip).
#pragma once
#include "uc_common.h"

namespace uc {
namespace pg {

constexpr int64_t kMostSequences = 4096;  // (a number for each stands in the LDS of the workgroup that hands out pages)

struct Cache {
  uint16_t *key, *value;  // [P, Hkv, B, D] of one layer
  int32_t *table, *lengths;
  int64_t layer_elems;    // P Hkv B D
  int32_t sequences, width, pages, heads;
  int32_t page, shift;    // tokens of a page, their log2
  int32_t page_elems;     // Hkv B D, below 2^31

  __host__ __device__ __forceinline__ int32_t capacity() const { return width << shift; }

  // Tokens of sequence s; a length outside [0, capacity] reads as the nearer end.
  __device__ __forceinline__ int32_t length(int32_t s) const { return clamped(lengths[s]); }
  __device__ __forceinline__ int32_t clamped(int32_t n) const {
    const int32_t most = capacity();
    return n < 0 ? 0 : n > most ? most : n;
  }
  // Pages that n tokens take.
  __device__ __forceinline__ int32_t pages_of(int32_t n) const { return (n + page - 1) >> shift; }
  __device__ __forceinline__ bool is_page(int32_t p) const { return static_cast<uint32_t>(p) < static_cast<uint32_t>(pages); }
};

// Checks a uc_paged_cache and fills `out` for one layer; UC_OK or UC_EINVAL with the error set.
int check_cache(const uc_paged_cache *c, int64_t layer, const char *what, Cache &out);

}  // namespace pg
}  // namespace uc
