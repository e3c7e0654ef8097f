// Attention over a paged cache of 4-bit codes: its operands, and what a query
// sees.
#pragma once

#include "kk_attention.h"

namespace kk {

__device__ __forceinline__ float low_half(uint32_t w) { return __half2float(__ushort_as_half(static_cast<unsigned short>(w))); }
__device__ __forceinline__ float high_half(uint32_t w) { return low_half(w >> 16); }

struct Paged4Rows : PagedRows {
  const uint8_t *k, *v;               // of `a`: table, lengths, counts and window
  const uint32_t *k_scale, *v_scale;  // a token's step and lowest value, fp16 each
  __device__ static float value_of(uint32_t byte, bool high, uint32_t scale) {
    return __builtin_fmaf(static_cast<float>(high ? byte >> 4 : byte & 15u), low_half(scale), high_half(scale));
  }
  __device__ float key(int64_t b, int h, int64_t j, int d) const {
    const int half = D / 2;
    const int64_t at = (page(b, j) * a.heads + h) * a.block + j % a.block;
    return value_of(k[at * half + d % half], d >= half, k_scale[at]);
  }
  __device__ float value(int64_t b, int h, int64_t j, int d) const {
    const int half = D / 2;
    const int64_t head = page(b, j) * a.heads + h, row = j % a.block;
    return value_of(v[(head * half + d % half) * a.block + row], d >= half, v_scale[head * a.block + row]);
  }
};

// Entry points of the kernels; false where a call is not theirs.
bool few_paged4_try(const QueryArgs& a, const Paged4Rows& rows, int dtype, int* status);

}  // namespace kk
