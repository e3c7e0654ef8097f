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

// Weights are kept beside 2^r, r a whole number near max (x + log2 step), but not
// below 2^-kLeast4 of the largest (a step is 0 or 2^-24 at the least); it follows
// where a product passes it by 2^kSlack4, or a weight by 2^kFar4.
constexpr float kLeast4 = 25.0f, kSlack4 = 7.0f, kFar4 = 32.0f;

// The value of lane J of each row of 16 lanes, in all of the row.
template <int J>
__device__ __forceinline__ float of_row(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + J, 0xF, 0xF, true));
}
// f(integral_constant<J>) for J = 0 .. N - 1.
template <int J, int N, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (J < N) {
    f(std::integral_constant<int, J>{});
    each<J + 1, N>(f);
  }
}

// What scores are multiplied by, |scale| 2^by: a normal number, since masked ones are
// -inf and 0 times them NaN.  (Below 2^-126, for queries of zeros or of subnormal values,
// it says nothing: scores are below 2^36 before it.)
__device__ __forceinline__ float unscaled4(float scale, int by) {
  return scale == 0.0f ? 1.0f : fmaxf(ldexpf(__builtin_fabsf(scale), by), 0x1p-126f);
}

// A key's step, NaN where it or the lowest value is not finite (a key with an
// infinite one is NaN in its codes of 0).
__device__ __forceinline__ float key_step(uint32_t scale) {
  const float step = low_half(scale), low = high_half(scale);
  return step + ((step - step) + (low - low));
}
// The low four bits of each byte of w, and the high ones, as halves code 2^-18
// (subnormal, code << 6), bytes 0, 2, 1, 3: two operations for two codes.  The
// matrix cores add up a subnormal's products to what its exponent would leave a normal
// number: further down in the half (a mask alone takes codes out where they lie) codes
// would lose up to ten bits of their sums, here one to four.
// CENTRE: less 8, for one operation more (sums of codes are then those of values
// around their middle, and fp32 keeps more of them).
struct Codes4 {
  uint32_t low[2], high[2];
};
template <bool CENTRE>
__device__ __forceinline__ Codes4 codes4(uint32_t w) {
  constexpr uint32_t kAt = 0x03c003c0u;
  Codes4 c{{w << 6 & kAt, w >> 2 & kAt}, {w << 2 & kAt, w >> 6 & kAt}};
  if constexpr (CENTRE) {
    const h2 middle = {static_cast<_Float16>(-0x1p-15f), static_cast<_Float16>(-0x1p-15f)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c.low[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, c.low[i]) + middle);
      c.high[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, c.high[i]) + middle);
    }
  }
  return c;
}
// What a token's values are beside: its lowest one, or step times 8 above it.
template <bool CENTRE>
__device__ __forceinline__ float base4(uint32_t scale) {
  return CENTRE ? __builtin_fmaf(low_half(scale), 8.0f, high_half(scale)) : high_half(scale);
}
__device__ __forceinline__ h8 halves8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(h8, (u4{a, b, c, d}));
}

// sum + the products of x[0 .. 15] with the values of lanes 0 .. 15 of each row: a
// fused product with a DPP operand each, which the compiler makes two instructions
// of.  (The first waits out what a DPP read needs behind a write of `of`, and what a
// read needs behind an exponential.)
__device__ __forceinline__ float dot_row(float sum, float of, const float (&x)[16]) {
#define KK_DOT_ROW(J, X) "v_fmac_f32_dpp %0, %1, %" #X " row_newbcast:" #J " row_mask:0xf bank_mask:0xf\n"
  asm("s_nop 1\n" KK_DOT_ROW(0, 2) KK_DOT_ROW(1, 3) KK_DOT_ROW(2, 4) KK_DOT_ROW(3, 5) KK_DOT_ROW(4, 6) KK_DOT_ROW(5, 7)
          KK_DOT_ROW(6, 8) KK_DOT_ROW(7, 9) KK_DOT_ROW(8, 10) KK_DOT_ROW(9, 11) KK_DOT_ROW(10, 12) KK_DOT_ROW(11, 13)
              KK_DOT_ROW(12, 14) KK_DOT_ROW(13, 15) KK_DOT_ROW(14, 16) KK_DOT_ROW(15, 17)
      : "+v"(sum)
      : "v"(of), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]), "v"(x[8]),
        "v"(x[9]), "v"(x[10]), "v"(x[11]), "v"(x[12]), "v"(x[13]), "v"(x[14]), "v"(x[15]));
#undef KK_DOT_ROW
  return sum;
}

// Two weights as the sum of two halves each; `less` holds -1, where the compiler
// does not see it: the rest is then one mixed-precision fused product, not a
// conversion and a difference.
__device__ __forceinline__ float minus_one() {
  float v = -1.0f;
  asm("" : "+s"(v));
  return v;
}
__device__ __forceinline__ void split4(float x, float y, float less, h2* hi, h2* lo) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  *hi = __builtin_convertvector((f2{x, y}), h2);
  *lo = __builtin_convertvector((f2{__builtin_fmaf(static_cast<float>((*hi)[0]), less, x),
                                    __builtin_fmaf(static_cast<float>((*hi)[1]), less, y)}), h2);
}

// Entry points of the kernels; false where a call is not theirs.
bool few_paged4_try(const QueryArgs& a, const Paged4Rows& rows, int dtype, int* status);
bool tiles_paged4_try(const QueryArgs& a, const Paged4Rows& rows, int dtype, int* status);

}  // namespace kk
