// A paged cache of 4-bit keys and values: tokens into their slots, and what the
// codes stand for.  Bound by memory (the codes' values: 44 MB in 7.4 us), by values that
// leave a byte a lane (3 x 2051 tokens of 12 heads of 64 in fp32, 43 MB: 15 us, where a
// copy takes 8.7) or by their launch (single tokens).
#include "kk_decode.h"

namespace kk {

struct Append4Args {
  const void* x[2];      // new keys, new values [B, T, Hk, D]
  int64_t xs[2][3];
  uint8_t* codes[2];     // [pages, Hk, block, D / 2] and [pages, Hk, D / 2, block]
  uint32_t* scales[2];   // [pages, Hk, block]: step and lowest value
  const void* slots;     // [B, T]
  int slots_dt;
  int64_t ss[2], tokens, limit;  // limit: slots of the pool
  int T, Hk, D, shift;
};

template <typename T, int VEC>
struct __attribute__((packed, aligned(sizeof(T)))) Row {
  T v[VEC];
};

constexpr int kAppend4Threads = 256;
constexpr int kAppend4Tokens = 32;  // of a block: eight lanes each
constexpr float kMost4 = 65504.0f;

// What is cached of x: fp16's range, no NaN.
__device__ __forceinline__ float cached(float x) { return x != x ? 0.0f : __builtin_amdgcn_fmed3f(x, -kMost4, kMost4); }

// clamp(rint((x - low) / step), 0, 15), of the exact quotient.  A difference, a
// reciprocal and a product in fp32 leave three roundings of 2^-24 of it: where it lies
// between 0 and 15.5, and so says which code, less than 2^-18.  Only within 2^-12 of a half
// does the quotient in 64 bits say which side it is on.  Others are clamped, however
// far off: a step that fp16 rounds to its smallest takes them to 22, a lowest value that
// it rounds up below 0.
__device__ __forceinline__ uint32_t code4(float x, float low, float step, float by) {
  const float q = (x - low) * by, r = rintf(q);
  float c = r;
  if (__builtin_fabsf(__builtin_fabsf(q - r) - 0.5f) < 0x1p-12f)
    c = static_cast<float>(rint((static_cast<double>(x) - static_cast<double>(low)) / static_cast<double>(step)));
  return static_cast<uint32_t>(__builtin_amdgcn_fmed3f(c, 0.0f, 15.0f));
}

// A block takes 32 tokens of one head of keys (blockIdx.z 0) or values (1), eight
// lanes a token: its lowest value, its step, then its codes through LDS, where a
// byte's two codes (values d and d + D / 2) meet.  Keys' bytes go out a row a
// token; of values a lane takes a token, so that tokens next to each other in a page
// are written together.  A byte is one token's alone: no two lanes share one.
template <typename T>
__global__ void __launch_bounds__(kAppend4Threads) cache4_append_kernel(Append4Args a) {
  constexpr int VEC = 16 / sizeof(T), LANES = kAppend4Threads / kAppend4Tokens;
  constexpr int NCH = 256 / (VEC * LANES);  // chunks of a lane at most
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // [tokens][pitch] codes
  __shared__ int64_t s_slot[kAppend4Tokens];
  const int which = blockIdx.z, h = blockIdx.y, D = a.D, pitch = D + 4;
  const int token = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kAppend4Tokens + token;
  int64_t slot = -1;
  if (n < a.tokens) {
    const int64_t b = n / a.T, t = n - b * a.T;
    slot = load_index(a.slots, a.slots_dt, b * a.ss[0] + t * a.ss[1]);
    if (slot >= a.limit) slot = -1;
    if (slot >= 0) {
      const T* x = static_cast<const T*>(a.x[which]) + b * a.xs[which][0] + t * a.xs[which][1] + h * a.xs[which][2];
      float v[NCH][VEC], lowest = INFINITY, most = -INFINITY;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int d = (c * LANES + lane) * VEC;
        if (d >= D) continue;
        const Row<T, VEC> in = *reinterpret_cast<const Row<T, VEC>*>(x + d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[c][e] = cached(to_f32(in.v[e]));
          lowest = fminf(lowest, v[c][e]);
          most = fmaxf(most, v[c][e]);
        }
      }
#pragma unroll
      for (int off = 1; off < LANES; off <<= 1) {
        lowest = fminf(lowest, __shfl_xor(lowest, off, 64));
        most = fmaxf(most, __shfl_xor(most, off, 64));
      }
      const __half low16 = __float2half(lowest);
      const float low = __half2float(low16);
      const __half step16 =
          __float2half(static_cast<float>((static_cast<double>(most) - static_cast<double>(low)) / 15.0));
      float step = __half2float(step16);
      step = step > 0.0f ? step : 0.0f;
      const float by = step > 0.0f ? 1.0f / step : 0.0f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int d = (c * LANES + lane) * VEC;
        if (d >= D) continue;
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          uint32_t w = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) w |= (step > 0.0f ? code4(v[c][e + i], low, step, by) : 0u) << (8 * i);
          *reinterpret_cast<uint32_t*>(lds + token * pitch + d + e) = w;
        }
      }
      if (lane == 0) {
        const int64_t page = slot >> a.shift, row = slot & ((int64_t{1} << a.shift) - 1);
        const uint32_t step_bits = step > 0.0f ? __half_as_ushort(step16) : 0u;
        a.scales[which][((page * a.Hk + h) << a.shift) + row] = step_bits | uint32_t{__half_as_ushort(low16)} << 16;
      }
    }
  }
  if (lane == 0) s_slot[token] = slot;
  __syncthreads();
  const int half = D / 2;
  const int64_t block = int64_t{1} << a.shift;
  if (which == 0) {
    const int words = half / 4;
    for (int i = threadIdx.x; i < kAppend4Tokens * words; i += kAppend4Threads) {
      const int r = i / words, w = i - r * words;
      const int64_t to = s_slot[r];
      if (to < 0) continue;
      const uint8_t* from = lds + r * pitch + 4 * w;
      const uint32_t both = *reinterpret_cast<const uint32_t*>(from) | *reinterpret_cast<const uint32_t*>(from + half) << 4;
      const int64_t at = (((to >> a.shift) * a.Hk + h) * block + (to & (block - 1))) * half;
      *reinterpret_cast<uint32_t*>(a.codes[0] + at + 4 * w) = both;
    }
  } else {
    const int r = threadIdx.x % kAppend4Tokens;
    const int64_t to = s_slot[r];
    if (to < 0) return;
    uint8_t* out = a.codes[1] + ((to >> a.shift) * a.Hk + h) * half * block + (to & (block - 1));
    for (int d = threadIdx.x / kAppend4Tokens; d < half; d += LANES)
      out[d * block] = static_cast<uint8_t>(lds[r * pitch + d] | lds[r * pitch + half + d] << 4);
  }
}

// low + step * code in fp32 (step times a code is exact there): a thread takes
// four bytes, which are two times four values next to each other.
__device__ __forceinline__ float4 values4(uint32_t w, const float2 (&s)[4]) {
  float4 v;
  v.x = __builtin_fmaf(static_cast<float>(w & 15u), s[0].x, s[0].y);
  v.y = __builtin_fmaf(static_cast<float>(w >> 8 & 15u), s[1].x, s[1].y);
  v.z = __builtin_fmaf(static_cast<float>(w >> 16 & 15u), s[2].x, s[2].y);
  v.w = __builtin_fmaf(static_cast<float>(w >> 24 & 15u), s[3].x, s[3].y);
  return v;
}
__device__ __forceinline__ float2 scale4(uint32_t w) {
  return make_float2(__half2float(__ushort_as_half(static_cast<unsigned short>(w))),
                     __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16))));
}
__global__ void __launch_bounds__(256) cache4_values_kernel(const uint32_t* k, const uint32_t* v, const uint32_t* ks,
                                                            const uint32_t* vs, float* out_k, float* out_v,
                                                            int64_t words, int half, int block) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= words) return;
  float2 s[4];
  if (blockIdx.y == 0) {
    const int per = half / 4;
    const int64_t row = i / per;
    const uint32_t w = k[i];
    s[0] = s[1] = s[2] = s[3] = scale4(ks[row]);
    float* out = out_k + row * 2 * half + 4 * (i - row * per);
    st_stream4(out, values4(w, s));
    st_stream4(out + half, values4(w >> 4, s));
  } else {
    const int per = block / 4;
    const int64_t line = i / per, head = line / half;
    const int row = 4 * static_cast<int>(i - line * per), d = static_cast<int>(line - head * half);
    const uint32_t w = v[i];
    const uint4 sw = *reinterpret_cast<const uint4*>(vs + head * block + row);
    s[0] = scale4(sw.x);
    s[1] = scale4(sw.y);
    s[2] = scale4(sw.z);
    s[3] = scale4(sw.w);
    float* out = out_v + (head * 2 * half + d) * block + row;
    st_stream4(out, values4(w, s));
    st_stream4(out + static_cast<int64_t>(half) * block, values4(w >> 4, s));
  }
}

}  // namespace kk

using namespace kk;

extern "C" {

int kk_cache4_append(const kk_tensor* k_codes, const kk_tensor* k_scales, const kk_tensor* v_codes,
                     const kk_tensor* v_scales, const kk_tensor* k, const kk_tensor* v, const kk_tensor* slots) {
  const char* who = "cache4_append";
  CacheShape c;
  KK_TRY(check_codes4(k_codes, k_scales, v_codes, v_scales, &c, who));
  KK_TRY(check_heads(k, "k", who));
  KK_TRY(check_heads(v, "v", who));
  if (k->dtype != v->dtype) return set_error(KK_E_ARG, "%s: k and v must have one dtype", who);
  for (int i = 0; i < 4; ++i)
    if (k->shape[i] != v->shape[i]) return set_error(KK_E_ARG, "%s: k and v must have one shape", who);
  if (k->shape[2] != c.heads || k->shape[3] != c.D)
    return set_error(KK_E_ARG, "%s: heads of k do not fit the cache's", who);
  KK_TRY(check_tensor(slots, "slots"));
  if (!is_index(slots->dtype) || slots->rank != 2 || slots->shape[0] != k->shape[0] || slots->shape[1] != k->shape[1])
    return set_error(KK_E_ARG, "%s: slots must be int32 or int64 [sequences, tokens]", who);
  Append4Args a{};
  const kk_tensor *xs[2] = {k, v}, *codes[2] = {k_codes, v_codes}, *scales[2] = {k_scales, v_scales};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = xs[i]->data;
    for (int j = 0; j < 3; ++j) a.xs[i][j] = xs[i]->strides[j];
    a.codes[i] = static_cast<uint8_t*>(codes[i]->data);
    a.scales[i] = static_cast<uint32_t*>(scales[i]->data);
  }
  a.slots = slots->data;
  a.slots_dt = slots->dtype;
  a.ss[0] = slots->strides[0];
  a.ss[1] = slots->strides[1];
  a.tokens = k->shape[0] * k->shape[1];
  a.limit = c.pages * c.block;
  if (k->shape[1] > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many tokens", who);
  a.T = static_cast<int>(k->shape[1]);
  a.Hk = static_cast<int>(c.heads);
  a.D = static_cast<int>(c.D);
  a.shift = __builtin_ctzll(static_cast<unsigned long long>(c.block));
  KK_TRY(require_ready());
  if (a.tokens == 0 || a.limit == 0) return KK_OK;
  const int64_t blocks = ceil_div(a.tokens, kAppend4Tokens);
  if (blocks > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many tokens", who);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(c.heads), 2);
  const unsigned bytes = static_cast<unsigned>(kAppend4Tokens * (c.D + 4));
  if (k->dtype == KK_F16)
    KK_LAUNCH(cache4_append_kernel<__half>, grid, dim3(kAppend4Threads), bytes, ctx().stream, a);
  else
    KK_LAUNCH(cache4_append_kernel<float>, grid, dim3(kAppend4Threads), bytes, ctx().stream, a);
  return check_launch("cache4_append_kernel");
}

int kk_cache4_values(const kk_tensor* out_k, const kk_tensor* out_v, const kk_tensor* k_codes,
                     const kk_tensor* k_scales, const kk_tensor* v_codes, const kk_tensor* v_scales) {
  const char* who = "cache4_values";
  CacheShape c;
  KK_TRY(check_codes4(k_codes, k_scales, v_codes, v_scales, &c, who));
  const kk_tensor* outs[2] = {out_k, out_v};
  const char* names[2] = {"out_k", "out_v"};
  for (int i = 0; i < 2; ++i) {
    KK_TRY(check_tensor(outs[i], names[i]));
    if (outs[i]->dtype != KK_F32 || outs[i]->rank != 4 || !is_contiguous(outs[i]) ||
        reinterpret_cast<uintptr_t>(outs[i]->data) % 16)
      return set_error(KK_E_ARG, "%s: %s must be f32 of four axes in one piece, 16-byte aligned", who, names[i]);
    if (outs[i]->shape[0] != c.pages || outs[i]->shape[1] != c.heads || outs[i]->shape[2] != (i ? c.D : c.block) ||
        outs[i]->shape[3] != (i ? c.block : c.D))
      return set_error(KK_E_ARG, "%s: %s must be [pages, heads, %s]", who, names[i], i ? "values, rows" : "rows, values");
  }
  KK_TRY(require_ready());
  const int64_t words = c.pages * c.heads * c.block * c.D / 8;
  if (words == 0) return KK_OK;
  const int64_t blocks = ceil_div(words, 256);
  if (blocks > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many pages", who);
  KK_LAUNCH(cache4_values_kernel, dim3(static_cast<unsigned>(blocks), 2), dim3(256), 0, ctx().stream,
            static_cast<const uint32_t*>(k_codes->data), static_cast<const uint32_t*>(v_codes->data),
            static_cast<const uint32_t*>(k_scales->data), static_cast<const uint32_t*>(v_scales->data),
            static_cast<float*>(out_k->data), static_cast<float*>(out_v->data), words, static_cast<int>(c.D / 2),
            static_cast<int>(c.block));
  return check_launch("cache4_values_kernel");
}

}  // extern "C"
