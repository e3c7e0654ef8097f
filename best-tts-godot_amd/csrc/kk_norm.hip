// Root-mean-square norms of a token's values with the residual's addition, and
// their result in 8 bits with a scale for each token.  Bound by memory (long
// calls: 8192 rows of 4096 fp16 with their residuals to 8 bits, 235 MB, in 56 us,
// 4.2 TB/s; 102 while the weights were read behind the row's sum and value by value) or
// by their launch (single tokens, 3.8 us).
#include "kk_decode.h"

namespace kk {

struct NormArgs {
  const void *x, *r;  // r: the residual, or NULL
  void *y, *sum;      // sum: x + r, or NULL
  float* scale;       // of a row's codes, where y is int8
  const void* w;      // or NULL
  int w_dt;
  int64_t rows, xs, rs, ys, ss;  // rows' strides
  int N;
  float eps;
};

// VEC values at any value's address: one 16-byte access (8 of mixed types).
template <typename T, int VEC>
struct __attribute__((packed, aligned(sizeof(T)))) Values {
  T v[VEC];
};

// The weights of values [at, at + VEC) of a row; 0 past its end.
template <typename T, int VEC>
__device__ __forceinline__ void load_weights(const NormArgs& a, int at, float (&w)[VEC]) {
  const T* from = static_cast<const T*>(a.w) + at;
  if (at + VEC <= a.N) {
    const Values<T, VEC> v = *reinterpret_cast<const Values<T, VEC>*>(from);
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = to_f32(v.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = at + e < a.N ? to_f32(from[e]) : 0.0f;
  }
}

// The sum, or the largest (NaN where one is), of the values of a row's LANES threads.
template <int LANES>
__device__ __forceinline__ double row_all(double v, bool largest, double* part) {
  auto join = [&](double a, double b) { return largest ? (b > a || b != b ? b : a) : a + b; };
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v = join(v, __shfl_xor(v, off, 64));
  if constexpr (LANES > 64) {
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < LANES / 64; ++i) v = join(v, part[i]);
  }
  return v;
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v, double* part) {
  v = wave_sum_dpp(v);
  if constexpr (LANES > 64) {
    float* p = reinterpret_cast<float*>(part);
    if (threadIdx.x % 64 == 0) p[threadIdx.x / 64] = v;
    __syncthreads();
    v = p[0];
#pragma unroll
    for (int i = 1; i < LANES / 64; ++i) v += p[i];
  }
  return v;
}

// h = x + r, y = h / sqrt(mean(h^2) + eps) w, in one pass: a row lies in the
// registers of LANES threads, NCH chunks of VEC values each.  8 bits: scale =
// max |y| / 127, code = rint(y / scale) = rint(127 h w / max |h w|), where the
// norm's factor falls out; h w in 64 bits, so that a quotient next to a half
// stays on its side of it (ten operations a value at the rate of fp32's, a tenth
// of the time that the value's bytes take).
template <typename TX, typename TR, typename TO, int VEC, int NCH, int LANES>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) rms_norm_kernel(NormArgs a) {
  constexpr bool CODES = sizeof(TO) == 1;
  constexpr int ROWS = LANES < 256 ? 256 / LANES : 1;
  using H = std::conditional_t<CODES, double, float>;
  __shared__ double part[2][LANES / 64];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / LANES;
  if (row >= a.rows) return;  // (rows share no barrier)
  const int lane = threadIdx.x % LANES;
  const TX* x = static_cast<const TX*>(a.x) + row * a.xs;
  const TR* r = static_cast<const TR*>(a.r) + row * a.rs;
  TR* sum = static_cast<TR*>(a.sum) + row * a.ss;
  TO* y = static_cast<TO*>(a.y) + row * a.ys;
  Values<TX, VEC> vx[NCH];
  Values<TR, VEC> vr[NCH];
  float w[NCH][VEC];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int at = (c * LANES + lane) * VEC;
    if (at + VEC <= a.N) {
      vx[c] = *reinterpret_cast<const Values<TX, VEC>*>(x + at);
      if (a.r) vr[c] = *reinterpret_cast<const Values<TR, VEC>*>(r + at);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        vx[c].v[e] = at + e < a.N ? x[at + e] : TX(0.0f);
        if (a.r) vr[c].v[e] = at + e < a.N ? r[at + e] : TR(0.0f);
      }
    }
  }
  if (a.w) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int at = (c * LANES + lane) * VEC;
      if (a.w_dt == KK_F32)
        load_weights<float>(a, at, w[c]);
      else
        load_weights<__half>(a, at, w[c]);
    }
  }
  float poison = 0.0f;  // NaN where a weight is not finite
  if (CODES && a.w) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) poison = __builtin_fmaf(w[c][e], 0.0f, poison);
  }
  H h[NCH][VEC], squares = 0;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int at = (c * LANES + lane) * VEC;
    Values<TR, VEC> out;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      H v = static_cast<H>(to_f32(vx[c].v[e]));
      if (a.r) v += static_cast<H>(to_f32(vr[c].v[e]));
      h[c][e] = v;
      squares = CODES ? static_cast<H>(fma(v, v, squares)) : squares + v * v;
      from_f32(out.v[e], static_cast<float>(v));
    }
    if (a.sum) {
      if (at + VEC <= a.N) {
        *reinterpret_cast<Values<TR, VEC>*>(sum + at) = out;
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (at + e < a.N) sum[at + e] = out.v[e];
      }
    }
  }
  if constexpr (CODES) {
    squares = row_all<LANES>(squares, false, part[0]);
  } else {
    squares = row_sum<LANES>(squares, part[0]);
  }
  const H by = H(1) / sqrt(squares / static_cast<H>(a.N) + static_cast<H>(a.eps));
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (!a.w) continue;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const H by_w = static_cast<H>(w[c][e]);
      h[c][e] = CODES ? h[c][e] * by_w : h[c][e] * by * by_w;
    }
  }
  if constexpr (CODES) {
    double top = 0.0;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) top = fmax(top, fabs(h[c][e]));
    // (fmax drops NaN, and a weight of 0 an infinity: squares that are not finite hold these)
    if (!(poison == 0.0f && squares < INFINITY)) top = NAN;
    top = row_all<LANES>(top, true, part[1]);
    if (lane == 0) a.scale[row] = top == 0.0 ? 0.0f : static_cast<float>(top * by / 127.0);
    const double code = top > 0.0 ? 127.0 / top : 0.0;
    if (!(top > 0.0)) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[c][e] = 0.0;
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double q = h[c][e] * code, near = rint(q);
        // (next to a half the quotient itself: 127 h w is exact where h w / max can be one)
        h[c][e] = fabs(fabs(q - near) - 0.5) < 1e-9 ? rint(127.0 * h[c][e] / top) : near;
      }
  } else if (!a.w) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[c][e] *= by;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int at = (c * LANES + lane) * VEC;
    Values<TO, VEC> out;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (CODES)
        out.v[e] = static_cast<int8_t>(static_cast<int>(h[c][e]));
      else
        from_f32(out.v[e], h[c][e]);
    }
    if (at + VEC <= a.N) {
      *reinterpret_cast<Values<TO, VEC>*>(y + at) = out;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (at + e < a.N) y[at + e] = out.v[e];
    }
  }
}

constexpr int kMostNorm = 16384;  // values of a row

template <typename TX, typename TR, typename TO, int VEC, int NCH, int LANES>
static int launch_norm(const NormArgs& a) {
  const int64_t blocks = ceil_div(a.rows, LANES < 256 ? 256 / LANES : 1);
  if (blocks > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "rms_norm: too many rows");
  KK_LAUNCH((rms_norm_kernel<TX, TR, TO, VEC, NCH, LANES>), dim3(static_cast<unsigned>(blocks)),
            dim3(LANES < 256 ? 256 : LANES), 0, ctx().stream, a);
  return check_launch("rms_norm_kernel");
}

template <typename TX, typename TR, typename TO>
static int launch_norm(const NormArgs& a) {
  constexpr int VEC = sizeof(TX) + sizeof(TR) == 4 ? 8 : 4;
  const int chunks = static_cast<int>(ceil_div(a.N, VEC));
  if (chunks <= 64) return launch_norm<TX, TR, TO, VEC, 1, 64>(a);
  if (chunks <= 256) return launch_norm<TX, TR, TO, VEC, 4, 64>(a);
  if (chunks <= 512) return launch_norm<TX, TR, TO, VEC, 2, 256>(a);
  if (chunks <= 1024) return launch_norm<TX, TR, TO, VEC, 4, 256>(a);
  return launch_norm<TX, TR, TO, VEC, kMostNorm / VEC / 1024, 1024>(a);
}

template <typename TX, typename TR>
static int launch_norm(const NormArgs& a, int out) {
  return out == KK_I8    ? launch_norm<TX, TR, int8_t>(a)
         : out == KK_F16 ? launch_norm<TX, TR, __half>(a)
                         : launch_norm<TX, TR, float>(a);
}

// A tensor as rows of N values next to each other, all `stride` apart.
static int check_rows(const kk_tensor* t, const char* name, const kk_tensor* like, int64_t* stride, const char* who) {
  KK_TRY(check_tensor(t, name));
  if (t->rank != like->rank) return set_error(KK_E_ARG, "%s: %s must have x's shape", who, name);
  for (int i = 0; i < t->rank; ++i)
    if (t->shape[i] != like->shape[i]) return set_error(KK_E_ARG, "%s: %s must have x's shape", who, name);
  *stride = 0;
  if (numel(t) == 0) return KK_OK;
  const int last = t->rank - 1;
  if (t->shape[last] != 1 && t->strides[last] != 1)
    return set_error(KK_E_ARG, "%s: a row's values of %s must lie next to each other", who, name);
  int64_t rows = 1;
  for (int i = last - 1; i >= 0; --i) {
    if (t->shape[i] == 1) continue;
    if (rows == 1)
      *stride = t->strides[i];
    else if (t->strides[i] != *stride * rows)
      return set_error(KK_E_ARG, "%s: rows of %s must be evenly spaced", who, name);
    rows *= t->shape[i];
  }
  return KK_OK;
}

static int rms_norm(const kk_tensor* out, const kk_tensor* scales, const kk_tensor* sum, const kk_tensor* x,
                    const kk_tensor* residual, const kk_tensor* weight, float eps, const char* who) {
  NormArgs a{};
  KK_TRY(check_tensor(x, "x"));
  if (x->rank < 1) return set_error(KK_E_ARG, "%s: x must have an axis", who);
  KK_TRY(check_rows(x, "x", x, &a.xs, who));
  KK_TRY(check_rows(out, "out", x, &a.ys, who));
  KK_TRY(check_writable(out, "out", who));
  if (!is_float(x->dtype)) return set_error(KK_E_ARG, "%s: x must be f32 or f16", who);
  if (scales ? out->dtype != KK_I8 : !is_float(out->dtype))
    return set_error(KK_E_ARG, "%s: out must be %s", who, scales ? "int8" : "f32 or f16");
  if (sum && !residual) return set_error(KK_E_ARG, "%s: sum without residual", who);
  if (residual) {
    KK_TRY(check_rows(residual, "residual", x, &a.rs, who));
    if (!is_float(residual->dtype)) return set_error(KK_E_ARG, "%s: residual must be f32 or f16", who);
  }
  if (sum) {
    KK_TRY(check_rows(sum, "sum", x, &a.ss, who));
    KK_TRY(check_writable(sum, "sum", who));
    if (sum->dtype != residual->dtype) return set_error(KK_E_ARG, "%s: sum must have residual's dtype", who);
  }
  const int64_t N = x->shape[x->rank - 1];
  a.rows = 1;
  for (int i = 0; i + 1 < x->rank; ++i) a.rows *= x->shape[i];
  if (scales) {
    KK_TRY(check_tensor(scales, "scales"));
    if (scales->dtype != KK_F32 || !is_contiguous(scales) || numel(scales) != a.rows)
      return set_error(KK_E_ARG, "%s: scales must be f32 in one piece, one a row", who);
  }
  if (weight) {
    KK_TRY(check_tensor(weight, "weight"));
    if (!is_float(weight->dtype) || weight->rank != 1 || weight->shape[0] != N ||
        (N > 1 && weight->strides[0] != 1))
      return set_error(KK_E_ARG, "%s: weight must be f32 or f16, a value for each of a row's, in one piece", who);
  }
  if (!(eps >= 0.0f) || eps == INFINITY) return set_error(KK_E_ARG, "%s: eps must be finite and not negative", who);
  if (N < 1 || N > kMostNorm)
    return set_error(KK_E_UNSUPPORTED, "%s: rows of %lld values (1 to %d)", who, static_cast<long long>(N), kMostNorm);
  if (sum && numel(x) > 0 && sum->data == out->data)
    return set_error(KK_E_ARG, "%s: out and sum must not be the same", who);
  KK_TRY(require_ready());
  if (a.rows == 0) return KK_OK;
  a.x = x->data;
  a.r = residual ? residual->data : nullptr;
  a.y = out->data;
  a.sum = sum ? sum->data : nullptr;
  a.scale = scales ? static_cast<float*>(scales->data) : nullptr;
  a.w = weight ? weight->data : nullptr;
  a.w_dt = weight ? weight->dtype : KK_F32;
  a.N = static_cast<int>(N);
  a.eps = eps;
  const bool rh = residual ? residual->dtype == KK_F16 : x->dtype == KK_F16;
  if (x->dtype == KK_F16)
    return rh ? launch_norm<__half, __half>(a, out->dtype) : launch_norm<__half, float>(a, out->dtype);
  return rh ? launch_norm<float, __half>(a, out->dtype) : launch_norm<float, float>(a, out->dtype);
}

}  // namespace kk

using namespace kk;

extern "C" {

int kk_rms_norm(const kk_tensor* out, const kk_tensor* sum, const kk_tensor* x, const kk_tensor* residual,
                const kk_tensor* weight, float eps) {
  return rms_norm(out, nullptr, sum, x, residual, weight, eps, "rms_norm");
}

int kk_rms_norm_quant(const kk_tensor* codes, const kk_tensor* scales, const kk_tensor* sum, const kk_tensor* x,
                      const kk_tensor* residual, const kk_tensor* weight, float eps) {
  if (!scales) return set_error(KK_E_ARG, "rms_norm_quant: scales is NULL");
  return rms_norm(codes, scales, sum, x, residual, weight, eps, "rms_norm_quant");
}

}  // extern "C"
