// The steps of an autoregressive token decoder around its attention: norms of
// queries and keys with the position rotation, keys and values into a cache
// of 8-bit codes, and penalties, biases and grammar masks on logits.  All are
// bound by memory (long calls) or by their launch (single tokens).
#include "kk_decode.h"

namespace kk {

// ------------------------------------------------------ norm and rotation
// What one launch does to queries (0) and keys (1).
struct RotArgs {
  const void* x[2];
  void* y[2];
  const void* w[2];  // norm weights, or NULL
  int w_dt[2];
  int heads[2];
  int64_t xs[2][3], ys[2][3];  // strides over sequences, tokens, heads
  const void* pos;
  int pos_dt;
  int64_t ps[2];
  const int64_t* turns;
  int T, D, half;    // half: pairs of a head that turn
  int interleaved, norm[2];
  float eps, amplitude;
};

// sin and cos of 2 pi f / 2^32: to the nearest quarter turn in whole numbers,
// then the Taylor series on the remaining eighth (the first terms left out are
// below 2e-9 and 2e-10), so that the error is that of the last rounding.
__device__ __forceinline__ float2 turn_cos_sin(uint32_t f) {
  const uint32_t quarter = (f + 0x20000000u) >> 30;
  const int32_t rest = static_cast<int32_t>(f - (quarter << 30));
  const float a = static_cast<float>(rest) * 0x1.921fb6p-30f;  // 2 pi / 2^32
  const float a2 = a * a;
  float s = 0x1.71de3ap-19f;                      //  1/9!
  s = __builtin_fmaf(s, a2, -0x1.a01a02p-13f);    // -1/7!
  s = __builtin_fmaf(s, a2, 0x1.111112p-7f);      //  1/5!
  s = __builtin_fmaf(s, a2, -0x1.555556p-3f);     // -1/3!
  s = __builtin_fmaf(a2 * a, s, a);
  float c = -0x1.27e4fcp-22f;                     // -1/10!
  c = __builtin_fmaf(c, a2, 0x1.a01a02p-16f);     //  1/8!
  c = __builtin_fmaf(c, a2, -0x1.6c16c2p-10f);    // -1/6!
  c = __builtin_fmaf(c, a2, 0x1.555556p-5f);      //  1/4!
  c = __builtin_fmaf(c, a2, -0.5f);
  c = __builtin_fmaf(c, a2, 1.0f);
  const float cq = (quarter & 1) ? -s : c, sq = (quarter & 1) ? c : s;
  return (quarter & 2) ? make_float2(-cq, -sq) : make_float2(cq, sq);
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
  T v[VEC];
};

// Stores a chunk, past the caches if STREAM and it is 16 bytes.
template <bool STREAM, typename T, int VEC>
__device__ __forceinline__ void put_chunk(T* p, const Chunk<T, VEC>& c) {
  if constexpr (STREAM && sizeof(c) == 16)
    __builtin_nontemporal_store(__builtin_bit_cast(kk_f4v, c), reinterpret_cast<kk_f4v*>(p));
  else
    *reinterpret_cast<Chunk<T, VEC>*>(p) = c;
}

constexpr int kRotThreads = 256;
constexpr int kRotPairs = 128;   // pairs of a head at most
constexpr int kRotTokens = 4;    // tokens of a block at most

// y = A R(pos) (x rsqrt(mean x^2 + eps) w) for each head: bound by memory, x
// once in and y once out.  A block takes `tokens` tokens; their angles' sines
// and cosines, the same for all heads, are formed once into LDS.  A head lies
// over `lanes` lanes, each with two chunks of VEC values that turn against
// each other (or, past the turned part, two that pass): no lane needs
// another's values but for the norm's sum.  The angle is pos * turns modulo
// 2^64 in 2^64ths of a turn, exact for any position.  4 x 4096 tokens of 40 fp16
// heads of 128: 65 us alone, 79 in a row of calls (4.3 TB/s of a copy's 4.75).
template <typename T, int VEC, int NCH, bool STREAM>
__global__ void __launch_bounds__(kRotThreads) qk_norm_rotary_kernel(RotArgs a, int64_t rows, int tokens, int lanes) {
  __shared__ float2 table[kRotTokens * kRotPairs];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens;
  const int here = static_cast<int>(rows - first < tokens ? rows - first : tokens);
  for (int i = threadIdx.x; i < here * a.half; i += kRotThreads) {
    const int64_t row = first + i / a.half;
    const int64_t at = (row / a.T) * a.ps[0] + (row % a.T) * a.ps[1];
    const uint64_t turn = static_cast<uint64_t>(load_index(a.pos, a.pos_dt, at)) *
                          static_cast<uint64_t>(a.turns[i % a.half]);
    const float2 cs = turn_cos_sin(static_cast<uint32_t>(turn >> 32));
    table[i] = make_float2(cs.x * a.amplitude, cs.y * a.amplitude);
  }
  __syncthreads();
  const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes, groups = kRotThreads / lanes;
  const int turned = (a.half + VEC - 1) / VEC, slots = (a.D + 2 * VEC - 1) / (2 * VEC);
  int at0[NCH], at1[NCH], pair[NCH];  // the lane's two chunks, and their first pair (-1: they pass)
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int s = lane + c * lanes;
    pair[c] = s < turned ? s * VEC : -1;
    if (s >= slots) {
      at0[c] = at1[c] = a.D;
    } else if (s >= turned || a.interleaved) {
      at0[c] = 2 * VEC * s;
      at1[c] = at0[c] + VEC;
    } else {
      at0[c] = s * VEC;
      at1[c] = a.half + s * VEC;
    }
  }
  for (int which = 0; which < 2; ++which) {
    if (!a.x[which]) continue;
    const int heads = a.heads[which];
    float w0[NCH][VEC], w1[NCH][VEC];
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        w0[c][e] = w1[c][e] = 1.0f;
        if (a.w[which] && at0[c] < a.D) w0[c][e] = load_as_f32(a.w[which], a.w_dt[which], at0[c] + e);
        if (a.w[which] && at1[c] < a.D) w1[c][e] = load_as_f32(a.w[which], a.w_dt[which], at1[c] + e);
      }
    for (int r = blockIdx.y * groups + group; r < here * heads; r += gridDim.y * groups) {
      const int tok = r / heads, head = r - tok * heads;
      const int64_t row = first + tok, b = row / a.T, t = row % a.T;
      const T* x = static_cast<const T*>(a.x[which]) + b * a.xs[which][0] + t * a.xs[which][1] +
                   head * a.xs[which][2];
      T* y = static_cast<T*>(a.y[which]) + b * a.ys[which][0] + t * a.ys[which][1] + head * a.ys[which][2];
      float u[NCH][VEC], v[NCH][VEC], sum = 0.0f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        Chunk<T, VEC> cu = {}, cv = {};
        if (at0[c] < a.D) cu = *reinterpret_cast<const Chunk<T, VEC>*>(x + at0[c]);
        if (at1[c] < a.D) cv = *reinterpret_cast<const Chunk<T, VEC>*>(x + at1[c]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          u[c][e] = to_f32(cu.v[e]);
          v[c][e] = to_f32(cv.v[e]);
          sum += u[c][e] * u[c][e] + v[c][e] * v[c][e];
        }
      }
      if (a.norm[which]) {
        for (int off = lanes / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        const float r = 1.0f / sqrtf(sum / static_cast<float>(a.D) + a.eps);
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            u[c][e] = u[c][e] * r * w0[c][e];
            v[c][e] = v[c][e] * r * w1[c][e];
          }
      }
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        Chunk<T, VEC> cu, cv;
        if (pair[c] >= 0 && !a.interleaved) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float2 cs = table[tok * a.half + pair[c] + e];
            from_f32(cu.v[e], u[c][e] * cs.x - v[c][e] * cs.y);
            from_f32(cv.v[e], v[c][e] * cs.x + u[c][e] * cs.y);
          }
        } else if (pair[c] >= 0 && VEC == 1) {
          const float2 cs = table[tok * a.half + pair[c]];
          from_f32(cu.v[0], u[c][0] * cs.x - v[c][0] * cs.y);
          from_f32(cv.v[0], v[c][0] * cs.x + u[c][0] * cs.y);
        } else if (pair[c] >= 0) {
#pragma unroll
          for (int e = 0; e + 1 < VEC; e += 2) {
            const float2 p = table[tok * a.half + pair[c] + e / 2];
            const float2 q = table[tok * a.half + pair[c] + VEC / 2 + e / 2];
            from_f32(cu.v[e], u[c][e] * p.x - u[c][e + 1] * p.y);
            from_f32(cu.v[e + 1], u[c][e + 1] * p.x + u[c][e] * p.y);
            from_f32(cv.v[e], v[c][e] * q.x - v[c][e + 1] * q.y);
            from_f32(cv.v[e + 1], v[c][e + 1] * q.x + v[c][e] * q.y);
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            from_f32(cu.v[e], u[c][e]);
            from_f32(cv.v[e], v[c][e]);
          }
        }
        if (at0[c] < a.D) put_chunk<STREAM>(y + at0[c], cu);
        if (at1[c] < a.D) put_chunk<STREAM>(y + at1[c], cv);
      }
    }
  }
}

// Whether rows of t start at multiples of `bytes` (VEC-wide accesses).
static bool rows_aligned(const kk_tensor* t, int bytes) {
  if (reinterpret_cast<uintptr_t>(t->data) % bytes) return false;
  for (int i = 0; i + 1 < t->rank; ++i)
    if (t->shape[i] > 1 && (t->strides[i] * dtype_size(t->dtype)) % bytes) return false;
  return true;
}

template <typename T, int VEC, int NCH, bool STREAM = false>
static int launch_rotary(const RotArgs& a, int64_t rows) {
  const int slots = (a.D + 2 * VEC - 1) / (2 * VEC);
  int lanes = 1;
  while (lanes * NCH < slots) lanes *= 2;
  const int groups = kRotThreads / lanes;
  // several tokens share a block's set-up once there are blocks for every CU
  // eight times over; few tokens spread their heads over blocks instead
  int tokens = 1;
  while (tokens < kRotTokens && rows / (2 * tokens) >= 8 * ctx().num_cus) tokens *= 2;
  const int64_t blocks = ceil_div(rows, tokens);
  const int widest = a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1];
  const int split = blocks * 4 <= ctx().num_cus ? static_cast<int>(ceil_div(int64_t{widest} * tokens, groups)) : 1;
  if (blocks > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "qk_norm_rotary: too many tokens");
  KK_LAUNCH((qk_norm_rotary_kernel<T, VEC, NCH, STREAM>), dim3(static_cast<unsigned>(blocks), split), dim3(kRotThreads), 0,
            ctx().stream, a, rows, tokens, lanes);
  return check_launch("qk_norm_rotary_kernel");
}

// --------------------------------------------------------- cache: appending
struct AppendArgs {
  const void* x[2];           // new keys, new values
  int64_t xs[2][3];
  int8_t* codes[2];           // [pages, Hk, block, D] and [pages, Hk, D, block]
  float* scales[2];           // [pages, Hk]
  const int32_t* table;       // [B, columns]
  int64_t table_stride;
  const void* starts;
  const void* counts;         // or NULL: T each
  int starts_dt, counts_dt;
  int64_t starts_st, counts_st, pages, columns;
  int T, Hk, D, block;
};

// rint(x / s) within +-127, of the exact quotient: the product with 1 / s is
// within one of it, and the remainder x - q s, which the FMA leaves exact
// where a half is near, says which side of the half x lies on.  Infinities
// saturate, NaN gives 0.
__device__ __forceinline__ int quantised(float x, float s, float rs) {
  if (!(s > 0.0f) || x != x) return 0;
  float q = rintf(fminf(fmaxf(x * rs, -127.0f), 127.0f));
  if (__builtin_fabsf(x) <= 127.0f * s) {
    const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
    const bool odd = static_cast<int>(q) & 1;
    if (r > h || (r == h && odd)) q += 1.0f;
    if (r < -h || (r == -h && odd)) q -= 1.0f;
  }
  return static_cast<int>(q);
}

constexpr int kAppendThreads = 256;

// New rows of one sequence into one of the pages they reach, for one head of
// keys (blockIdx.z even) or values (odd): the block that has a page alone
// reads and writes it, so no two blocks meet.  s' = max(s, largest / 127)
// where the page holds rows before the new ones (which are brought to s'),
// largest / 127 where it holds none.  Bound by memory (long calls): rows come in
// 16 bytes a lane, the second time from the caches; keys' codes go out as they
// come, values' codes through LDS, where a row of the page is 16 tokens of one
// value, so that both write whole pieces of lines.  3 x 2051 fp32 tokens, 12 heads
// of 64, pages of 32: 18 us for 47 MB (29 us one value a lane, values' codes
// scattered); 32 single tokens of 8 heads of 128: 6 us.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(AppendArgs a) {
  __shared__ float part[kAppendThreads / 64];
  extern __shared__ __attribute__((aligned(16))) uint8_t turned[];  // values: [D][block + 4]
  constexpr int VEC = WIDE ? 16 / sizeof(T) : 1;
  const int b = blockIdx.x, h = blockIdx.y, which = blockIdx.z & 1, D = a.D;
  int64_t count = a.T;
  if (a.counts) count = load_index(a.counts, a.counts_dt, b * a.counts_st);
  const PageRows w = page_rows(load_index(a.starts, a.starts_dt, b * a.starts_st), count, a.T, a.block, a.columns,
                               blockIdx.z >> 1);
  if (w.rows <= 0) return;
  const int64_t page = a.table[b * a.table_stride + w.column];
  if (page < 0 || page >= a.pages) return;
  const int64_t xt = a.xs[which][1];
  const T* x = static_cast<const T*>(a.x[which]) + b * a.xs[which][0] + w.token * xt + h * a.xs[which][2];
  const int per = D / VEC, n = w.rows * per;  // pieces of a row, and all
  float top = 0.0f;
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const int r = i / per, d = (i - r * per) * VEC;
    const Chunk<T, VEC> c = *reinterpret_cast<const Chunk<T, VEC>*>(x + r * xt + d);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float v = __builtin_fabsf(to_f32(c.v[e]));
      if (v < INFINITY) top = fmaxf(top, v);
    }
  }
  top = wave_max_dpp(top);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = top;
  float* scale = a.scales[which] + page * a.Hk + h;
  const float before = w.held ? *scale : 0.0f;
  __syncthreads();
  top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  // a page of values below 2^-119 keeps a scale that can be divided by
  const float want = top > 0.0f ? fmaxf(top / 127.0f, 0x1p-126f) : 0.0f;
  const float s = fmaxf(before, want);
  int8_t* codes = a.codes[which] + (page * a.Hk + h) * a.block * D;
  if (threadIdx.x == 0) *scale = s;
  if (w.held && s != before) {
    // what the page holds, four codes at once: of a row of keys, or of a value's tokens
    const double by = static_cast<double>(before) / s;
    uint32_t* words = reinterpret_cast<uint32_t*>(codes);
    const int row = which ? a.block / 4 : w.held * D / 4, used = which ? (w.held + 3) / 4 : row;
    for (int i = threadIdx.x; i < (which ? D : 1) * used; i += kAppendThreads) {
      const int r = i / used, at = i - r * used;
      const uint32_t old = words[r * row + at];
      uint32_t now = old;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (which && 4 * at + e >= w.held) continue;
        const int c = static_cast<int8_t>(old >> (8 * e));
        const uint32_t q = static_cast<uint8_t>(static_cast<int8_t>(rint(c * by)));
        now = (now & ~(0xffu << (8 * e))) | q << (8 * e);
      }
      if (now != old) words[r * row + at] = now;
    }
    __syncthreads();  // (a word may hold rows of both kinds)
  }
  const float rs = s > 0.0f ? 1.0f / s : 0.0f;
  const int pitch = a.block + 4;
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const int r = i / per, d = (i - r * per) * VEC;
    const Chunk<T, VEC> c = *reinterpret_cast<const Chunk<T, VEC>*>(x + r * xt + d);
    Chunk<int8_t, VEC> q;
#pragma unroll
    for (int e = 0; e < VEC; ++e) q.v[e] = static_cast<int8_t>(quantised(to_f32(c.v[e]), s, rs));
    if (which) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) turned[(d + e) * pitch + w.held + r] = static_cast<uint8_t>(q.v[e]);
    } else {
      *reinterpret_cast<Chunk<int8_t, VEC>*>(codes + (w.held + r) * D + d) = q;
    }
  }
  if (!which) return;
  __syncthreads();
  const int first = w.held / 16, groups = (w.held + w.rows + 15) / 16 - first;
  for (int i = threadIdx.x; i < D * groups; i += kAppendThreads) {
    const int d = i / groups, t = 16 * (first + i - d * groups);
    const uint8_t* from = turned + d * pitch + t;
    int8_t* to = codes + d * a.block + t;
    if (t >= w.held && t + 16 <= w.held + w.rows) {
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = reinterpret_cast<const uint32_t*>(from)[e];
      *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
    } else {
      for (int e = 0; e < 16; ++e)
        if (t + e >= w.held && t + e < w.held + w.rows) to[e] = static_cast<int8_t>(from[e]);
    }
  }
}

// What the codes of a cache stand for: codes in, four times their bytes out.  A
// wave takes 256 codes of one page and head at a time (pages hold a multiple
// of that), so the scale is one value a wave, and stores whole lines.  9.6
// million codes: 8.6 us, 5.6 TB/s.
constexpr int kValuesEach = 4;  // rounds of a block
__global__ void __launch_bounds__(256) cache_values_kernel(const int8_t* k, const int8_t* v, const float* ks,
                                                           const float* vs, float* out_k, float* out_v, int64_t waves,
                                                           int64_t waves_a_page) {
  const int lane = threadIdx.x % 64;
  const int8_t* codes = blockIdx.y ? v : k;
  const float* scales = blockIdx.y ? vs : ks;
  float* out = blockIdx.y ? out_v : out_k;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (4 * kValuesEach) + threadIdx.x / 64;
  uint32_t w[kValuesEach];
  float s[kValuesEach];
#pragma unroll
  for (int i = 0; i < kValuesEach; ++i) {
    const int64_t at = first + 4 * i < waves ? first + 4 * i : waves - 1;
    w[i] = reinterpret_cast<const uint32_t*>(codes)[at * 64 + lane];
    s[i] = scales[at / waves_a_page];
  }
#pragma unroll
  for (int i = 0; i < kValuesEach; ++i) {
    if (first + 4 * i >= waves) continue;
    float4 x;
    x.x = static_cast<float>(static_cast<int8_t>(w[i])) * s[i];
    x.y = static_cast<float>(static_cast<int8_t>(w[i] >> 8)) * s[i];
    x.z = static_cast<float>(static_cast<int8_t>(w[i] >> 16)) * s[i];
    x.w = static_cast<float>(static_cast<int8_t>(w[i] >> 24)) * s[i];
    st_stream4(out + ((first + 4 * i) * 64 + lane) * 4, x);
  }
}

// ------------------------------------------------------------------- logits
struct LogitArgs {
  const void* x;
  int64_t xs;
  float* y;
  int64_t ys;
  const void *history, *lengths;
  int history_dt, lengths_dt;
  int64_t hs, lengths_st, L;
  const float *rep, *pres, *freq;
  int64_t rep_st, pres_st, freq_st;
  const float* bias;
  int64_t bias_st;
  const int32_t* allowed;
  int64_t allowed_st;
  int64_t V;
};

constexpr int kLogitThreads = 256;
constexpr int kLogitTile = 8192;

// x = a logit, c how often its token is in the row's history:
// c > 0: x / r where x > 0, else x r; less f c + p; then the bias, and -inf
// where the mask has no bit.  Bound by memory.  A block takes kLogitTile tokens
// of a row and counts the row's history among them in LDS (whole numbers: no
// order of the atomic additions shows), then passes over its logits, four a lane.
// 64 rows of 131072 fp16 logits and 4096 tokens: 13.8 us, 3.8 TB/s (38 us one
// logit a lane).
template <typename T>
__global__ void __launch_bounds__(kLogitThreads) process_logits_kernel(LogitArgs a) {
  constexpr int VEC = 4;
  __shared__ __attribute__((aligned(16))) uint32_t count[kLogitTile];
  const int64_t row = blockIdx.y, lo = static_cast<int64_t>(blockIdx.x) * kLogitTile;
  const int n = static_cast<int>(a.V - lo < kLogitTile ? a.V - lo : kLogitTile);
  const bool counted = a.history != nullptr;
  if (counted) {
    for (int i = threadIdx.x; i < n; i += kLogitThreads) count[i] = 0;
    __syncthreads();
    int64_t len = a.L;
    if (a.lengths) {
      const int64_t l = load_index(a.lengths, a.lengths_dt, row * a.lengths_st);
      len = l < 0 ? 0 : (l < a.L ? l : a.L);
    }
    constexpr int kIds = 4;  // in flight
    for (int64_t i = threadIdx.x; i < len; i += kIds * kLogitThreads) {
      int64_t id[kIds];
#pragma unroll
      for (int e = 0; e < kIds; ++e) {
        const int64_t at = i + e * kLogitThreads;
        id[e] = at < len ? load_index(a.history, a.history_dt, row * a.hs + at) - lo : -1;
      }
#pragma unroll
      for (int e = 0; e < kIds; ++e)
        if (id[e] >= 0 && id[e] < n) atomicAdd(&count[id[e]], 1u);
    }
    __syncthreads();
  }
  const float rep = a.rep ? a.rep[row * a.rep_st] : 1.0f, pres = a.pres ? a.pres[row * a.pres_st] : 0.0f;
  const float freq = a.freq ? a.freq[row * a.freq_st] : 0.0f;
  const T* x = static_cast<const T*>(a.x) + row * a.xs + lo;
  const float* bias = a.bias ? a.bias + row * a.bias_st + lo : nullptr;
  const int32_t* allowed = a.allowed ? a.allowed + row * a.allowed_st + lo / 32 : nullptr;
  float* y = a.y + row * a.ys + lo;
  auto one = [&](float v, uint32_t c, float add, bool there) {
    if (c) {
      v = v > 0.0f ? v / rep : v * rep;
      v = v - freq * static_cast<float>(c) - pres;
    }
    v += add;
    return there ? v : -INFINITY;
  };
  for (int i = threadIdx.x * VEC; i < n; i += kLogitThreads * VEC) {
    if (i + VEC <= n) {
      Chunk<T, VEC> c;  // (rows start anywhere)
      Chunk<float, VEC> add = {};
      Chunk<uint32_t, VEC> often = {};
      kk_f4u out;
      __builtin_memcpy(&c, x + i, sizeof c);
      if (bias) __builtin_memcpy(&add, bias + i, sizeof add);
      if (counted) often = *reinterpret_cast<const Chunk<uint32_t, VEC>*>(count + i);
      const uint32_t bits = allowed ? static_cast<uint32_t>(allowed[i >> 5]) >> (i & 31) : 0xffffffffu;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float v = one(to_f32(c.v[e]), often.v[e], add.v[e], bits >> e & 1);
        out[e] = bias || often.v[e] || !(bits >> e & 1) ? v : to_f32(c.v[e]);  // (-0 stays -0)
      }
      __builtin_nontemporal_store(out, reinterpret_cast<kk_f4u*>(y + i));
      continue;
    }
    for (int e = i; e < n && e < i + VEC; ++e) {
      const float v = to_f32(x[e]);
      const uint32_t often = counted ? count[e] : 0;
      const bool there = !allowed || (allowed[e >> 5] >> (e & 31) & 1);
      y[e] = bias || often || !there ? one(v, often, bias ? bias[e] : 0.0f, there) : v;
    }
  }
}

}  // namespace kk

using namespace kk;

extern "C" {

int kk_qk_norm_rotary(const kk_tensor* out_q, const kk_tensor* out_k, const kk_tensor* q, const kk_tensor* k,
                      const kk_tensor* q_weight, const kk_tensor* k_weight, const kk_tensor* positions,
                      const kk_tensor* turns, float eps, int interleaved, float amplitude) {
  const char* who = "qk_norm_rotary";
  RotArgs a{};
  const kk_tensor *xs[2] = {q, k}, *ys[2] = {out_q, out_k}, *ws[2] = {q_weight, k_weight};
  const char *names[2] = {"q", "k"}, *outs[2] = {"out_q", "out_k"}, *weights[2] = {"q_weight", "k_weight"};
  KK_TRY(check_heads(q, "q", who));
  const int64_t B = q->shape[0], T = q->shape[1], D = q->shape[3];
  if (D < 1 || D > 2 * kRotPairs)
    return set_error(KK_E_UNSUPPORTED, "%s: heads of %lld values (1 to %d)", who, static_cast<long long>(D),
                     2 * kRotPairs);
  if (!(eps >= 0.0f)) return set_error(KK_E_ARG, "%s: eps must not be negative", who);
  bool wide = true;
  for (int i = 0; i < 2; ++i) {
    if (!xs[i]) {
      if (ys[i] || ws[i]) return set_error(KK_E_ARG, "%s: %s given without k", who, ys[i] ? outs[i] : weights[i]);
      continue;
    }
    KK_TRY(check_heads(xs[i], names[i], who));
    KK_TRY(check_heads(ys[i], outs[i], who));
    KK_TRY(check_writable(ys[i], outs[i], who));
    if (xs[i]->dtype != q->dtype || ys[i]->dtype != q->dtype)
      return set_error(KK_E_ARG, "%s: %s and %s must have q's dtype", who, names[i], outs[i]);
    if (xs[i]->shape[0] != B || xs[i]->shape[1] != T || xs[i]->shape[3] != D)
      return set_error(KK_E_ARG, "%s: k must have q's sequences, tokens and values a head", who);
    for (int j = 0; j < 4; ++j)
      if (ys[i]->shape[j] != xs[i]->shape[j])
        return set_error(KK_E_ARG, "%s: %s must have the shape of %s", who, outs[i], names[i]);
    if (xs[i]->shape[2] > 65535) return set_error(KK_E_UNSUPPORTED, "%s: too many heads", who);
    if (ws[i]) {
      KK_TRY(check_tensor(ws[i], weights[i]));
      if (!is_float(ws[i]->dtype) || ws[i]->rank != 1 || ws[i]->shape[0] != D || !is_contiguous(ws[i]))
        return set_error(KK_E_ARG, "%s: %s must be %lld f32 or f16 values in one piece", who, weights[i],
                         static_cast<long long>(D));
      a.w[i] = ws[i]->data;
      a.w_dt[i] = ws[i]->dtype;
      a.norm[i] = 1;
    }
    a.x[i] = xs[i]->data;
    a.y[i] = ys[i]->data;
    a.heads[i] = static_cast<int>(xs[i]->shape[2]);
    for (int j = 0; j < 3; ++j) {
      a.xs[i][j] = xs[i]->strides[j];
      a.ys[i][j] = ys[i]->strides[j];
    }
    wide = wide && rows_aligned(xs[i], 16) && rows_aligned(ys[i], 16);
  }
  if (turns) {
    KK_TRY(check_tensor(turns, "turns"));
    if (turns->dtype != KK_I64 || turns->rank != 1 || !is_contiguous(turns))
      return set_error(KK_E_ARG, "%s: turns must be int64 values in one piece", who);
    if (2 * turns->shape[0] > D)
      return set_error(KK_E_ARG, "%s: %lld pairs do not fit a head of %lld values", who,
                       static_cast<long long>(turns->shape[0]), static_cast<long long>(D));
    a.turns = static_cast<const int64_t*>(turns->data);
    a.half = static_cast<int>(turns->shape[0]);
  }
  if (a.half) {
    KK_TRY(check_tensor(positions, "positions"));
    if (!is_index(positions->dtype)) return set_error(KK_E_ARG, "%s: positions must be int32 or int64", who);
    const int r = positions->rank;
    if (r < 1 || r > 2 || (positions->shape[r - 1] != T && positions->shape[r - 1] != 1) ||
        (r == 2 && positions->shape[0] != B && positions->shape[0] != 1))
      return set_error(KK_E_ARG, "%s: positions must be [tokens] or [sequences, tokens]", who);
    a.pos = positions->data;
    a.pos_dt = positions->dtype;
    a.ps[0] = r == 2 && positions->shape[0] > 1 ? positions->strides[0] : 0;
    a.ps[1] = positions->shape[r - 1] > 1 ? positions->strides[r - 1] : 0;
  }
  if (T > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many tokens", who);
  a.T = static_cast<int>(T);
  a.D = static_cast<int>(D);
  a.interleaved = interleaved != 0;
  a.eps = eps;
  a.amplitude = amplitude;
  KK_TRY(require_ready());
  if (B * T == 0 || a.heads[0] + a.heads[1] == 0) return KK_OK;
  // sixteen-byte chunks where both chunks of a lane are whole and aligned
  const int vec = q->dtype == KK_F16 ? 8 : 4;
  wide = wide && D % (2 * vec) == 0 && (2 * a.half) % (2 * vec) == 0;
  // outputs beyond what the caches hold go past them (32 + 8 heads of 128 in fp16,
  // through the caches and past them: 112 MB 53 and 55 us, 144 MB 62 and 66, 168 MB
  // 83 and 79, 256 MB 116 and 111; fp32 144 MB 56 and 61, 256 MB 110 and 107)
  const bool stream = B * T * (a.heads[0] + a.heads[1]) * D * dtype_size(q->dtype) > int64_t{152} << 20;
  if (q->dtype == KK_F16)
    return !wide    ? launch_rotary<__half, 1, 2>(a, B * T)
           : stream ? launch_rotary<__half, 8, 1, true>(a, B * T)
                    : launch_rotary<__half, 8, 1>(a, B * T);
  return !wide    ? launch_rotary<float, 1, 2>(a, B * T)
         : stream ? launch_rotary<float, 4, 1, true>(a, B * T)
                  : launch_rotary<float, 4, 1>(a, B * T);
}

int kk_cache_append(const kk_tensor* k_codes, const kk_tensor* k_scales, const kk_tensor* v_codes,
                    const kk_tensor* v_scales, const kk_tensor* k, const kk_tensor* v, const kk_tensor* table,
                    const kk_tensor* starts, const kk_tensor* counts) {
  const char* who = "cache_append";
  CacheShape c;
  KK_TRY(check_cache(k_codes, k_scales, v_codes, v_scales, table, &c, who));
  KK_TRY(check_heads(k, "k", who));
  KK_TRY(check_heads(v, "v", who));
  const int64_t B = k->shape[0], T = k->shape[1];
  for (int j = 0; j < 4; ++j)
    if (k->shape[j] != v->shape[j]) return set_error(KK_E_ARG, "%s: k and v must have one shape", who);
  if (k->dtype != v->dtype) return set_error(KK_E_ARG, "%s: k and v must have one dtype", who);
  if (k->shape[2] != c.heads || k->shape[3] != c.D)
    return set_error(KK_E_ARG, "%s: the cache holds %lld heads of %lld values", who,
                     static_cast<long long>(c.heads), static_cast<long long>(c.D));
  if (table->shape[0] != B) return set_error(KK_E_ARG, "%s: table must have a row a sequence", who);
  KK_TRY(check_per_row(starts, "starts", B, true, who));
  if (counts) KK_TRY(check_per_row(counts, "counts", B, true, who));
  if (B > 0x7fffffff || T > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many rows", who);
  AppendArgs a{};
  const kk_tensor *xs[2] = {k, v}, *codes[2] = {k_codes, v_codes}, *scales[2] = {k_scales, v_scales};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = xs[i]->data;
    for (int j = 0; j < 3; ++j) a.xs[i][j] = xs[i]->strides[j];
    a.codes[i] = static_cast<int8_t*>(codes[i]->data);
    a.scales[i] = static_cast<float*>(scales[i]->data);
  }
  a.table = static_cast<const int32_t*>(table->data);
  a.table_stride = c.table_stride;
  a.starts = starts->data;
  a.starts_dt = starts->dtype;
  a.starts_st = row_stride(starts);
  if (counts) {
    a.counts = counts->data;
    a.counts_dt = counts->dtype;
    a.counts_st = row_stride(counts);
  }
  a.pages = c.pages;
  a.columns = c.columns;
  a.T = static_cast<int>(T);
  a.Hk = static_cast<int>(c.heads);
  a.D = static_cast<int>(c.D);
  a.block = static_cast<int>(c.block);
  KK_TRY(require_ready());
  if (B * T * c.heads == 0) return KK_OK;
  // T rows starting anywhere in a page reach this many pages at most
  const int64_t reach = (T + c.block - 2) / c.block + 1;
  if (2 * reach > 65535) return set_error(KK_E_UNSUPPORTED, "%s: too many tokens in a call", who);
  const dim3 grid(static_cast<unsigned>(B), static_cast<unsigned>(c.heads), static_cast<unsigned>(2 * reach));
  const size_t lds = c.D * (c.block + 4);
  const bool wide = rows_aligned(k, 16) && rows_aligned(v, 16);
  auto launch = [&](auto kernel) {
    if (lds > 60000) KK_TRY(allow_large_lds(reinterpret_cast<const void*>(kernel)));
    KK_LAUNCH(kernel, grid, dim3(kAppendThreads), lds, ctx().stream, a);
    return check_launch("cache_append_kernel");
  };
  if (k->dtype == KK_F16) return wide ? launch(cache_append_kernel<__half, true>) : launch(cache_append_kernel<__half, false>);
  return wide ? launch(cache_append_kernel<float, true>) : launch(cache_append_kernel<float, false>);
}

int kk_cache_values(const kk_tensor* out_k, const kk_tensor* out_v, const kk_tensor* k_codes,
                    const kk_tensor* k_scales, const kk_tensor* v_codes, const kk_tensor* v_scales) {
  const char* who = "cache_values";
  CacheShape c;
  KK_TRY(check_codes(k_codes, k_scales, v_codes, v_scales, &c, who));
  const kk_tensor *outs[2] = {out_k, out_v}, *codes[2] = {k_codes, v_codes};
  const char* names[2] = {"out_k", "out_v"};
  for (int i = 0; i < 2; ++i) {
    KK_TRY(check_tensor(outs[i], names[i]));
    if (outs[i]->dtype != KK_F32 || outs[i]->rank != 4 || !is_contiguous(outs[i]) ||
        reinterpret_cast<uintptr_t>(outs[i]->data) % 16)
      return set_error(KK_E_ARG, "%s: %s must be f32 of four axes in one piece, 16-byte aligned", who, names[i]);
    for (int j = 0; j < 4; ++j)
      if (outs[i]->shape[j] != codes[i]->shape[j])
        return set_error(KK_E_ARG, "%s: %s must have the shape of its codes", who, names[i]);
  }
  KK_TRY(require_ready());
  const int64_t waves_a_page = c.block * c.D / 256, waves = c.pages * c.heads * waves_a_page;
  if (waves == 0) return KK_OK;
  const int64_t blocks = ceil_div(waves, 4 * kValuesEach);
  if (blocks > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many pages", who);
  KK_LAUNCH(cache_values_kernel, dim3(static_cast<unsigned>(blocks), 2), dim3(256), 0, ctx().stream,
            static_cast<const int8_t*>(k_codes->data), static_cast<const int8_t*>(v_codes->data),
            static_cast<const float*>(k_scales->data), static_cast<const float*>(v_scales->data),
            static_cast<float*>(out_k->data), static_cast<float*>(out_v->data), waves, waves_a_page);
  return check_launch("cache_values_kernel");
}

int kk_process_logits(const kk_tensor* out, const kk_tensor* logits, const kk_tensor* history,
                      const kk_tensor* history_lengths, const kk_tensor* repetition, const kk_tensor* presence,
                      const kk_tensor* frequency, const kk_tensor* bias, const kk_tensor* allowed) {
  const char* who = "process_logits";
  LogitArgs a{};
  KK_TRY(check_tensor(logits, "logits"));
  KK_TRY(check_tensor(out, "out"));
  if (logits->rank != 2 || !is_float(logits->dtype))
    return set_error(KK_E_ARG, "%s: logits must be [rows, vocabulary], f32 or f16", who);
  const int64_t B = logits->shape[0], V = logits->shape[1];
  KK_TRY(check_by_row(logits, "logits", B, V, &a.xs, who));
  if (out->dtype != KK_F32 || out->rank != 2 || out->shape[0] != B)
    return set_error(KK_E_ARG, "%s: out must be f32 of the shape of logits", who);
  KK_TRY(check_by_row(out, "out", B, V, &a.ys, who));
  KK_TRY(check_writable(out, "out", who));
  if (history) {
    KK_TRY(check_tensor(history, "history"));
    if (!is_index(history->dtype) || history->rank != 2 || history->shape[0] != B)
      return set_error(KK_E_ARG, "%s: history must be [rows, tokens], int32 or int64", who);
    a.L = history->shape[1];
    KK_TRY(check_by_row(history, "history", B, a.L, &a.hs, who));
    a.history = a.L > 0 ? history->data : nullptr;
    a.history_dt = history->dtype;
    if (history_lengths) {
      KK_TRY(check_per_row(history_lengths, "history_lengths", B, true, who));
      a.lengths = history_lengths->data;
      a.lengths_dt = history_lengths->dtype;
      a.lengths_st = row_stride(history_lengths);
    }
  } else if (history_lengths || repetition || presence || frequency) {
    return set_error(KK_E_ARG, "%s: penalties need the history", who);
  }
  const kk_tensor* per_row[3] = {repetition, presence, frequency};
  const char* names[3] = {"repetition", "presence", "frequency"};
  const float** values[3] = {&a.rep, &a.pres, &a.freq};
  int64_t* strides[3] = {&a.rep_st, &a.pres_st, &a.freq_st};
  for (int i = 0; i < 3; ++i) {
    if (!per_row[i]) continue;
    KK_TRY(check_per_row(per_row[i], names[i], B, false, who));
    *values[i] = static_cast<const float*>(per_row[i]->data);
    *strides[i] = row_stride(per_row[i]);
  }
  if (bias) {
    if (bias->dtype != KK_F32) return set_error(KK_E_ARG, "%s: bias must be f32", who);
    KK_TRY(check_by_row(bias, "bias", B, V, &a.bias_st, who));
    a.bias = static_cast<const float*>(bias->data);
  }
  if (allowed) {
    if (allowed->dtype != KK_I32) return set_error(KK_E_ARG, "%s: allowed must be int32 words of bits", who);
    KK_TRY(check_by_row(allowed, "allowed", B, ceil_div(V, 32), &a.allowed_st, who));
    a.allowed = static_cast<const int32_t*>(allowed->data);
  }
  a.x = logits->data;
  a.y = static_cast<float*>(out->data);
  a.V = V;
  KK_TRY(require_ready());
  if (B * V == 0) return KK_OK;
  const int64_t tiles = ceil_div(V, kLogitTile);
  if (B > 65535 || tiles > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many rows", who);
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(B));
  if (logits->dtype == KK_F16)
    KK_LAUNCH((process_logits_kernel<__half>), grid, dim3(kLogitThreads), 0, ctx().stream, a);
  else
    KK_LAUNCH((process_logits_kernel<float>), grid, dim3(kLogitThreads), 0, ctx().stream, a);
  return check_launch("process_logits_kernel");
}

}  // extern "C"
