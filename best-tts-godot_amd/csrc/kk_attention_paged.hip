// Attention of few queries over a paged cache of 8-bit codes: a step of single
// tokens, with the query heads that share a key head together.
#include "kk_attention.h"

namespace kk {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

// Eight codes as halves, exactly: a byte with its sign turned over is the low
// half of 1024 + 128 + code, from which a packed sum takes 1152.
__device__ __forceinline__ h8 codes_h8(uint32_t lo, uint32_t hi) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  uint32_t w[4];
  lo ^= 0x80808080u;
  hi ^= 0x80808080u;
  w[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x05010400u);
  w[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x05030402u);
  w[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x05010400u);
  w[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x05030402u);
  h8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const h2 v = __builtin_bit_cast(h2, w[i]) + off;
    r[2 * i] = v[0];
    r[2 * i + 1] = v[1];
  }
  return r;
}

constexpr int kFewThreads = 256;
constexpr int kFewWaves = kFewThreads / 64;

// out = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m), a wave its own
// steps of 64 tokens, on the matrix cores (v_mfma_f32_16x16x32_f16): bound by
// the codes' way from memory, so nothing is staged in LDS: each code is read
// once, straight into the registers of the lane that multiplies it, a step's
// values and the next step's keys (where there are registers for them) before
// the step's products.
//
// Scores are formed transposed, S^T = K Q^T, 16 tokens by 16 queries: a lane
// (n = l % 16, g = l / 16) holds a query's column, and with token 16 g + 4 a + i
// in row 4 g + i of tile a it holds tokens 16 g .. 16 g + 15 of the step: what
// the second product O^T = V^T P^T takes from it as they are, next to 16
// consecutive codes of V's rows.  A group of 16 tokens lies in one page, so
// its scales are one value a lane.
//
// Codes are exact in fp16.  fp16 queries are taken as they are, fp32 ones as
// the sum of two halves after a power of two that brings the row's largest to
// 2^14 (22 bits; smaller values keep 2^-38 of the largest).  Weights p times
// the page's scale, over a power of two r >= all scales so far, are rounded to
// fp16 (half a step of the output's type) or split the same way; 2^15 p <= 2^15
// keeps 24 bits above fp16's smallest value.
template <typename T, int KH, int NT>
__global__ void __launch_bounds__(kFewThreads, NT == 1 && KH < 4 ? 2 : 1)
    few_paged_kernel(QueryArgs a, PagedRows rows, Cut cut) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // halves of a query or weight
  constexpr int DT = 4 * KH;
  extern __shared__ float lds[];
  Unit u;
  if (!find_unit(rows, cut, &u)) return;
  const PagedArgs& p = rows.a;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = lane % 16, g = lane / 16;
  const int D = a.D, R = static_cast<int>(cut.rows);

  // the lane's queries: n + 16 nt, values 64 h + 16 g + 8 e + 0 .. 7 in slot 2 h + e
  h8 qf[NT][2 * KH][P];
  float cq[NT];
  int64_t qlo[NT], qhi[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = n + 16 * nt < R ? n + 16 * nt : R - 1;
    const int t = r / a.group, head = u.h * a.group + r % a.group;
    const Seen w = rows.seen(u.b, t);
    qlo[nt] = w.lo;
    qhi[nt] = w.hi;
    const T* q = static_cast<const T*>(a.q) + u.b * a.qs[0] + t * a.qs[1] + head * a.qs[2];
    T x[2 * KH][8];
#pragma unroll
    for (int s = 0; s < 2 * KH; ++s) {
      const int d = 64 * (s / 2) + 16 * g + 8 * (s % 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = d < D ? q[d + i] : T(0.0f);
    }
    cq[nt] = a.scale;
    if constexpr (P == 1) {
#pragma unroll
      for (int s = 0; s < 2 * KH; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[nt][s][0][i] = __builtin_bit_cast(_Float16, x[s][i]);
    } else {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < 2 * KH; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, __builtin_fabsf(x[s][i]));
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const int up = 14 + 127 - static_cast<int>(__float_as_uint(top) >> 23);
      cq[nt] = ldexpf(a.scale, -up);
#pragma unroll
      for (int s = 0; s < 2 * KH; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = ldexpf(x[s][i], up);
          const _Float16 hi = static_cast<_Float16>(y);
          qf[nt][s][0][i] = hi;
          qf[nt][s][P - 1][i] = static_cast<_Float16>(y - static_cast<float>(hi));
        }
    }
  }

  const int shift = __builtin_ctz(p.block);
  const int32_t* table = p.table + u.b * p.table_stride;
  // page of the 16 tokens from t on, -1 where there is none
  auto page_at = [&](int64_t t) -> int {
    const int64_t column = t >> shift;
    if (t >= u.hi || column >= p.columns) return -1;
    const int id = table[column];
    return id < p.pages ? id : -1;
  };
  const int64_t t_first = u.lo + wave * kStep;
  constexpr int kStride = kFewWaves * kStep;
  const int kg = n / 4;
  auto load_keys = [&](int64_t t0, int page, uint4 (&k)[4][KH]) {
    const int row = static_cast<int>((t0 + 16 * kg) & (p.block - 1)) + lane % 4;
    const int8_t* from = p.k + ((int64_t{page} * p.heads + u.h) * p.block + row) * D + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        k[i][h] = make_uint4(0, 0, 0, 0);
        if (page >= 0 && 64 * h + 16 * g < D) k[i][h] = *reinterpret_cast<const uint4*>(from + 4 * i * D + 64 * h);
      }
  };

  f4 acc[NT][DT];
  float m[NT], l[NT];
  int er = 27;  // r = 2^(er - 127)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -3.4028235e38f;
    l[nt] = 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[nt][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  constexpr bool kAhead = KH < 4;
  int pk = page_at(t_first + 16 * kg), pv = page_at(t_first + 16 * g);
  uint4 k[4][KH];
  if (kAhead && t_first < u.hi) load_keys(t_first, pk, k);
  int pk1 = page_at(t_first + kStride + 16 * kg), pv1 = page_at(t_first + kStride + 16 * g);
  for (int64_t t0 = t_first; t0 < u.hi; t0 += kStride) {
    uint4 k1[4][KH], v[DT];
    if (!kAhead) load_keys(t0, pk, k);
    const int vrow = static_cast<int>((t0 + 16 * g) & (p.block - 1));
    const int64_t at = int64_t{pv} * p.heads + u.h;
    const int8_t* from = p.v + (at * D + n) * p.block + vrow;
    float ks = 0.0f, vs = 0.0f;
    if (pv >= 0) {
      ks = p.k_scale[at];
      vs = p.v_scale[at];
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      v[i] = make_uint4(0, 0, 0, 0);
      if (pv >= 0 && 16 * i < D) v[i] = *reinterpret_cast<const uint4*>(from + 16 * i * p.block);
    }
    const bool more = t0 + kStride < u.hi;
    if (kAhead && more) load_keys(t0 + kStride, pk1, k1);
    const int pk2 = page_at(t0 + 2 * kStride + 16 * kg), pv2 = page_at(t0 + 2 * kStride + 16 * g);

    f4 s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const h8 k0 = codes_h8(k[i][h].x, k[i][h].y), k1 = codes_h8(k[i][h].z, k[i][h].w);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = P - 1; e >= 0; --e) {
            s[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[nt][2 * h][e], s[nt][i], 0, 0, 0);
            s[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[nt][2 * h + 1][e], s[nt][i], 0, 0, 0);
          }
      }

    // the scales' power of two: the same in all lanes
    const uint32_t vbits = __float_as_uint(__builtin_fabsf(vs));
    const bool finite = vbits < 0x7f800000u;
    int e1 = finite ? static_cast<int>(vbits >> 23) + 1 : 0;
    e1 = e1 > 254 ? 254 : e1;
    float keep_r = 1.0f;
    if (__any(e1 > er)) {
      for (int off = 16; off < 64; off <<= 1) {
        const int o = __shfl_xor(e1, off, 64);
        e1 = o > e1 ? o : e1;
      }
      const int up = e1 > er ? e1 : er;
      keep_r = ldexpf(1.0f, er - up);
      er = up;
    }
    const float vw = vs * __uint_as_float(static_cast<uint32_t>(127 + 15 + 127 - er) << 23);

    h8 pf[NT][2][P];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float by = cq[nt] * ks;
      int64_t lo = qlo[nt] - (t0 + 16 * g), hi = qhi[nt] - (t0 + 16 * g);
      if (pv < 0) hi = 0;
      const int a0 = lo < 0 ? 0 : (lo > 16 ? 16 : static_cast<int>(lo));
      const int a1 = hi < 0 ? 0 : (hi > 16 ? 16 : static_cast<int>(hi));
      const bool whole = __all(a0 == 0 && a1 == 16 && finite);
      float x[16], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] = s[nt][j / 4][j % 4] * by;
        if (!whole) x[j] = j >= a0 && j < a1 ? x[j] : -INFINITY;
        top = fmaxf(top, x[j]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      top = fmaxf(top, m[nt]);
      if (__any(top > m[nt]) || keep_r != 1.0f) {
        const float keep = __builtin_amdgcn_exp2f(m[nt] - top);
        m[nt] = top;
        l[nt] *= keep;
        const float both = keep * keep_r;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][i][e] *= both;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float e = __builtin_amdgcn_exp2f(x[j] - m[nt]);
        l[nt] += e;
        float w = e * vw;
        if (!whole) w = j >= a0 && j < a1 ? w : 0.0f;  // (a scale that is not finite)
        const _Float16 hi16 = static_cast<_Float16>(w);
        pf[nt][j / 8][0][j % 8] = hi16;
        if constexpr (P == 2) pf[nt][j / 8][1][j % 8] = static_cast<_Float16>(w - static_cast<float>(hi16));
      }
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      if (16 * i >= D) continue;
      const h8 v0 = codes_h8(v[i].x, v[i].y), v1 = codes_h8(v[i].z, v[i].w);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = P - 1; e >= 0; --e) {
          acc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[nt][0][e], acc[nt][i], 0, 0, 0);
          acc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[nt][1][e], acc[nt][i], 0, 0, 0);
        }
    }
    if (kAhead && more) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < KH; ++h) k[i][h] = k1[i][h];
    }
    pk = pk1;
    pv = pv1;
    pk1 = pk2;
    pv1 = pv2;
  }

  // join the waves: m and l of a wave's queries, then the sums, in LDS
  const int pitch = D + 4;
  float* wm = lds;                        // [waves][R], then [R] the block's
  float* wl = wm + (kFewWaves + 1) * R;
  float* sums = wl + (kFewWaves + 1) * R;  // [waves][R][pitch]
  sums += (4 - (2 * (kFewWaves + 1) * R) % 4) % 4;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += __shfl_xor(l[nt], 16, 64);
    l[nt] += __shfl_xor(l[nt], 32, 64);
    const int r = n + 16 * nt;
    if (g == 0 && r < R) {
      wm[wave * R + r] = m[nt];
      wl[wave * R + r] = l[nt];
    }
  }
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = n + 16 * nt;
    if (r >= R) continue;
    float top = wm[r], sum = 0.0f;
    for (int w = 1; w < kFewWaves; ++w) top = fmaxf(top, wm[w * R + r]);
    for (int w = 0; w < kFewWaves; ++w) sum += wl[w * R + r] * exp2f(wm[w * R + r] - top);
    if (wave == 0 && g == 0) {
      wm[kFewWaves * R + r] = top;
      wl[kFewWaves * R + r] = sum;
    }
    const float by = ldexpf(exp2f(m[nt] - top), er - 127 - 15);
#pragma unroll
    for (int i = 0; i < DT; ++i)
      if (16 * i < D) *reinterpret_cast<f4*>(sums + (wave * R + r) * pitch + 16 * i + 4 * g) = acc[nt][i] * by;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * D; i += kFewThreads) {
    float* at = sums + (i / D) * pitch + i % D;
    float v = at[0];
    for (int w = 1; w < kFewWaves; ++w) v += at[w * R * pitch];
    at[0] = v;
  }
  __syncthreads();
  put_rows<T, kFewThreads>(a, cut, u, sums, pitch, wm + kFewWaves * R, wl + kFewWaves * R, sums + R * pitch);
}

template <typename T, int KH, int NT>
static int launch_few(const QueryArgs& a, const PagedRows& rows, int64_t queries) {
  const int64_t capacity = rows.a.columns * rows.a.block;
  const int64_t seen = rows.a.window ? rows.a.window + a.T - 1 : capacity;
  Cut cut;
  int64_t blocks;
  KK_TRY(plan_cut(a.B, rows.a.heads, queries, a.D, seen < capacity ? seen : capacity, 8, int64_t{8} * ctx().num_cus,
                  &cut, &blocks, "cache_attention"));
  // the waves' sums, or (once they are joined in the first) the chunks' weights
  const int R = static_cast<int>(queries);
  size_t floats = 2 * (kFewWaves + 1) * R + 4 + static_cast<size_t>(kFewWaves) * R * (a.D + 4);
  const size_t joined = 2 * (kFewWaves + 1) * R + 4 + static_cast<size_t>(R) * (a.D + 4 + kMaxChunks);
  floats = floats > joined ? floats : joined;
  const void* kernel = reinterpret_cast<const void*>(few_paged_kernel<T, KH, NT>);
  if (floats * 4 > 65536) KK_TRY(allow_large_lds(kernel));
  KK_LAUNCH((few_paged_kernel<T, KH, NT>), dim3(static_cast<unsigned>(blocks)), dim3(kFewThreads), floats * 4,
            ctx().stream, a, rows, cut);
  return check_launch("few_paged_kernel");
}

template <typename T, int NT>
static int launch_few(const QueryArgs& a, const PagedRows& rows, int64_t queries) {
  if (a.D <= 64) return launch_few<T, 1, NT>(a, rows, queries);
  if constexpr (NT == 1)
    if (a.D > 128) return launch_few<T, 4, 1>(a, rows, queries);
  return launch_few<T, 2, NT>(a, rows, queries);
}

bool few_paged_try(const QueryArgs& a, const PagedArgs& p, int dtype, int* status) {
  const int64_t queries = int64_t{a.T} * a.group;
  if (queries > (a.D > 128 ? 16 : 32)) return false;  // (two tiles of queries of 256 values pass the registers)
  const PagedRows rows{p, a.T, a.D};
  if (dtype == KK_F16)
    *status = queries > 16 ? launch_few<__half, 2>(a, rows, queries) : launch_few<__half, 1>(a, rows, queries);
  else
    *status = queries > 16 ? launch_few<float, 2>(a, rows, queries) : launch_few<float, 1>(a, rows, queries);
  return true;
}

}  // namespace kk
