// Attention of few queries over a paged cache of 8-bit codes: a step of single
// tokens, with the query heads that share a key head together.
#include "kk_attention.h"

namespace kk {

constexpr int kFewThreads = 256;
constexpr int kFewWaves = kFewThreads / 64;

// out = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m), a wave its own
// steps of 64 tokens, on the matrix cores (v_mfma_f32_16x16x32_f16): bound by
// the codes' way from memory.  A wave loads the next step's codes, 16 bytes a
// lane in the order of memory, while it works on a step, and hands them to the
// lanes that multiply them through a part of LDS that is its own (no barrier).
// 32 sequences of 16384 to 32768 tokens, 8 key heads of 128 values in pages of
// 64, 32 query heads: 314 us, 5.1 TB/s of 6.2 that a kernel reaches which only
// reads such pages (544 us where each lane loads the rows that it multiplies,
// every 16 bytes of them in another line).
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
// 2^14 (22 bits; smaller values keep 2^-38 of the largest).  Weights times
// their page's scale, over a power of two of the largest such product that the
// query has met (so that a page of large scale without weight takes no bits from
// the others), are split into two halves as well, also for fp16 queries (rounded to
// one, the output was 1.4 times as far off for the same time); 2^15 p <= 2^15 keeps
// 24 bits above fp16's smallest value.
template <typename T, int DT, int NT, bool EXACT>
__global__ void __launch_bounds__(kFewThreads, NT == 1 && EXACT ? 2 : 1)
    few_paged_kernel(QueryArgs a, PagedRows rows, Cut cut) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // halves of a query
  constexpr int PW = 2;                      // halves of a weight
  constexpr int KH = (DT + 3) / 4;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  Unit u;
  if (!find_unit(rows, cut, &u)) return;
  const PagedArgs& p = rows.a;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int n = lane % 16, g = lane / 16;
  const int C = EXACT ? DT : a.D / 16, D = 16 * C, R = static_cast<int>(cut.rows);

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
      for (int i = 0; i < 8; ++i) {
        const T v = q[(d < D ? d : 0) + i];
        x[s][i] = d < D ? v : T(0.0f);
      }
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

  // Chunks of 16 bytes of a step: DT x 64 of keys, row by row of D / 16, and as
  // many of values, row by row of 4; the lane loads those at 64 i + lane.  In LDS
  // a row's chunks are exchanged by a key of the row, so that eight lanes that
  // read or write together meet eight different places.
  const int shift = __builtin_ctz(p.block);
  const bool paired = C % 8 == 4, eight = C % 8 == 0;
  auto key_of = [&](int row) {
    return eight ? (row & 3) | (row >> 2 & 4) : paired ? (row >> 1 & 1) | (row >> 3 & 2) : 0;
  };
  const int size = 2 * 64 * D;
  const int tail = 2 * (kFewWaves + 1) * R * 4 + 15 & ~15;  // the waves' m and l come first
  char* mine = reinterpret_cast<char*>(lds) + tail + wave * size;
  int to_k[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    const int q = 64 * i + lane, row = q / C, chunk = q - row * C;
    to_k[i] = row * D + 16 * (chunk ^ key_of(row));
  }
  // the lane's group of 16 tokens and row among 16 of the values: in the order of memory
  const int vg = p.block == 16 ? lane / 16 : p.block == 32 ? lane / 32 * 2 + lane % 2 : lane % 4;
  const int vr = p.block == 16 ? lane % 16 : p.block == 32 ? lane % 32 / 2 : lane / 4;
  const int to_v = 64 * D + 64 * vr + 16 * (vg ^ (vr >> 1 & 3));
  const char* from_k = mine + (16 * (n / 4) + n % 4) * D;
  const int nkey = key_of(16 * (n / 4) + n % 4);
  const char* from_v = mine + 64 * D + 64 * n + 16 * (g ^ (n >> 1 & 3));

  const int32_t* table = p.table + u.b * p.table_stride;
  const int64_t t_first = u.lo + wave * kStep;
  constexpr int kStride = kFewWaves * kStep;
  // The table's entry for tokens t0 + 16 (lane % 4) on, as it stands (past the
  // table its last), and the page, -1 where there is none: apart, so that an
  // entry is waited for where its page is needed, a step later.
  auto entry_at = [&](int64_t t0) -> int {
    const int64_t column = (t0 + 16 * (lane % 4)) >> shift;
    return table[column < p.columns ? column : p.columns - 1];
  };
  auto page_of = [&](int64_t t0, int entry) -> int {
    const int64_t t = t0 + 16 * (lane % 4);
    return t < u.hi && t >> shift < p.columns && entry < p.pages ? entry : -1;
  };
  // Where there is no page, page 0 is read, and its tokens get no weight.
  u4 ck[DT], cv[DT];
  const int64_t page_bytes = int64_t{p.block} * D;
  auto load_k = [&](int64_t t0, int pages) {
    if (p.block >= 64) {
      const int page = __builtin_amdgcn_readfirstlane(pages < 0 ? 0 : pages);
      const int8_t* k = p.k + (int64_t{page} * p.heads + u.h) * page_bytes + static_cast<int>(t0 & (p.block - 1)) * D;
#pragma unroll
      for (int i = 0; i < DT; ++i)
        if (i < C) ck[i] = *reinterpret_cast<const u4*>(k + 1024 * i + 16 * lane);
    } else {
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        if (i >= C) continue;
        const int q = 64 * i + lane, of = q / D, page = __shfl(pages, of, 64);
        const int8_t* k = p.k + (int64_t{page < 0 ? 0 : page} * p.heads + u.h) * page_bytes +
                          static_cast<int>((t0 + 16 * of) & (p.block - 1)) * D + 16 * (q - of * D);
        ck[i] = *reinterpret_cast<const u4*>(k);
      }
    }
  };
  auto load_v = [&](int64_t t0, int pages) {
    const int page = __shfl(pages, vg, 64);
    const int8_t* v = p.v + (int64_t{page < 0 ? 0 : page} * p.heads + u.h) * page_bytes + vr * p.block +
                      static_cast<int>((t0 + 16 * vg) & (p.block - 1));
#pragma unroll
    for (int i = 0; i < DT; ++i)
      if (i < C) cv[i] = *reinterpret_cast<const u4*>(v + 16 * i * p.block);
  };

  f4 acc[NT][DT];
  float m[NT], l[NT];
  float mv[NT];  // log2 of the largest weight times page scale that the lane's query has met, kLeastSize below m at the least
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -3.4028235e38f;
    l[nt] = 0.0f;
    mv[nt] = -3.4028235e38f;
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[nt][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // In flight during a step: the codes and scales of the next, the pages of the
  // one after.  (All are waited for at once; a load given out at a step's
  // start and needed in it would add its whole way from memory to each step.)
  float ks1 = 0.0f, vs1 = 0.0f;
  auto load_scales = [&](int pages) {
    const int page = __shfl(pages, g, 64);
    const int64_t at = int64_t{page < 0 ? 0 : page} * p.heads + u.h;
    ks1 = p.k_scale[at];
    vs1 = p.v_scale[at];
  };
  int entry1 = entry_at(t_first + kStride), pages = page_of(t_first, entry_at(t_first));
  if (t_first < u.hi) {
    load_scales(pages);
    load_k(t_first, pages);
    load_v(t_first, pages);
  }
  for (int64_t t0 = t_first; t0 < u.hi; t0 += kStride) {
    const bool there = __shfl(pages, g, 64) >= 0;
    const float ks = ks1, vs = there ? vs1 : 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DT; ++i)
      if (i < C) {
        *reinterpret_cast<u4*>(mine + to_k[i]) = ck[i];
        *reinterpret_cast<u4*>(mine + to_v + 1024 * i) = cv[i];
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int pages1 = page_of(t0 + kStride, entry1);
    entry1 = entry_at(t0 + 2 * kStride);
    if (t0 + kStride < u.hi) {
      load_scales(pages1);
      load_k(t0 + kStride, pages1);
      load_v(t0 + kStride, pages1);
    }

    f4 s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (4 * h >= C) continue;
        const int chunk = 4 * h + g;  // (lanes past the row's end read another row's, against zeros of q)
        const u4 w = *reinterpret_cast<const u4*>(from_k + 4 * i * D + 16 * ((chunk < C ? chunk : 0) ^ nkey));
        const h8 k0 = codes_h8(w.x, w.y), k1 = codes_h8(w.z, w.w);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = P - 1; e >= 0; --e) {
            s[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[nt][2 * h][e], s[nt][i], 0, 0, 0);
            s[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[nt][2 * h + 1][e], s[nt][i], 0, 0, 0);
          }
      }

    const uint32_t vbits = __float_as_uint(__builtin_fabsf(vs));
    const bool finite = vbits < 0x7f800000u;
    // log2 of the scale, rounded up
    const float ev = finite && vbits ? static_cast<float>(static_cast<int>(vbits >> 23) - 126) : -INFINITY;

    h8 pf[NT][2][PW];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float by = cq[nt] * ks;
      int64_t lo = qlo[nt] - (t0 + 16 * g), hi = qhi[nt] - (t0 + 16 * g);
      if (!there) hi = 0;
      const int a0 = lo < 0 ? 0 : (lo > 16 ? 16 : static_cast<int>(lo));
      const int a1 = hi < 0 ? 0 : (hi > 16 ? 16 : static_cast<int>(hi));
      const bool whole = __all(a0 == 0 && a1 == 16 && finite);
      float x[16], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        x[j] = s[nt][j / 4][j % 4] * by;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = j >= a0 && j < a1 ? x[j] : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, x[j]);
      float sized = top + ev;
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      // m and mv are whole numbers, so that the sums are scaled by powers of two
      if (__any(top > m[nt] || sized > mv[nt])) {
        top = fmaxf(ceilf(top), m[nt]);
        sized = fmaxf(sized, __shfl_xor(sized, 16, 64));
        sized = fmaxf(sized, __shfl_xor(sized, 32, 64));
        const float most = fmaxf(fmaxf(ceilf(sized), top - kLeastSize), mv[nt]);
        const float keep = __builtin_amdgcn_exp2f(mv[nt] - most);
        l[nt] *= __builtin_amdgcn_exp2f(m[nt] - top);
        m[nt] = top;
        mv[nt] = most;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][i][e] *= keep;
      }
      const float vw = a1 <= a0 ? 0.0f : finite ? sized_by(vs, __builtin_amdgcn_exp2f(m[nt] - mv[nt] + 15.0f)) : vs;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] = __builtin_amdgcn_exp2f(x[j] - m[nt]);
        l[nt] += x[j];
        x[j] *= vw;
      }
      if (!whole) {  // (past a scale that is not finite)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = j >= a0 && j < a1 ? x[j] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float w = x[j];
        const _Float16 hi16 = static_cast<_Float16>(w);
        pf[nt][j / 8][0][j % 8] = hi16;
        pf[nt][j / 8][1][j % 8] = static_cast<_Float16>(w - static_cast<float>(hi16));
      }
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      if (16 * i >= D) continue;
      const u4 w = *reinterpret_cast<const u4*>(from_v + 1024 * i);
      const h8 v0 = codes_h8(w.x, w.y), v1 = codes_h8(w.z, w.w);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = PW - 1; e >= 0; --e) {
          acc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[nt][0][e], acc[nt][i], 0, 0, 0);
          acc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[nt][1][e], acc[nt][i], 0, 0, 0);
        }
    }
    pages = pages1;
  }

  // join the waves: m and l of a wave's queries, then the sums, in LDS
  const int pitch = D + 4;
  float* wm = lds;                        // [waves][R], then [R] the block's
  float* wl = wm + (kFewWaves + 1) * R;
  float* sums = reinterpret_cast<float*>(reinterpret_cast<char*>(lds) + tail);  // [waves][R][pitch]
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
    const float by = exp2f(mv[nt] - top - 15.0f);
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
  const int64_t slot = int64_t{R} * (D + 2);
  const Part part{u.b,  u.h, R, u.chunk, u.chunks, 0, cut.part + u.slot * slot, slot * cut.heads,
                  cut.arrived + u.b * cut.heads + u.h};
  put_rows<T, kFewThreads>(a, part, sums, pitch, wm + kFewWaves * R, wl + kFewWaves * R, sums + R * pitch);
}

template <typename T, int DT, int NT, bool EXACT>
static int launch_few(const QueryArgs& a, const PagedRows& rows, int64_t queries) {
  const int64_t capacity = rows.a.columns * rows.a.block;
  const int64_t seen = rows.a.window && rows.a.window < capacity ? rows.a.window + a.T - 1 : capacity;
  Cut cut;
  int64_t blocks;
  KK_TRY(plan_cut(a.B, rows.a.heads, queries, a.D, seen < capacity ? seen : capacity, 16, int64_t{4} * ctx().num_cus,
                  &cut, &blocks, "cache_attention"));
  // codes; then the waves' sums; then, beside the first's, the chunks' weights
  const int R = static_cast<int>(queries);
  const size_t codes = size_t{kFewWaves} * 2 * 64 * a.D, sums = size_t{kFewWaves} * R * (a.D + 4) * 4;
  const size_t joined = static_cast<size_t>(R) * (a.D + 4 + 2 * kMaxChunks) * 4;
  size_t bytes = codes > sums ? codes : sums;
  bytes = (2 * (kFewWaves + 1) * R * 4 + 15) / 16 * 16 + (bytes > joined ? bytes : joined);
  const void* kernel = reinterpret_cast<const void*>(few_paged_kernel<T, DT, NT, EXACT>);
  if (bytes > 65536) KK_TRY(allow_large_lds(kernel));
  KK_LAUNCH((few_paged_kernel<T, DT, NT, EXACT>), dim3(static_cast<unsigned>(blocks)), dim3(kFewThreads), bytes,
            ctx().stream, a, rows, cut);
  return check_launch("few_paged_kernel");
}

template <typename T, int NT>
static int launch_few(const QueryArgs& a, const PagedRows& rows, int64_t queries) {
  switch (a.D) {
    case 64: return launch_few<T, 4, NT, true>(a, rows, queries);
    case 96: return launch_few<T, 6, NT, true>(a, rows, queries);
    case 128: return launch_few<T, 8, NT, true>(a, rows, queries);
  }
  return launch_few<T, 8, NT, false>(a, rows, queries);
}

bool few_paged_try(const QueryArgs& a, const PagedArgs& p, int dtype, int* status) {
  const int64_t queries = int64_t{a.T} * a.group;
  if (p.pages < 1 || p.columns < 1 || a.D > 128 || queries > 32) return false;
  const PagedRows rows{p, a.T, a.D};
  if (dtype == KK_F16)
    *status = queries > 16 ? launch_few<__half, 2>(a, rows, queries) : launch_few<__half, 1>(a, rows, queries);
  else
    *status = queries > 16 ? launch_few<float, 2>(a, rows, queries) : launch_few<float, 1>(a, rows, queries);
  return true;
}

}  // namespace kk
