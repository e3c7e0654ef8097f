// Attention of few queries over a paged cache of 4-bit codes: a step of single
// tokens, with the query heads that share a key head together.
#include "kk_attention4.h"

namespace kk {

constexpr int kFew4Threads = 256;
constexpr int kFew4Waves = kFew4Threads / 64;

// find_unit for more sequences than a wave has lanes, by all threads: each a run of
// sequences (512 sequences of up to 500 tokens, 8 key heads of 128: 139 us where each
// wave goes through them 64 at a time, 101 here).
__device__ __forceinline__ bool find_unit_by_block(const Paged4Rows& rows, const Cut& cut, Unit* u, float* lds) {
  int64_t* const sums = reinterpret_cast<int64_t*>(lds);  // [2][waves]
  Unit* const found = reinterpret_cast<Unit*>(sums + 2 * kFew4Waves);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t id = blockIdx.x / cut.heads, each = ceil_div(cut.B, kFew4Threads);
  const int64_t b0 = threadIdx.x * each, b1 = b0 + each < cut.B ? b0 + each : cut.B;
  auto steps_of = [&](int64_t b) -> int64_t {
    const Seen s = rows.span(b);
    return ceil_div(s.hi - (s.lo / kStep) * kStep, kStep);
  };
  int64_t total = 0;
  for (int64_t b = b0; b < b1; ++b) total += steps_of(b);
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  if (lane == 0) sums[wave] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kFew4Waves; ++w) total += sums[w];
  const int64_t c = chunk_size(total, cut.units, cut.most, cut.least);
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += chunk_count(steps_of(b), c);
  int64_t upto = mine;
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t o = __shfl_up(upto, off, 64);
    if (lane >= off) upto += o;
  }
  if (lane == 63) sums[kFew4Waves + wave] = upto;
  __syncthreads();
  int64_t all = 0;
  for (int w = 0; w < kFew4Waves; ++w) {
    if (w < wave) upto += sums[kFew4Waves + w];
    all += sums[kFew4Waves + w];
  }
  if (id >= all) return false;
  if (id < upto && id >= upto - mine) {
    int64_t first = upto - mine, b = b0, n = steps_of(b);
    for (; id >= first + chunk_count(n, c); n = steps_of(b)) {
      first += chunk_count(n, c);
      ++b;
    }
    const Seen s = rows.span(b);
    const int64_t size = chunk_steps(n, c) * kStep, lo = (s.lo / kStep) * kStep + (id - first) * size;
    found->b = b;
    found->chunks = static_cast<int>(chunk_count(n, c));
    found->chunk = static_cast<int>(id - first);
    found->slot = first * cut.heads;
    found->lo = lo;
    found->hi = lo + size < s.hi ? lo + size : s.hi;
  }
  __syncthreads();
  u->h = static_cast<int>(blockIdx.x % cut.heads);
  u->b = uniform(found->b);
  u->chunks = static_cast<int>(uniform(found->chunks));
  u->chunk = static_cast<int>(uniform(found->chunk));
  u->slot = uniform(found->slot) + u->h;
  u->lo = uniform(found->lo);
  u->hi = uniform(found->hi);
  __syncthreads();
  return true;
}

// out = sum_j 2^(x_j - r) (step_j code_j + low_j) / sum_j 2^(x_j - r), x_j = c (step_j q . code_j + low_j sum(q)):
// a wave its own steps of 64 tokens, on the matrix cores (v_mfma_f32_16x16x32_f16),
// codes straight from memory to the registers that multiply them (codes4).  Bound by the
// codes' way from memory and, near it, by the vector units: 32 sequences of up to 32768
// tokens, 8 key heads of 128 (855 MB), 32 query heads in fp16: 168 us, 5.1 TB/s.
//
// Scores are formed transposed, S^T = K Q^T, 16 tokens by 16 queries: a lane
// (n = l % 16, g = l / 16) holds a query's column, and with token 16 g + 4 i + e in row
// 4 g + e of tile i it holds the tokens 16 g .. 16 g + 15 of the step: what the second
// product O^T = V^T P^T takes from it as they are, next to 16 consecutive codes of
// V's rows, and those whose scales the 16 lanes of its row have loaded, one each,
// which a DPP move hands to all of them.  A group of 16 tokens lies in one page.
//
// A lane's word of keys is one fragment: values d and d + D / 2 of four d.  Values'
// rows d and d + D / 2 are fragments of their own.  Queries are brought to 2^14 by a
// power of two for each row; fp32 ones are the sum of two halves (22 bits).  Weights times
// their value's step, beside 2^r, are the sum of two halves also for fp16 queries (in
// one, the output is 1.4 times as far off).
template <typename T, int W, int NT, bool BIG>
__global__ void __launch_bounds__(kFew4Threads, NT * W * sizeof(T) <= 28 ? 2 : 1) few_paged4_kernel(QueryArgs a, Paged4Rows rows, Cut cut) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // halves of a query
  constexpr int D = 32 * W, HALF = D / 2;
  constexpr bool CENTRE = P == 2;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  Unit u;
  if (cut.B > 64 ? !find_unit_by_block(rows, cut, &u, lds) : !find_unit(rows, cut, &u)) return;
  const PagedArgs& p = rows.a;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int n = lane % 16, g = lane / 16, R = static_cast<int>(cut.rows);

  // the lane's queries n + 16 nt: of fragment j, values 4 (W g + j) + {0, 2, 1, 3}, and those + HALF
  h8 qf[NT][W][P];
  float cq[NT], sum[NT];
  int64_t qlo[NT], qhi[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = n + 16 * nt < R ? n + 16 * nt : R - 1;
    const int t = row / a.group, head = u.h * a.group + row % a.group;
    const Seen w = rows.seen(u.b, t);
    qlo[nt] = w.lo;
    qhi[nt] = w.hi;
    const T* q = static_cast<const T*>(a.q) + u.b * a.qs[0] + t * a.qs[1] + head * a.qs[2];
    struct __attribute__((packed, aligned(sizeof(T)))) Four {
      T v[4];
    };
    const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
    float x[W][8], top = 0.0f, all = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Four f = *reinterpret_cast<const Four*>(q + s * HALF + 4 * (W * g + j));
        const int order[4] = {0, 2, 1, 3};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = to_f32(f.v[order[e]]) * sign;
          x[j][4 * s + e] = v;
          top = fmaxf(top, __builtin_fabsf(v));
        }
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const int up = 13 + 127 - static_cast<int>(__float_as_uint(top) >> 23);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = ldexpf(x[j][e], up);
        all += y;
        const _Float16 hi = static_cast<_Float16>(y);
        qf[nt][j][0][e] = hi;
        if constexpr (P == 2) qf[nt][j][P - 1][e] = static_cast<_Float16>(y - static_cast<float>(hi));
      }
    all += __shfl_xor(all, 16, 64);
    all += __shfl_xor(all, 32, 64);
    // scores come out 2^(up - 18) too large
    sum[nt] = all * 0x1p-18f;
    cq[nt] = unscaled4(a.scale, 18 - up);
  }

  const int shift = __builtin_ctz(p.block);
  const int32_t* table = p.table + u.b * p.table_stride;
  const int64_t t_first = u.lo + wave * kStep, page_bytes = int64_t{p.block} * HALF;
  constexpr int kStride = kFew4Waves * kStep;
  // The table's entry for tokens t on, as it stands (past the table its last), and
  // the page, -1 where there is none: apart, so that an entry is waited for where its
  // page is needed, a step later.  BIG: a step's tokens lie in one page.
  auto entry_at = [&](int64_t t) -> int {
    const int64_t column = t >> shift;
    return table[column < p.columns ? column : p.columns - 1];
  };
  auto page_of = [&](int64_t t, int entry) -> int {
    const int page = t < u.hi && t >> shift < p.columns && entry < p.pages ? entry : -1;
    return BIG ? __builtin_amdgcn_readfirstlane(page) : page;
  };
  // of keys the lane's group of tokens is n / 4, of values and scales g; where
  // there is no page, page 0 is read, and its tokens get no weight
  const int tk = 16 * (n / 4) + n % 4, group_k = BIG ? 0 : 16 * (n / 4), group_g = BIG ? 0 : 16 * g;
  // (codes are read once, past the caches: 182 against 168 us for the case below)
  typedef uint32_t Words __attribute__((ext_vector_type(W), aligned(4)));
  Words ck[4];
  u4 cv[W];
  uint32_t ks1 = 0, vs1 = 0;
  // (of tokens t0 + i, within a page: all of them where BIG)
  auto in_page = [&](int64_t t0, int i) -> int {
    const int first = static_cast<int>(t0) & (p.block - 1);
    return BIG ? first + i : (first + i) & (p.block - 1);
  };
  auto load_k = [&](int64_t t0, int page_k, int page_g) {
    const int64_t head_k = int64_t{page_k < 0 ? 0 : page_k} * p.heads + u.h;
    const int64_t head_g = BIG ? head_k : int64_t{page_g < 0 ? 0 : page_g} * p.heads + u.h;
    const uint8_t* k = rows.k + head_k * page_bytes + static_cast<uint32_t>(in_page(t0, tk) * HALF + 4 * W * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) ck[i] = __builtin_nontemporal_load(reinterpret_cast<const Words*>(k + 4 * i * HALF));
    ks1 = rows.k_scale[head_g * p.block + static_cast<uint32_t>(in_page(t0, lane))];
  };
  auto load_v = [&](int64_t t0, int page_g) {
    const int64_t head = int64_t{page_g < 0 ? 0 : page_g} * p.heads + u.h;
    const uint8_t* v = rows.v + head * page_bytes + static_cast<uint32_t>(n * p.block + in_page(t0, 16 * g));
#pragma unroll
    for (int i = 0; i < W; ++i) cv[i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(v + 16 * i * p.block));
    vs1 = rows.v_scale[head * p.block + static_cast<uint32_t>(in_page(t0, lane))];
  };

  const float less = minus_one();
  f4 acc[NT][2 * W];  // rows d of the first half (even) and the second (odd)
  float r[NT], l[NT], lows[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    r[nt] = -3.4028235e38f;
    l[nt] = lows[nt] = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) acc[nt][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Keys of the next step are asked for once this step's are multiplied, values
  // likewise: each has the other's half of a step for its way.
  int entry_k = entry_at(t_first + group_k), entry_g = BIG ? entry_k : entry_at(t_first + group_g);
  int page_g = page_of(t_first + group_g, entry_g);
  if (t_first < u.hi) {
    load_k(t_first, BIG ? page_g : page_of(t_first + group_k, entry_k), page_g);
    load_v(t_first, page_g);
  }
  auto next_entries = [&](int64_t t) {
    entry_g = entry_at(t + group_g);
    entry_k = BIG ? entry_g : entry_at(t + group_k);
  };
  next_entries(t_first + kStride);
  for (int64_t t0 = t_first; t0 < u.hi; t0 += kStride) {
    f4 s[NT][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const Codes4 c = codes4<CENTRE>(ck[i][j]);
        const h8 k = halves8(c.low[0], c.low[1], c.high[0], c.high[1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = P - 1; e >= 0; --e) s[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[nt][j][e], s[nt][i], 0, 0, 0);
      }
    }
    const bool there = page_g >= 0;  // of the lane's own token, too: it is of group g
    const float kstep = there ? key_step(ks1) : 0.0f, klow = there ? base4<CENTRE>(ks1) : 0.0f;
    const float vstep = there ? low_half(vs1) : 0.0f, vlow = there ? base4<CENTRE>(vs1) : 0.0f;
    const int page1 = page_of(t0 + kStride + group_g, entry_g);
    if (t0 + kStride < u.hi) load_k(t0 + kStride, BIG ? page1 : page_of(t0 + kStride + group_k, entry_k), page1);
    next_entries(t0 + 2 * kStride);

    // log2 of the token's step, rounded up, and the largest of the wave's
    const uint32_t bits = __float_as_uint(vstep) & 0x7fffffffu;
    const float ev = bits ? static_cast<float>(static_cast<int>(bits >> 23) - 126) : -INFINITY;
    const float limit = fminf(kSlack4 - wave_max_dpp(ev), kFar4);
    const float vs = vstep * 256.0f;

    h8 pf[NT][2][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int64_t lo = qlo[nt] - (t0 + 16 * g), hi = there ? qhi[nt] - (t0 + 16 * g) : 0;
      const int a0 = lo < 0 ? 0 : (lo > 16 ? 16 : static_cast<int>(lo));
      const int a1 = hi < 0 ? 0 : (hi > 16 ? 16 : static_cast<int>(hi));
      const bool whole = __all(a0 == 0 && a1 == 16);
      float x[16], top = -INFINITY;
      each<0, 16>([&](auto c) {
        constexpr int J = decltype(c)::value;
        x[J] = __builtin_fmaf(of_row<J>(kstep), s[nt][J / 4][J % 4], of_row<J>(klow) * sum[nt]);
      });
      if (!whole) {
        int first = a0, past = a1;
        asm volatile("" : "+v"(first), "+v"(past));  // (a branch: its tests are for few steps)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = j >= first && j < past ? x[j] : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 16; j += 2) top = fmaxf(fmaxf(top, x[j]), x[j + 1]);
      top *= cq[nt];
      if (__any(top > r[nt] + limit)) {
        float sized = -INFINITY;
        each<0, 16>([&](auto c) {
          constexpr int J = decltype(c)::value;
          sized = fmaxf(sized, __builtin_fmaf(x[J], cq[nt], of_row<J>(ev)));
        });
        sized = fmaxf(ceilf(sized), ceilf(top) - kLeast4);
        sized = fmaxf(sized, __shfl_xor(sized, 16, 64));
        sized = fmaxf(fmaxf(sized, __shfl_xor(sized, 32, 64)), r[nt]);
        const float keep = __builtin_amdgcn_exp2f(r[nt] - sized);
        r[nt] = sized;
        l[nt] *= keep;
        lows[nt] *= keep;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) acc[nt][i] *= keep;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], cq[nt], -r[nt]));
        l[nt] += x[j];
      }
      if (whole) {
        lows[nt] = dot_row(lows[nt], vlow, x);
        each<0, 16>([&](auto c) {
          constexpr int J = decltype(c)::value;
          x[J] *= of_row<J>(vs);
        });
      } else {  // (past scales that are not finite)
        int first = a0, past = a1;
        asm volatile("" : "+v"(first), "+v"(past));
        each<0, 16>([&](auto c) {
          constexpr int J = decltype(c)::value;
          const bool sees = J >= first && J < past;
          const float low = of_row<J>(vlow), by = of_row<J>(vs);
          lows[nt] = __builtin_fmaf(sees ? low : 0.0f, x[J], lows[nt]);
          x[J] = sees ? x[J] * by : 0.0f;
        });
      }
#pragma unroll
      for (int j = 0; j < 16; j += 2) {  // tokens j / 4 * 4 + {0, 2} and {1, 3}
        const int i = j / 4 * 4 + j % 4 / 2;
        h2 w0, w1;
        split4(x[i], x[i + 2], less, &w0, &w1);
        pf[nt][j / 8][0][j % 8] = w0[0];
        pf[nt][j / 8][0][j % 8 + 1] = w0[1];
        pf[nt][j / 8][1][j % 8] = w1[0];
        pf[nt][j / 8][1][j % 8 + 1] = w1[1];
      }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Codes4 c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = codes4<CENTRE>(cv[i][j]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // tokens 16 g + 8 h on
        const h8 low = halves8(c[2 * h].low[0], c[2 * h].low[1], c[2 * h + 1].low[0], c[2 * h + 1].low[1]);
        const h8 high = halves8(c[2 * h].high[0], c[2 * h].high[1], c[2 * h + 1].high[0], c[2 * h + 1].high[1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 1; e >= 0; --e) {
            acc[nt][2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(low, pf[nt][h][e], acc[nt][2 * i], 0, 0, 0);
            acc[nt][2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, pf[nt][h][e], acc[nt][2 * i + 1], 0, 0, 0);
          }
      }
    }
    if (t0 + kStride < u.hi) load_v(t0 + kStride, page1);
    page_g = page1;
  }

  // join the waves: r and l of a wave's queries, then the sums, in LDS
  constexpr int pitch = D + 4;
  float* wm = lds;  // [waves][R], then [R] the block's
  float* wl = wm + (kFew4Waves + 1) * R;
  const int tail = (2 * (kFew4Waves + 1) * R * 4 + 15) & ~15;
  float* sums = reinterpret_cast<float*>(reinterpret_cast<char*>(lds) + tail);  // [waves][R][pitch]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += __shfl_xor(l[nt], 16, 64);
    l[nt] += __shfl_xor(l[nt], 32, 64);
    lows[nt] += __shfl_xor(lows[nt], 16, 64);
    lows[nt] += __shfl_xor(lows[nt], 32, 64);
    const int row = n + 16 * nt;
    if (g == 0 && row < R) {
      wm[wave * R + row] = r[nt];
      wl[wave * R + row] = l[nt];
    }
  }
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = n + 16 * nt;
    if (row >= R) continue;
    float top = wm[row], all = 0.0f;
    for (int w = 1; w < kFew4Waves; ++w) top = fmaxf(top, wm[w * R + row]);
    for (int w = 0; w < kFew4Waves; ++w) all += wl[w * R + row] * exp2f(wm[w * R + row] - top);
    if (wave == 0 && g == 0) {
      wm[kFew4Waves * R + row] = top;
      wl[kFew4Waves * R + row] = all;
    }
    // (codes were 2^-18 as large, weights 2^8 times)
    const float by = exp2f(r[nt] - top), low = lows[nt] * by;
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f4*>(sums + (wave * R + row) * pitch + h * HALF + 16 * i + 4 * g) =
            acc[nt][2 * i + h] * (by * 0x1p10f) + low;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * D; i += kFew4Threads) {
    float* at = sums + (i / D) * pitch + i % D;
    float v = at[0];
    for (int w = 1; w < kFew4Waves; ++w) v += at[w * R * pitch];
    at[0] = v;
  }
  __syncthreads();
  const int64_t slot = int64_t{R} * (D + 2);
  const Part part{u.b,  u.h, R, u.chunk, u.chunks, 0, cut.part + u.slot * slot, slot * cut.heads,
                  cut.arrived + u.b * cut.heads + u.h};
  put_rows<T, kFew4Threads>(a, part, sums, pitch, wm + kFew4Waves * R, wl + kFew4Waves * R, sums + R * pitch);
}

template <typename T, int W, int NT, bool BIG>
static int launch_few4(const QueryArgs& a, const Paged4Rows& rows, int64_t queries) {
  const int64_t capacity = rows.a.columns * rows.a.block;
  const int64_t seen = rows.a.window && rows.a.window < capacity ? rows.a.window + a.T - 1 : capacity;
  Cut cut;
  int64_t blocks;
  KK_TRY(plan_cut(a.B, rows.a.heads, queries, a.D, seen < capacity ? seen : capacity, 16, int64_t{8} * ctx().num_cus,
                  &cut, &blocks, "cache4_attention"));
  // the waves' sums; then, beside the first's, the chunks' weights
  const int R = static_cast<int>(queries);
  const size_t sums = size_t{kFew4Waves} * R * (a.D + 4) * 4;
  const size_t joined = static_cast<size_t>(R) * (a.D + 4 + 2 * kMaxChunks) * 4;
  const size_t bytes = (2 * (kFew4Waves + 1) * R * 4 + 15) / 16 * 16 + (sums > joined ? sums : joined);
  if (bytes > 65536) KK_TRY(allow_large_lds(reinterpret_cast<const void*>(few_paged4_kernel<T, W, NT, BIG>)));
  KK_LAUNCH((few_paged4_kernel<T, W, NT, BIG>), dim3(static_cast<unsigned>(blocks)), dim3(kFew4Threads), bytes, ctx().stream, a,
            rows, cut);
  return check_launch("few_paged4_kernel");
}

template <typename T, int W, int NT>
static int launch_few4(const QueryArgs& a, const Paged4Rows& rows, int64_t queries) {
  return rows.a.block >= kStep ? launch_few4<T, W, NT, true>(a, rows, queries)
                               : launch_few4<T, W, NT, false>(a, rows, queries);
}

template <typename T, int NT>
static int launch_few4(const QueryArgs& a, const Paged4Rows& rows, int64_t queries) {
  switch (a.D) {
    case 32: return launch_few4<T, 1, NT>(a, rows, queries);
    case 64: return launch_few4<T, 2, NT>(a, rows, queries);
    case 96: return launch_few4<T, 3, NT>(a, rows, queries);
    case 128: return launch_few4<T, 4, NT>(a, rows, queries);
  }
  if constexpr (NT == 1) switch (a.D) {
    case 160: return launch_few4<T, 5, NT>(a, rows, queries);
    case 192: return launch_few4<T, 6, NT>(a, rows, queries);
    case 224: return launch_few4<T, 7, NT>(a, rows, queries);
    case 256: return launch_few4<T, 8, NT>(a, rows, queries);
  }
  return set_error(KK_E_UNSUPPORTED, "cache4_attention: heads of %d values", a.D);
}

bool few_paged4_try(const QueryArgs& a, const Paged4Rows& rows, int dtype, int* status) {
  const int64_t queries = int64_t{a.T} * a.group;
  if (rows.a.pages < 1 || rows.a.columns < 1 || queries > (a.D > 128 ? 16 : 32)) return false;
  if (dtype == KK_F16)
    *status = queries > 16 ? launch_few4<__half, 2>(a, rows, queries) : launch_few4<__half, 1>(a, rows, queries);
  else
    *status = queries > 16 ? launch_few4<float, 2>(a, rows, queries) : launch_few4<float, 1>(a, rows, queries);
  return true;
}

}  // namespace kk
