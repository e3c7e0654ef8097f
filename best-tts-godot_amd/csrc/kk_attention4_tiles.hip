// Attention of many queries (a chunk of new tokens) over a paged cache of 4-bit
// codes.
#include "kk_attention4.h"

namespace kk {

constexpr int kLeastTokens4 = 256;  // of a block that shares them

// The same sums as those of few queries, on v_mfma_f32_32x32x16_f16: 32 queries a
// wave, a step of SUB times 32 tokens (64 where the registers hold them), scores
// transposed.  A lane (n = l %
// 32, h = l / 32) holds a query's column, and with token 16 h + 4 b + c of 32 in row 8 b +
// 4 h + c it holds 16 tokens next to each other, whose scales the lanes of its rows
// of 16 have loaded, one each.  A wave reads codes from the caches straight into
// the registers that multiply them (its three neighbours read the same ones):
// nothing goes through LDS, and no wave waits for another.  Bound by the vector units
// (codes, exponentials, weights to halves) beside the products: 2 x 1531 queries of 32
// heads of 128 over up to 4099 tokens in 291 us, 400 TFLOP/s of fp16.
//
// Keys' lowest values (beside fp32 queries: their middles, in two halves and, past
// 2^15, 16 times a third, since a step times 8 passes fp16's range) times the query's
// sum, in three halves, are added by a product of their own.  Queries, codes and
// weights as there: in one half a weight (251 us for the queries above) outputs are up
// to 13 times as far off as their own rounding to fp16.
//
// SHARE: cut.row_waves waves (4, 2 or 1: as many as have queries) share the tokens
// with the others, which have the same queries; the first of them add all up in LDS.
template <typename T, int W, int SUB, bool BIG, int WAVES, bool SHARE>
__global__ void __launch_bounds__(64 * WAVES, W <= 4 ? 2 : 1)
    tile_paged4_kernel(QueryArgs a, Paged4Rows rows, TileCut cut) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // halves of a query
  constexpr bool CENTRE = P == 2;
  constexpr int DOWN = CENTRE ? 11 : 8;  // (16 times a sum of 256 values below 2^14 stays a half)
  constexpr int D = 32 * W, HALF = D / 2, KF = 2 * W, RT = (W + 1) / 2, kTokens4 = 32 * SUB;
  const int lane = threadIdx.x % 64, row_waves = SHARE ? cut.row_waves : WAVES, sharers = WAVES / row_waves;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) % row_waves;
  const int which = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) / row_waves;
  const int n = lane % 32, hf = lane / 32;
  const PagedArgs& p = rows.a;
  // neighbouring blocks of an XCD share keys and values; the longest rows first
  const uint3 at = xcd_tile();  // (split, tile, sequence and head)
  const int tile = cut.tiles - 1 - static_cast<int>(at.y), heads = p.heads;
  const int64_t b = at.z / heads, first = static_cast<int64_t>(tile) * kTileRows;
  const int head = at.z % heads;
  const int count = static_cast<int>(cut.rows - first < kTileRows ? cut.rows - first : kTileRows);

  // the tokens that any of the block's queries sees, and its share of them
  int64_t lo = rows.seen(b, first / a.group).lo, hi = 0;
  {
    int64_t t1 = (first + count - 1) / a.group;
    const int64_t there = rows.count(b);
    t1 = t1 < there ? t1 : there - 1;
    if (t1 >= first / a.group) hi = rows.seen(b, t1).hi;
  }
  lo = lo / kTokens4 * kTokens4;
  const int64_t steps = hi > lo ? ceil_div(hi - lo, kTokens4) : 0;
  int64_t share = ceil_div(steps, cut.splits);
  share = share < kLeastTokens4 / kTokens4 ? kLeastTokens4 / kTokens4 : share;
  const int chunks = steps <= share ? 1 : static_cast<int>(ceil_div(steps, share));
  const int chunk = static_cast<int>(at.x);
  if (chunk >= chunks) return;
  lo = uniform(lo + chunk * share * kTokens4);
  hi = uniform(chunk + 1 < chunks ? lo + share * kTokens4 : hi);
  if constexpr (SHARE) {
    const int64_t each = ceil_div(ceil_div(hi - lo, kTokens4), sharers) * kTokens4;
    lo += which * each;
    hi = lo + each < hi ? lo + each : hi;
  }

  // the lane's query: of fragment j, values 8 W hf + 4 j + {0, 2, 1, 3}, and those + HALF
  const int row = wave * 32 + n < count ? wave * 32 + n : count - 1;
  const int64_t qt = (first + row) / a.group;
  const Seen qs = rows.seen(b, qt);
  h8 qf[KF][P], sum_f = {};
  float cq;
  {
    const int qhead = head * a.group + static_cast<int>((first + row) % a.group);
    const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + qt * a.qs[1] + qhead * a.qs[2];
    struct __attribute__((packed, aligned(sizeof(T)))) Four {
      T v[4];
    };
    const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
    float x[KF][8], top = 0.0f, all = 0.0f;
#pragma unroll
    for (int j = 0; j < KF; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Four f = *reinterpret_cast<const Four*>(q + s * HALF + 8 * W * hf + 4 * j);
        const int order[4] = {0, 2, 1, 3};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][4 * s + e] = to_f32(f.v[order[e]]) * sign;
          top = fmaxf(top, __builtin_fabsf(x[j][4 * s + e]));
        }
      }
    top = max_halves(top);
    const int up = 13 + 127 - static_cast<int>(__float_as_uint(top) >> 23);
#pragma unroll
    for (int j = 0; j < KF; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = ldexpf(x[j][e], up);
        all += y;
        const _Float16 top16 = static_cast<_Float16>(y);
        qf[j][0][e] = top16;
        if constexpr (P == 2) qf[j][P - 1][e] = static_cast<_Float16>(y - static_cast<float>(top16));
      }
    // scores come out 2^(up - DOWN) too large (codes are 2^-18 as large, steps 2^(18 - DOWN) times)
    all = sum_halves(all) * (CENTRE ? 0x1p-11f : 0x1p-8f);
    cq = unscaled4(a.scale, DOWN - up);
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      const _Float16 part = static_cast<_Float16>(all);
      sum_f[e] = hf ? static_cast<_Float16>(0.0f) : part;
      if (CENTRE && e < 2) sum_f[3 + e] = sum_f[e];
      if (CENTRE) sum_f[5 + e] = sum_f[e] * static_cast<_Float16>(16.0f);
      all -= static_cast<float>(part);
    }
  }

  // what the wave's queries see: some of [from, upto), all of [all_from, all_upto)
  int64_t from = qs.lo, upto = qs.hi, all_from = qs.lo, all_upto = qs.hi;
  for (int off = 1; off < 32; off <<= 1) {
    auto least = [&](int64_t v) { const int64_t o = __shfl_xor(v, off, 64); return o < v ? o : v; };
    auto most = [&](int64_t v) { const int64_t o = __shfl_xor(v, off, 64); return o > v ? o : v; };
    from = least(from);
    upto = most(upto);
    all_from = most(all_from);
    all_upto = least(all_upto);
  }
  from = uniform(from);
  upto = uniform(upto);
  all_from = uniform(all_from);
  all_upto = uniform(all_upto);
  if (wave * 32 >= count) upto = 0;
  const int64_t begin = lo > from / kTokens4 * kTokens4 ? lo : from / kTokens4 * kTokens4;
  const int64_t end = hi < upto ? hi : upto;

  const int shift = __builtin_ctz(p.block);
  const int32_t* table = p.table + b * p.table_stride;
  const int64_t page_bytes = int64_t{p.block} * HALF;
  const int group_k = n >> 2 & 1;                       // of 16 tokens, of the lane's key row
  const int tk = 16 * group_k + 4 * (n >> 3) + (n & 3);  // its token of 32
  const int ts = 16 * hf + n % 16;                       // the token whose scales it loads
  // the pages of a step: of keys' groups, of values' and scales'; -1 where there is none
  auto page_at = [&](int64_t t) -> int {
    const int64_t column = t >> shift;
    const int entry = table[column < p.columns ? column : p.columns - 1];
    return t < hi && column < p.columns && entry < p.pages ? entry : -1;
  };
  struct Words {
    uint32_t w[KF];
  };
  Words ck[SUB];
  u4 cv[SUB][RT];
  uint32_t ks1[SUB], kl1[SUB], vs1[SUB];
  int pk[SUB], pg[SUB];  // (BIG: one page for all)
  auto find_pages = [&](int64_t t0) {
    if constexpr (BIG) {
      pk[0] = __builtin_amdgcn_readfirstlane(page_at(t0));
#pragma unroll
      for (int s = 0; s < SUB; ++s) pg[s] = pk[s] = pk[0];
    } else {
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        pk[s] = page_at(t0 + 32 * s + 16 * group_k);
        pg[s] = page_at(t0 + 32 * s + 16 * hf);
      }
    }
  };
  // (where there is no page, page 0 is read, and its tokens get no weight)
  auto load_k = [&](int64_t t0) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int in_page = static_cast<int>((t0 + 32 * s) & (p.block - 1));
      const int64_t head_k = int64_t{pk[s] < 0 ? 0 : pk[s]} * heads + head, head_g = int64_t{pg[s] < 0 ? 0 : pg[s]} * heads + head;
      const int at_k = BIG ? in_page + tk : static_cast<int>((t0 + 32 * s + tk) & (p.block - 1));
      const int at_g = BIG ? in_page + ts : static_cast<int>((t0 + 32 * s + ts) & (p.block - 1));
      ck[s] = *reinterpret_cast<const Words*>(rows.k + head_k * page_bytes + (at_k * HALF + 8 * W * hf));
      kl1[s] = rows.k_scale[head_k * p.block + at_k];
      ks1[s] = rows.k_scale[head_g * p.block + at_g];
    }
  };
  auto load_v = [&](int64_t t0) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int in_page = static_cast<int>((t0 + 32 * s) & (p.block - 1));
      const int64_t head_g = int64_t{pg[s] < 0 ? 0 : pg[s]} * heads + head;
      const int at_v = BIG ? in_page + 16 * hf : static_cast<int>((t0 + 32 * s + 16 * hf) & (p.block - 1));
      const int at_g = BIG ? in_page + ts : static_cast<int>((t0 + 32 * s + ts) & (p.block - 1));
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int d = 32 * i + n < HALF ? 32 * i + n : HALF - 1;  // (rows past the last: not put out)
        cv[s][i] = *reinterpret_cast<const u4*>(rows.v + head_g * page_bytes + (d * p.block + at_v));
      }
      vs1[s] = rows.v_scale[head_g * p.block + at_g];
    }
  };

  f16v acc[RT][2];
  float r = -3.4028235e38f, l = 0.0f, lows = 0.0f;
  const float less = minus_one();
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][0][e] = acc[i][1][e] = 0.0f;

  // of two waves that share vector units one comes first, so that they do not come to
  // multiply, and to wait for the vector units, at the same times (a wave's slot:
  // bits 0 to 3 of HW_ID; 310 against 291 us)
  if (__builtin_amdgcn_s_getreg(4 | 3 << 11) & 1) __builtin_amdgcn_s_setprio(1);
  if (begin < end) {
    find_pages(begin);
    load_k(begin);
    load_v(begin);
  }
  for (int64_t t0 = begin; t0 < end; t0 += kTokens4) {
    f16v s[SUB];
    float vs[SUB], low[SUB], ev[SUB], most = -INFINITY;
    bool there[SUB], none = false;
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[k][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < KF; ++j) {
        const Codes4 c = codes4<CENTRE>(ck[k].w[j]);
        const h8 kf = halves8(c.low[0], c.low[1], c.high[0], c.high[1]);
#pragma unroll
        for (int e = P - 1; e >= 0; --e) s[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[j][e], s[k], 0, 0, 0);
      }
      const float kstep = key_step(ks1[k]) * (CENTRE ? 0x1p7f : 0x1p10f);
      each<0, 16>([&](auto c) {
        constexpr int J = decltype(c)::value;
        s[k][J] *= of_row<J>(kstep);
      });
      // and keys' lowest values times the query's sum
      h8 base = {};
      if constexpr (CENTRE) {
        const float all = hf ? 0.0f : base4<true>(kl1[k]);
        const _Float16 far16 = static_cast<_Float16>(__builtin_fabsf(all) >= 0x1p15f ? all * 0x1p-4f : 0.0f);
        const float near = __builtin_fmaf(static_cast<float>(far16), -16.0f, all);
        const _Float16 most16 = static_cast<_Float16>(near);
        base[0] = base[1] = base[2] = most16;
        base[3] = base[4] = static_cast<_Float16>(near - static_cast<float>(most16));
        base[5] = base[6] = base[7] = far16;
      } else {
        const uint32_t low = hf ? 0u : (kl1[k] >> 16) * 0x10001u;
        base = halves8(low, low & 0xffffu, 0u, 0u);
      }
      s[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(base, sum_f, s[k], 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      there[k] = pg[k] >= 0;
      none = none || !there[k];
      const float vstep = there[k] ? low_half(vs1[k]) : 0.0f, vlow = there[k] ? base4<CENTRE>(vs1[k]) : 0.0f;
      const uint32_t bits = __float_as_uint(vstep) & 0x7fffffffu;
      ev[k] = bits ? static_cast<float>(static_cast<int>(bits >> 23) - 126) : -INFINITY;
      most = fmaxf(most, ev[k]);
      vs[k] = vstep * 256.0f;
      low[k] = vlow;
    }
    const float limit = fminf(kSlack4 - wave_max_dpp(most), kFar4);
    if (t0 + kTokens4 < end) {
      find_pages(t0 + kTokens4);
      load_k(t0 + kTokens4);
    }

    // what the lane's query sees of tokens 32 k + 16 hf + J: bit 16 k + J
    uint32_t seen = 0xffffffffu;
    const bool tested = t0 < all_from || t0 + kTokens4 > all_upto || __any(none);
    if (tested) {
#pragma unroll
      for (int k = 0; k < SUB; ++k) {
        const int64_t below = qs.lo - (t0 + 32 * k + 16 * hf), past = qs.hi - (t0 + 32 * k + 16 * hf);
        const int a0 = below < 0 ? 0 : below > 16 ? 16 : static_cast<int>(below);
        const int a1 = !there[k] || past < 0 ? 0 : past > 16 ? 16 : static_cast<int>(past);
        const uint32_t w = a1 > a0 ? (0xffffu >> (16 - (a1 - a0))) << a0 : 0u;
        seen = k ? (seen & 0xffffu) | w << 16 : (seen & 0xffff0000u) | w;
      }
      asm volatile("" : "+v"(seen));  // (a branch: its tests are for few steps)
#pragma unroll
      for (int k = 0; k < SUB; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[k][e] = seen >> (16 * k + e) & 1 ? s[k][e] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < SUB; ++k)
#pragma unroll
      for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(top, s[k][e]), s[k][e + 1]);
    top *= cq;
    if (__any(top > r + limit)) {
      float sized = -INFINITY;
#pragma unroll
      for (int k = 0; k < SUB; ++k)
        each<0, 16>([&](auto c) {
          constexpr int J = decltype(c)::value;
          sized = fmaxf(sized, __builtin_fmaf(s[k][J], cq, of_row<J>(ev[k])));
        });
      sized = fmaxf(fmaxf(ceilf(max_halves(sized)), ceilf(max_halves(top)) - kLeast4), r);
      const float keep = __builtin_amdgcn_exp2f(r - sized);
      r = sized;
      l *= keep;
      lows *= keep;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          acc[i][0][e] *= keep;
          acc[i][1][e] *= keep;
        }
    }
    h8 pf[SUB][2][2];
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
      float x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][j], cq, -r));
        l += x[j];
      }
      if (!tested) {
        lows = dot_row(lows, low[k], x);
        each<0, 16>([&](auto c) {
          constexpr int J = decltype(c)::value;
          x[J] *= of_row<J>(vs[k]);
        });
      } else {  // (past scales that are not finite)
        uint32_t bits = seen >> (16 * k);
        asm volatile("" : "+v"(bits));
        each<0, 16>([&](auto c) {
          constexpr int J = decltype(c)::value;
          const bool sees = bits >> J & 1;
          const float m = of_row<J>(low[k]), by = of_row<J>(vs[k]);
          lows = __builtin_fmaf(sees ? m : 0.0f, x[J], lows);
          x[J] = sees ? x[J] * by : 0.0f;
        });
      }
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        // halves of tokens j / 4 * 4 + {0, 2} and {1, 3}
        const int i = j / 4 * 4 + j % 4 / 2;
        h2 w0, w1;
        split4(x[i], x[i + 2], less, &w0, &w1);
        pf[k][j / 8][0][j % 8] = w0[0];
        pf[k][j / 8][0][j % 8 + 1] = w0[1];
        pf[k][j / 8][1][j % 8] = w1[0];
        pf[k][j / 8][1][j % 8 + 1] = w1[1];
      }
    }
#pragma unroll
    for (int k = 0; k < SUB; ++k)
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        Codes4 c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = codes4<CENTRE>(cv[k][i][j]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // tokens 16 hf + 8 u on
          const h8 low = halves8(c[2 * u].low[0], c[2 * u].low[1], c[2 * u + 1].low[0], c[2 * u + 1].low[1]);
          const h8 high = halves8(c[2 * u].high[0], c[2 * u].high[1], c[2 * u + 1].high[0], c[2 * u + 1].high[1]);
#pragma unroll
          for (int e = 1; e >= 0; --e) {
            acc[i][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(low, pf[k][u][e], acc[i][0], 0, 0, 0);
            acc[i][1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(high, pf[k][u][e], acc[i][1], 0, 0, 0);
          }
        }
      }
    if (t0 + kTokens4 < end) load_v(t0 + kTokens4);
  }

  // codes were 2^-18 as large, weights 2^8 times
  l = sum_halves(l);
  float base = sum_halves(lows), unit = 0x1p10f;
  if constexpr (SHARE) {
    extern __shared__ __attribute__((aligned(16))) float lds[];  // [sharers - 1][row_waves][D + 2][32]
    const int size = (D + 2) * 32;
    float* const theirs = lds + wave * size + n;  // of the second; the others' are row_waves * size on
    auto place = [&](int i, int h, int e) { return (32 * i + 8 * (e / 4) + 4 * hf + e % 4 + h * HALF) * 32; };
    auto there = [&](int i, int e) { return 32 * i + 8 * (e / 4) + 4 * hf < HALF; };
    if (which) {
      float* const to = theirs + (which - 1) * row_waves * size;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (there(i, e)) to[place(i, h, e)] = __builtin_fmaf(acc[i][h][e], unit, base);
      if (hf == 0) {
        to[D * 32] = r;
        to[D * 32 + 32] = l;
      }
    }
    __syncthreads();
    if (which) return;
    float top = r;
    for (int k = 0; k < sharers - 1; ++k) top = fmaxf(top, theirs[k * row_waves * size + D * 32]);
    float by = __builtin_amdgcn_exp2f(r - top);
    r = top;
    l *= by;
    unit *= by;
    base *= by;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][h][e] = __builtin_fmaf(acc[i][h][e], unit, base);
    for (int k = 0; k < sharers - 1; ++k) {
      const float* from = theirs + k * row_waves * size;
      by = __builtin_amdgcn_exp2f(from[D * 32] - top);
      l += from[D * 32 + 32] * by;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (there(i, e)) acc[i][h][e] = __builtin_fmaf(from[place(i, h, e)], by, acc[i][h][e]);
    }
    unit = 1.0f;
    base = 0.0f;
  }
  const int64_t pair = at.z * static_cast<int64_t>(cut.tiles) + tile;
  if (cut.splits > 1 && chunk == 0 && threadIdx.x == 0) cut.parts[pair] = chunks;
  if (wave * 32 + n >= count) return;
  if (chunks > 1) {
    float* to = cut.part + (pair * cut.splits + chunk) * part_floats(D);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int d = 32 * i + 8 * c + 4 * hf;
          if (d >= HALF) continue;
          const f4 v = f4{acc[i][h][4 * c], acc[i][h][4 * c + 1], acc[i][h][4 * c + 2], acc[i][h][4 * c + 3]} * unit + base;
          *reinterpret_cast<f4*>(to + row * D + h * HALF + d) = v;
        }
    if (hf == 0) {
      to[kTileRows * D + row] = r;
      to[kTileRows * D + kTileRows + row] = l;
    }
    return;
  }
  const float by = l != 0.0f ? 1.0f / l : 0.0f;
  const int qhead = head * a.group + static_cast<int>((first + row) % a.group);
  T* y = static_cast<T*>(a.y) + b * a.ys[0] + qt * a.ys[1] + qhead * a.ys[2];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 32 * i + 8 * c + 4 * hf;
        if (d >= HALF) continue;
        struct __attribute__((packed, aligned(sizeof(T)))) Four {
          T v[4];
        } o;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          from_f32(o.v[e], l != 0.0f ? __builtin_fmaf(acc[i][h][4 * c + e], unit, base) * by : 0.0f);
        *reinterpret_cast<Four*>(y + h * HALF + d) = o;
      }
}

template <typename T, int W, bool BIG, int WAVES, bool SHARE>
static int launch_tiles4(const QueryArgs& a, const Paged4Rows& rows, const TileCut& cut, int64_t pairs) {
  const char* who = "cache4_attention";
  const dim3 grid(static_cast<unsigned>(cut.splits), static_cast<unsigned>(cut.tiles), static_cast<unsigned>(pairs));
  KK_TRY(check_xcd_grid(grid, who));
  constexpr int SUB = W <= (sizeof(T) == 4 ? 2 : SHARE && !BIG ? 3 : 4) ? 2 : 1;  // (what spills nothing)
  const unsigned bytes = SHARE ? (WAVES - cut.row_waves) * (32 * W + 2) * 32 * 4 : 0;
  if (bytes > 65536)
    KK_TRY(allow_large_lds(reinterpret_cast<const void*>(tile_paged4_kernel<T, W, SUB, BIG, WAVES, SHARE>)));
  KK_LAUNCH((tile_paged4_kernel<T, W, SUB, BIG, WAVES, SHARE>), grid, dim3(64 * WAVES), bytes, ctx().stream, a, rows, cut);
  KK_TRY(check_launch("tile_paged4_kernel"));
  if (cut.splits == 1) return KK_OK;
  KK_LAUNCH((join_parts_kernel<T, Paged4Rows>), dim3(static_cast<unsigned>(pairs * cut.tiles * (kTileRows / (kTileThreads / 64)))),
            dim3(kTileThreads), 0, ctx().stream, a, rows, cut);
  return check_launch("join_parts_kernel");
}

// Tokens shared by the waves of a block where it has 64 queries at most (16 sequences of
// 64 queries a key head over up to 4000 tokens: 115 us where the other waves idle,
// 65 here), and by eight waves, of which one block fits a CU, where whole rounds of a
// tile's blocks take five eighths of the CUs or more (fp16 heads of 128, 128 blocks: 148 us
// with four waves, 124 with eight; 176: 83 and 72; heads of 64 in fp32, 144 blocks: 60
// and 60); else four waves, and as many blocks as fit two a CU.
template <typename T, int W, bool BIG>
static int launch_tiles4(const QueryArgs& a, const Paged4Rows& rows, int64_t tokens) {
  const int64_t queries = int64_t{a.T} * a.group, pairs = a.B * rows.a.heads, tiles = ceil_div(queries, kTileRows);
  const int64_t cus = ctx().num_cus, blocks = pairs * tiles;
  TileCut cut{};
  cut.rows = queries;
  cut.tiles = static_cast<int>(tiles);
  cut.row_waves = queries <= 32 ? 1 : queries <= 64 ? 2 : 4;
  if constexpr (W <= 4)
    if (cut.row_waves < 4 || cus / blocks * blocks * 8 >= cus * 5) {
      plan_parts(blocks, tokens, kLeastTokens4, a.D, blocks < cus ? cus - blocks + 1 : 1, &cut);
      return launch_tiles4<T, W, BIG, 8, true>(a, rows, cut, pairs);
    }
  plan_parts(blocks, tokens, kLeastTokens4, a.D, 2 * cus, &cut);
  if constexpr (W > 4)
    if (cut.row_waves < 4) return launch_tiles4<T, W, BIG, 4, true>(a, rows, cut, pairs);
  return launch_tiles4<T, W, BIG, 4, false>(a, rows, cut, pairs);
}

template <typename T, bool BIG>
static int launch_tiles4(const QueryArgs& a, const Paged4Rows& rows, int64_t tokens) {
  switch (a.D / 32) {
    case 1: return launch_tiles4<T, 1, BIG>(a, rows, tokens);
    case 2: return launch_tiles4<T, 2, BIG>(a, rows, tokens);
    case 3: return launch_tiles4<T, 3, BIG>(a, rows, tokens);
    case 4: return launch_tiles4<T, 4, BIG>(a, rows, tokens);
    case 5: return launch_tiles4<T, 5, BIG>(a, rows, tokens);
    case 6: return launch_tiles4<T, 6, BIG>(a, rows, tokens);
    case 7: return launch_tiles4<T, 7, BIG>(a, rows, tokens);
  }
  return launch_tiles4<T, 8, BIG>(a, rows, tokens);
}

bool tiles_paged4_try(const QueryArgs& a, const Paged4Rows& rows, int dtype, int* status) {
  const PagedArgs& p = rows.a;
  if (p.pages < 1 || p.columns < 1) return false;
  const int64_t capacity = p.columns * p.block;
  const int64_t seen = p.window && p.window < capacity ? p.window + a.T - 1 : capacity;
  const int64_t tokens = seen < capacity ? seen : capacity;
  // (past the grid's axes: one query a wave)
  if (a.B * p.heads > 65535 || int64_t{a.T} * a.group > int64_t{65535} * kTileRows) return false;
  if (p.block >= 64)
    *status = dtype == KK_F16 ? launch_tiles4<__half, true>(a, rows, tokens) : launch_tiles4<float, true>(a, rows, tokens);
  else
    *status = dtype == KK_F16 ? launch_tiles4<__half, false>(a, rows, tokens) : launch_tiles4<float, false>(a, rows, tokens);
  return true;
}

}  // namespace kk
