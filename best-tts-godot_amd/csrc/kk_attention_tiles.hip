// Attention of many queries (a chunk of new tokens, the frames of an utterance)
// over a paged cache of 8-bit codes or an encoder's states.
#include "kk_attention.h"

namespace kk {

typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kTileThreads = 256;
constexpr int kTileRows = 128;  // queries of a block: 32 a wave

struct TileCut {
  int splits;          // blocks that share the tokens of a tile of queries
  int tiles;           // of kTileRows queries in a sequence and key head
  int64_t rows;        // queries of a sequence and key head: T * group
  int wide;            // rows of q, k and v take 16-byte accesses
  float* part;
  int* arrived;
};

// Where the tile kernel's operands come from.
enum Source { kPaged, kHalf, kFloat };

// LDS of a block, in bytes: keys [TT][pitch], values [32 DT][pitch] (a copy for each
// half of a split value), exponents and largest magnitudes of fp32 rows; later
// the sums.
constexpr int key_pitch(int DT) { return 64 * DT + 16; }
constexpr int value_pitch(int TT) { return 2 * TT + 16; }
constexpr int tile_bytes(int SRC, int DT, int TT) {
  return (TT * key_pitch(DT) + 32 * DT * value_pitch(TT)) * (SRC == kFloat ? 2 : 1) + (SRC == kFloat ? 6 * TT * 4 : 0);
}

__device__ __forceinline__ float other_half(float v) {  // the value of lane l ^ 32
  return __shfl_xor(v, 32, 64);
}

// Whether a mask differs from query to query, and what it lets query t see of
// tokens t0 .. t0 + TT - 1 (of those in `w`).
__device__ __forceinline__ bool rows_masked_by_query(const PagedRows&, const QueryArgs&) { return false; }
template <typename T>
__device__ __forceinline__ bool rows_masked_by_query(const DenseRows<T>& rows, const QueryArgs& a) {
  return rows.a.mask && rows.a.ms[1] != 0 && a.T > 1;
}
template <class Rows>
__device__ __forceinline__ uint64_t query_mask(const Rows& rows, const QueryArgs& a, int64_t b, int64_t t, int64_t t0,
                                               int TT, uint64_t w) {
  if (!rows_masked_by_query(rows, a)) return w;
  uint64_t r = 0;
  const uint8_t* mask = rows.a.mask + b * rows.a.ms[0] + t * rows.a.ms[1] + t0 * rows.a.ms[2];
  for (int j = 0; j < TT; ++j)
    if ((w >> j & 1) && mask[j * rows.a.ms[2]]) r |= uint64_t{1} << j;
  return r;
}

// out = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m) for 128 queries of a key
// head (all its query heads, token by token) on the matrix cores
// (v_mfma_f32_32x32x16_f16), 32 a wave, over tiles of TT tokens that the block
// brings to LDS as halves: keys row by row, values a row each of a head's
// values.  Scores are formed transposed, S^T = K Q^T: a lane (n = l % 32,
// h = l / 32) holds a query's column, so its maximum and sum need one exchange
// with lane l ^ 32, and with the tokens' order in the keys' rows (row_of) its
// registers are, eight by eight, what the product O^T = V^T P^T takes.
//
// 8-bit codes and fp16 values are exact as halves; fp32 operands are the sum of
// two, after a power of two for each row that brings its largest to 2^14, so
// that 22 bits are kept whatever the rows' sizes, and the product of the two
// low halves (2^-22) is left out.  Weights of fp16 queries are rounded to fp16
// (half a step of the output's type); 2^15 p <= 2^15 keeps 24 bits above
// fp16's smallest value.
//
// A state that is not finite poisons whole sums here (0 times it is NaN) where
// only queries that see it should be: a block that meets one marks its part, and
// its queries are formed one by one.
template <typename T, class Rows, int SRC, int DT, int TT>
__global__ void __launch_bounds__(kTileThreads, DT <= (SRC == kFloat ? 2 : 4) ? 2 : 1)
    attention_tile_kernel(QueryArgs a, Rows rows, TileCut cut) {
  constexpr int PQ = sizeof(T) == 4 ? 2 : 1, PK = SRC == kFloat ? 2 : 1, PW = PQ;
  constexpr int KS = 2 * DT, NS = TT / 32, G = TT / 16;
  constexpr int KP = key_pitch(DT), VP = value_pitch(TT);
  constexpr bool kAhead = SRC != kFloat || DT <= 4;  // (fp32 heads past 128 values leave no registers for it)
  extern __shared__ __attribute__((aligned(16))) char tile_lds[];
  char* lds_k = tile_lds;
  char* lds_v = lds_k + PK * TT * KP;
  uint32_t* largest = reinterpret_cast<uint32_t*>(lds_v + PK * 32 * DT * VP);  // [2][keys, values][TT]
  float* key_scale = reinterpret_cast<float*>(largest + 4 * TT);
  int* value_exp = reinterpret_cast<int*>(key_scale + TT);

  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int n = lane % 32, hf = lane / 32, D = a.D;
  // neighbouring blocks of an XCD share keys and values; the longest rows first
  const uint3 at = xcd_tile();  // (split, tile, sequence and head)
  const int tile = cut.tiles - 1 - static_cast<int>(at.y), heads = a.heads / a.group;
  const int64_t b = at.z / heads, first = static_cast<int64_t>(tile) * kTileRows;
  const int h = at.z % heads;
  const int count = static_cast<int>(cut.rows - first < kTileRows ? cut.rows - first : kTileRows);

  // the tokens that any of the queries sees, and this block's share of them
  const Seen s0 = rows.seen(b, first / a.group);
  int64_t lo = s0.lo, hi = s0.hi;
  if constexpr (SRC == kPaged) {
    int64_t t1 = (first + count - 1) / a.group;
    const int64_t there = rows.count(b);
    t1 = t1 < there ? t1 : there - 1;
    if (t1 >= first / a.group) hi = rows.seen(b, t1).hi;
  }
  lo = lo / TT * TT;
  const int64_t steps = ceil_div(hi - lo, TT);
  int64_t each = ceil_div(steps, cut.splits);
  each = each < 4 ? 4 : each;
  const int chunks = steps <= each ? 1 : static_cast<int>(ceil_div(steps, each));
  const int chunk = static_cast<int>(at.x);
  if (chunk >= chunks) return;
  lo = uniform(lo + chunk * each * TT);
  hi = uniform(chunk + 1 < chunks ? lo + each * TT : hi);

  // the lane's query
  const int row = wave * 32 + n < count ? wave * 32 + n : count - 1;
  const int64_t qt = (first + row) / a.group;
  const int qhead = h * a.group + static_cast<int>((first + row) % a.group);
  const Seen qs = rows.seen(b, qt);
  float cq = a.scale;
  h8 qf[KS][PQ];
  {
    const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + qt * a.qs[1] + qhead * a.qs[2];
    T x[KS][8];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * hf;
      if (cut.wide && d < D) {
        if constexpr (PQ == 1) {
          const h8 v = *reinterpret_cast<const h8*>(q + d);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[s][i] = __builtin_bit_cast(__half, static_cast<_Float16>(v[i]));
        } else {
          const f4 v0 = *reinterpret_cast<const f4*>(q + d), v1 = *reinterpret_cast<const f4*>(q + d + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[s][i] = v0[i];
            x[s][i + 4] = v1[i];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[s][i] = d + i < D ? q[d + i] : T(0.0f);
      }
    }
    if constexpr (PQ == 1) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[s][0][i] = __builtin_bit_cast(_Float16, x[s][i]);
    } else {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, __builtin_fabsf(x[s][i]));
      top = fmaxf(top, other_half(top));
      const int up = 14 + 127 - static_cast<int>(__float_as_uint(top) >> 23);
      cq = ldexpf(a.scale, -up);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = ldexpf(x[s][i], up);
          const _Float16 y0 = static_cast<_Float16>(y);
          qf[s][0][i] = y0;
          qf[s][PQ - 1][i] = static_cast<_Float16>(y - static_cast<float>(y0));
        }
    }
  }

  // ---- from memory: a tile's values in registers, one tile ahead
  // token tk of 32 lies in row 8 j + 4 h + r, where its score comes out in
  // register 4 j + r of half h: tokens 16 (j / 2) + 8 h + 4 (j % 2) + r
  auto row_of = [](int tk) { return (tk & ~31) | (tk & 16) | (tk & 4) << 1 | (tk & 8) >> 1 | (tk & 3); };
  constexpr int kKeyUnits = SRC == kPaged ? TT * 2 * DT : TT * 4 * DT;  // 16 codes, or 8 values
  constexpr int kVD = SRC == kHalf ? 8 : 4;                             // values of 4 tokens, or 16 codes of a row
  constexpr int kValueUnits = SRC == kPaged ? 32 * DT * G : TT / 4 * (32 * DT / kVD);
  constexpr int UK = (kKeyUnits + kTileThreads - 1) / kTileThreads;
  constexpr int UV = (kValueUnits + kTileThreads - 1) / kTileThreads;
  u4 ck[SRC == kFloat ? 2 * UK : UK], cv[SRC == kPaged ? UV : 4 * UV];

  // paged: the units' table entries a tile before their codes, the scales of
  // the wave's groups of 16 tokens (lane % G) with them
  int entry_k[UK], entry_v[UV], entry_s = 0, page_s = -1;
  float ks = 0.0f, vs = 0.0f, ks1 = 0.0f, vs1 = 0.0f;
  // dense: bit j: token j of the tile may be seen by the block's queries
  uint64_t word = 0;
  uint8_t mask_byte = 0;

  auto entry = [&](int64_t t) -> int {
    if constexpr (SRC == kPaged) {
      const int64_t column = t >> __builtin_ctz(rows.a.block);
      return rows.a.table[b * rows.a.table_stride + (column < rows.a.columns ? column : rows.a.columns - 1)];
    }
    return 0;
  };
  auto entries = [&](int64_t t0) {
    if constexpr (SRC == kPaged) {
#pragma unroll
      for (int i = 0; i < UK; ++i) entry_k[i] = entry(t0 + (tid + kTileThreads * i) / (2 * DT) % TT);
#pragma unroll
      for (int i = 0; i < UV; ++i) entry_v[i] = entry(t0 + 16 * ((tid + kTileThreads * i) % G));
      entry_s = entry(t0 + 16 * (lane % G));
    }
  };
  auto fetch = [&](int64_t t0) {
    if constexpr (SRC == kPaged) {
      const auto& p = rows.a;
      const int64_t page_bytes = int64_t{p.block} * D;
      auto base = [&](int e) { return (int64_t{e >= 0 && e < p.pages ? e : 0} * p.heads + h) * page_bytes; };
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = tid + kTileThreads * i, tk = u / (2 * DT), c = u % (2 * DT);
        ck[i] = u4{0, 0, 0, 0};
        if (u < kKeyUnits && 16 * c < D)
          ck[i] = *reinterpret_cast<const u4*>(p.k + base(entry_k[i]) +
                                               static_cast<int>((t0 + tk) & (p.block - 1)) * D + 16 * c);
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = tid + kTileThreads * i, d = u / G, g = u % G;
        cv[i] = u4{0, 0, 0, 0};
        if (u < kValueUnits && d < D)
          cv[i] = *reinterpret_cast<const u4*>(p.v + base(entry_v[i]) + d * p.block +
                                               static_cast<int>((t0 + 16 * g) & (p.block - 1)));
      }
      const int64_t t = t0 + 16 * (lane % G);
      page_s = t < hi && t >> __builtin_ctz(p.block) < p.columns && entry_s < p.pages ? entry_s : -1;
      const int64_t sc = int64_t{page_s < 0 ? 0 : page_s} * p.heads + h;
      ks1 = p.k_scale[sc];
      vs1 = p.v_scale[sc];
    } else {
      using S = std::conditional_t<SRC == kHalf, __half, float>;
      const auto& p = rows.a;
      const S* k = static_cast<const S*>(p.k) + b * p.ks[0] + h * p.ks[2];
      const S* v = static_cast<const S*>(p.v) + b * p.vs[0] + h * p.vs[2];
      // what no query of the block may see is not read
      bool sees = t0 + lane < hi && lane < TT;
      if (sees && p.mask && (p.ms[1] == 0 || a.T == 1)) sees = p.mask[b * p.ms[0] + (t0 + lane) * p.ms[2]] != 0;
      word = __ballot(sees);
      auto load8 = [&](const S* from, int d, bool there, u4* to) {  // 16 bytes of half, 32 of float
        constexpr int W = SRC == kFloat ? 2 : 1;
        if (cut.wide) {
#pragma unroll
          for (int w = 0; w < W; ++w)
            to[w] = there && d < D ? *reinterpret_cast<const u4*>(from + d + 4 * w) : u4{0, 0, 0, 0};
        } else {
          S e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = there && d + i < D ? from[d + i] : S(0.0f);
#pragma unroll
          for (int w = 0; w < W; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (SRC == kFloat)
                to[w][i] = __float_as_uint(e[4 * w + i]);
              else
                to[w][i] = __half_as_ushort(e[2 * i]) | static_cast<uint32_t>(__half_as_ushort(e[2 * i + 1])) << 16;
            }
        }
      };
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = tid + kTileThreads * i, tk = u / (4 * DT), d = 8 * (u % (4 * DT));
        load8(k + (t0 + tk) * p.ks[1], d, u < kKeyUnits && (word >> (tk & 63) & 1), ck + (SRC == kFloat ? 2 * i : i));
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = tid + kTileThreads * i;
        const int d = kVD * (u % (32 / kVD) + 32 / kVD * (u / (32 / kVD * (TT / 4)))), tq = u / (32 / kVD) % (TT / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool there = u < kValueUnits && (word >> (4 * tq + j) & 1);
          const S* from = v + (t0 + 4 * tq + j) * p.vs[1];
          if constexpr (SRC == kHalf) {
            load8(from, d, there, cv + 4 * i + j);
          } else if (cut.wide) {
            cv[4 * i + j] = there && d < D ? *reinterpret_cast<const u4*>(from + d) : u4{0, 0, 0, 0};
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) cv[4 * i + j][e] = there && d + e < D ? __float_as_uint(from[d + e]) : 0;
          }
        }
      }
    }
  };
  uint32_t bad = 0;  // bit 15 or 31: a half that is not finite; of fp32, all: an exponent of 255
  auto magnitudes = [&](int which) {  // fp32: the rows' largest
    uint32_t* lk = largest + 2 * TT * which;
    uint32_t* lv = lk + TT;
#pragma unroll
    for (int i = 0; i < UK; ++i) {
      const int u = tid + kTileThreads * i;
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, ck[(2 * i + e / 4) % (2 * UK)][e % 4] & 0x7fffffffu);
      if (u < kKeyUnits) atomicMax(lk + u / (4 * DT), m);
      bad |= m >= 0x7f800000u ? 0x80000000u : 0u;
    }
#pragma unroll
    for (int i = 0; i < UV; ++i) {
      const int u = tid + kTileThreads * i, tq = u / (32 / kVD) % (TT / 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, cv[(4 * i + j) % (4 * UV)][e] & 0x7fffffffu);
        if (u < kValueUnits) atomicMax(lv + 4 * tq + j, m);
        bad |= m >= 0x7f800000u ? 0x80000000u : 0u;
      }
    }
  };
  auto stage = [&](int which) {
    if constexpr (SRC == kPaged) {
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = tid + kTileThreads * i, tk = u / (2 * DT), c = u % (2 * DT);
        if (u >= kKeyUnits) continue;
        h8* to = reinterpret_cast<h8*>(lds_k + row_of(tk) * KP + 32 * c);
        to[0] = codes_h8(ck[i][0], ck[i][1]);
        to[1] = codes_h8(ck[i][2], ck[i][3]);
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = tid + kTileThreads * i, d = u / G, g = u % G;
        if (u >= kValueUnits) continue;
        h8* to = reinterpret_cast<h8*>(lds_v + d * VP + 32 * g);
        to[0] = codes_h8(cv[i][0], cv[i][1]);
        to[1] = codes_h8(cv[i][2], cv[i][3]);
      }
    } else if constexpr (SRC == kHalf) {
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = tid + kTileThreads * i, tk = u / (4 * DT), c = u % (4 * DT);
        if (u >= kKeyUnits) continue;
        *reinterpret_cast<u4*>(lds_k + row_of(tk) * KP + 16 * c) = ck[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (ck[i][e] & 0x7c007c00u) + 0x04000400u;
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = tid + kTileThreads * i;
        if (u >= kValueUnits) continue;
        const int d = kVD * (u % (32 / kVD) + 32 / kVD * (u / (32 / kVD * (TT / 4)))), tq = u / (32 / kVD) % (TT / 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // the d-th value of four tokens
          const uint32_t sel = e % 2 ? 0x07060302u : 0x05040100u;
          typedef uint32_t u2 __attribute__((ext_vector_type(2)));
          const u2 w = {__builtin_amdgcn_perm(cv[(4 * i + 1) % (4 * UV)][e / 2], cv[4 * i][e / 2], sel),
                        __builtin_amdgcn_perm(cv[(4 * i + 3) % (4 * UV)][e / 2], cv[(4 * i + 2) % (4 * UV)][e / 2], sel)};
          *reinterpret_cast<u2*>(lds_v + (d + e) * VP + 8 * tq) = w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) bad |= (cv[(4 * i + j) % (4 * UV)][e] & 0x7c007c00u) + 0x04000400u;
      }
    } else {
      const uint32_t* lk = largest + 2 * TT * which;
      const uint32_t* lv = lk + TT;
      auto split = [](float x, int up, _Float16* hi16, _Float16* lo16) {
        const float y = __builtin_amdgcn_ldexpf(x, up);
        *hi16 = static_cast<_Float16>(y);
        *lo16 = static_cast<_Float16>(y - static_cast<float>(*hi16));
      };
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = tid + kTileThreads * i, tk = u / (4 * DT), c = u % (4 * DT);
        if (u >= kKeyUnits) continue;
        const int up = 141 - static_cast<int>(lk[tk] >> 23);
        h8 y0, y1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          _Float16 p0, p1;
          split(__uint_as_float(ck[(2 * i + e / 4) % (2 * UK)][e % 4]), up, &p0, &p1);
          y0[e] = p0;
          y1[e] = p1;
        }
        *reinterpret_cast<h8*>(lds_k + row_of(tk) * KP + 16 * c) = y0;
        *reinterpret_cast<h8*>(lds_k + (TT + row_of(tk)) * KP + 16 * c) = y1;
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = tid + kTileThreads * i;
        if (u >= kValueUnits) continue;
        const int d = kVD * (u % (32 / kVD) + 32 / kVD * (u / (32 / kVD * (TT / 4)))), tq = u / (32 / kVD) % (TT / 4);
        const u4 top = *reinterpret_cast<const u4*>(lv + 4 * tq);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h4 y0, y1;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            _Float16 p0, p1;
            split(__uint_as_float(cv[(4 * i + j) % (4 * UV)][e]), 141 - static_cast<int>(top[j] >> 23), &p0, &p1);
            y0[j] = p0;
            y1[j] = p1;
          }
          *reinterpret_cast<h4*>(lds_v + (d + e) * VP + 8 * tq) = y0;
          *reinterpret_cast<h4*>(lds_v + (32 * DT + d + e) * VP + 8 * tq) = y1;
        }
      }
      if (tid < TT) key_scale[tid] = ldexpf(1.0f, static_cast<int>(lk[tid] >> 23) - 141);
      if (tid >= 64 && tid < 64 + TT) value_exp[tid - 64] = static_cast<int>(lv[tid - 64] >> 23);
      if (tid >= 128 && tid < 128 + 2 * TT) largest[2 * TT * (which ^ 1) + tid - 128] = 0;
    }
  };

  f16v acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
  float m = -3.4028235e38f, l = 0.0f;
  int er = SRC == kPaged ? 27 : 0;  // values are scaled by 2^-(er - 127) (paged), 2^-(er - 141) (fp32)

  if constexpr (SRC == kFloat) {
    if (tid < 2 * TT) largest[tid] = 0;
    __syncthreads();
  }
  if (lo < hi) {
    entries(lo);
    if (kAhead) fetch(lo);
    if (kAhead) entries(lo + TT);
  }
  const bool mine = wave * 32 < count;
  int which = 0;
  for (int64_t t0 = lo; t0 < hi; t0 += TT, which ^= 1) {
    if (!kAhead) fetch(t0);
    if constexpr (SRC == kFloat) magnitudes(which);
    __syncthreads();  // the tile before is read
    stage(which);
    const uint64_t here = word;
    const int page = page_s;
    ks = ks1;
    vs = page < 0 ? 0.0f : vs1;
    if (kAhead && t0 + TT < hi) {
      fetch(t0 + TT);
      entries(t0 + 2 * TT);
    }
    __syncthreads();
    if (!mine) continue;
    // what the lane's query sees of its tokens 32 s + 16 (i / 8) + 8 hf + i % 8: bit 16 s + i
    uint32_t seen = 0xffffffffu >> (32 - 16 * NS);
    {
      const int64_t below = qs.lo - t0, upto = qs.hi - t0;
      const bool whole = below <= 0 && upto >= TT;
      bool all = whole;
      if constexpr (SRC == kPaged)
        all = all && page >= 0 && (__float_as_uint(vs) & 0x7f800000u) != 0x7f800000u;
      else
        all = all && here == ~uint64_t{0} >> (64 - TT);
      if (SRC != kPaged && rows_masked_by_query(rows, a)) all = false;
      if (!__all(all)) {
        uint64_t w = 0;  // by token
        const int lo32 = below < 0 ? 0 : below > TT ? TT : static_cast<int>(below);
        const int hi32 = upto < 0 ? 0 : upto > TT ? TT : static_cast<int>(upto);
        if (hi32 > lo32) w = (~uint64_t{0} >> (64 - (hi32 - lo32))) << lo32;
        if constexpr (SRC == kPaged) {
          const uint64_t pages = __ballot(page >= 0);
#pragma unroll
          for (int g = 0; g < G; ++g)
            if (!(pages >> g & 1)) w &= ~(uint64_t{0xffff} << (16 * g));
        } else {
          w = query_mask(rows, a, b, qt, t0, TT, w & here);
        }
        w >>= 8 * hf;
        seen = 0;
#pragma unroll
        for (int s = 0; s < 2 * NS; ++s) seen |= (static_cast<uint32_t>(w >> (16 * s)) & 0xffu) << (8 * s);
        if (!__any(seen != 0)) continue;
      } else {
        seen = 0xffffffffu;  // (no test below)
      }
    }
    const bool tested = !__all(seen == 0xffffffffu) ;

    f16v s[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[j][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const char* from = lds_k + (32 * j + n) * KP + 32 * k + 16 * hf;
        const h8 k0 = *reinterpret_cast<const h8*>(from);
        if constexpr (PK == 2) {
          const h8 k1 = *reinterpret_cast<const h8*>(from + TT * KP);
          s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qf[k][0], s[j], 0, 0, 0);
        }
        if constexpr (PQ == 2) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qf[k][PQ - 1], s[j], 0, 0, 0);
        s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qf[k][0], s[j], 0, 0, 0);
      }
    }

    // the values' power of two
    float keep_r = 1.0f;
    if constexpr (SRC != kHalf) {
      int e1 = 0;
      if constexpr (SRC == kPaged) {
        const uint32_t bits = __float_as_uint(__builtin_fabsf(vs));
        e1 = bits < 0x7f800000u ? static_cast<int>(bits >> 23) + 1 : 0;
        e1 = e1 > 254 ? 254 : e1;
      } else {
        e1 = lane < TT ? value_exp[lane % TT] : 0;
      }
      if (__any(e1 > er)) {
        for (int off = 1; off < 64; off <<= 1) {
          const int o = __shfl_xor(e1, off, 64);
          e1 = o > e1 ? o : e1;
        }
        const int up = __builtin_amdgcn_readfirstlane(e1 > er ? e1 : er);
        keep_r = ldexpf(1.0f, er - up);
        er = up;
      }
    }
    float by[G], vw[G];
    if constexpr (SRC == kPaged) {
      const float r1 = __uint_as_float(static_cast<uint32_t>(254 - er) << 23);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        by[g] = cq * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), g));
        vw[g] = r1 * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), g));
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        f4 kc = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (SRC == kFloat)
          kc = *reinterpret_cast<const f4*>(key_scale + 32 * j + 16 * (c / 2) + 8 * hf + 4 * (c % 2));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[j][4 * c + e] * (SRC == kPaged ? by[(2 * j + c / 2) % G] : cq);
          if constexpr (SRC == kFloat) x *= kc[e];
          s[j][4 * c + e] = x;
        }
      }
    if (tested) {
#pragma unroll
      for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[j][e] = seen >> (16 * j + e) & 1 ? s[j][e] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[j][e]);
    top = fmaxf(fmaxf(top, other_half(top)), m);
    if (__any(top > m) || keep_r != 1.0f) {
      const float keep = __builtin_amdgcn_exp2f(m - top), both = keep * keep_r;
      m = top;
      l *= keep;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= both;
    }
    const float less = m - 15.0f;  // weights are 2^15 times as large, and their sum
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = __builtin_amdgcn_exp2f(s[j][8 * k + e] - less);
          l += w[e];
        }
        if constexpr (SRC == kPaged) {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] *= vw[(2 * j + k) % G];
          if (tested) {  // (past a scale that is not finite)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = seen >> (16 * j + 8 * k + e) & 1 ? w[e] : 0.0f;
          }
        }
        if constexpr (SRC == kFloat) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            typedef int i4 __attribute__((ext_vector_type(4)));
            const i4 ve = *reinterpret_cast<const i4*>(value_exp + 32 * j + 16 * k + 8 * hf + 4 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * c + e] = __builtin_amdgcn_ldexpf(w[4 * c + e], ve[e] - er);
          }
        }
        h8 pf[PW];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pf[0][e] = static_cast<_Float16>(w[e]);
          if constexpr (PW == 2) pf[PW - 1][e] = static_cast<_Float16>(w[e] - static_cast<float>(pf[0][e]));
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const char* from = lds_v + (32 * i + n) * VP + 64 * j + 32 * k + 16 * hf;
          const h8 v0 = *reinterpret_cast<const h8*>(from);
          if constexpr (PK == 2) {
            const h8 v1 = *reinterpret_cast<const h8*>(from + 32 * DT * VP);
            acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, pf[0], acc[i], 0, 0, 0);
          }
          if constexpr (PW == 2) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, pf[PW - 1], acc[i], 0, 0, 0);
          acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, pf[0], acc[i], 0, 0, 0);
        }
      }
  }

  // the sums by rows, in LDS
  if (SRC == kHalf) bad &= 0x80008000u;
  const bool marked = __syncthreads_or(SRC != kPaged && bad != 0);
  const int pitch = D + 4;
  float* sums = reinterpret_cast<float*>(tile_lds);
  float* wm = sums + kTileRows * pitch;
  float* wl = wm + kTileRows;
  l += other_half(l);
  const int r = wave * 32 + n;
  if (r < count) {
    const float by = SRC == kHalf ? 1.0f : ldexpf(1.0f, er - (SRC == kPaged ? 127 : 141));
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 32 * i + 8 * c + 4 * hf;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) sums[r * pitch + d + e] = acc[i][4 * c + e] * by;
      }
    if (hf == 0) {
      wm[r] = marked ? NAN : m;
      wl[r] = l;
    }
  }
  __syncthreads();
  const int64_t pair = at.z * static_cast<int64_t>(cut.tiles) + tile, slot = int64_t{kTileRows} * (D + 2);
  const Part part{b, h, count, chunk, chunks, first, cut.part + pair * cut.splits * slot, slot, cut.arrived + pair};
  if (put_rows<T, kTileThreads>(a, part, sums, pitch, wm, wl, wl + kTileRows)) return;
  __syncthreads();
  for (int i = wave; i < count; i += kTileThreads / 64) {
    const int64_t at_row = first + i;
    one_query<T>(a, rows, b, at_row / a.group, h * a.group + static_cast<int>(at_row % a.group), sums + wave * kMaxHead);
  }
}

template <typename T, class Rows, int SRC, int DT, int TT>
static int launch_tiles(const QueryArgs& a, const Rows& rows, int64_t tokens, int wide, const char* who) {
  const int64_t queries = int64_t{a.T} * a.group, pairs = a.B * (a.heads / a.group);
  const int64_t tiles = ceil_div(queries, kTileRows);
  TileCut cut{};
  cut.rows = queries;
  cut.wide = wide;
  cut.part = static_cast<float*>(ctx().scratch);
  cut.arrived = ctx().row_counters;
  // where there are fewer blocks than two a CU, the tokens are cut, into parts
  // of four tiles at least
  const int64_t blocks = pairs * tiles;
  int64_t splits = ceil_div(2 * ctx().num_cus, blocks);
  const int64_t room = static_cast<int64_t>(kScratchBytes / 4) / (int64_t{kTileRows} * (a.D + 2)) / blocks;
  const int64_t parts = ceil_div(tokens, 4 * TT);
  splits = splits < parts ? splits : parts;
  splits = splits < kMaxChunks ? splits : kMaxChunks;
  splits = splits < room ? splits : room;
  if (splits < 1 || blocks > kRowCounters) splits = 1;
  cut.splits = static_cast<int>(splits);
  cut.tiles = static_cast<int>(tiles);
  const dim3 grid(static_cast<unsigned>(splits), static_cast<unsigned>(tiles), static_cast<unsigned>(pairs));
  KK_TRY(check_xcd_grid(grid, who));
  int64_t bytes = (int64_t{kTileRows} * (a.D + 4) + 2 * kTileRows + (splits > 1 ? splits * kTileRows : 0)) * 4;
  if (bytes < tile_bytes(SRC, DT, TT)) bytes = tile_bytes(SRC, DT, TT);
  if (bytes < 4 * kMaxHead * 4) bytes = 4 * kMaxHead * 4;
  if (bytes > 65536) KK_TRY(allow_large_lds(reinterpret_cast<const void*>(attention_tile_kernel<T, Rows, SRC, DT, TT>)));
  KK_LAUNCH((attention_tile_kernel<T, Rows, SRC, DT, TT>), grid, dim3(kTileThreads), static_cast<unsigned>(bytes),
            ctx().stream, a, rows, cut);
  return check_launch("attention_tile_kernel");
}

template <typename T, class Rows, int SRC>
static int launch_tiles(const QueryArgs& a, const Rows& rows, int64_t tokens, int wide, const char* who) {
  return a.D <= 64    ? launch_tiles<T, Rows, SRC, 2, 64>(a, rows, tokens, wide, who)
         : a.D <= 96  ? launch_tiles<T, Rows, SRC, 3, 64>(a, rows, tokens, wide, who)
         : a.D <= 128 ? launch_tiles<T, Rows, SRC, 4, 64>(a, rows, tokens, wide, who)
                      : launch_tiles<T, Rows, SRC, 8, 32>(a, rows, tokens, wide, who);
}

// Whether rows of an operand start at multiples of 16 bytes.
static bool rows_of_16(const void* p, const int64_t* strides, int size) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] * size % 16) return false;
  return true;
}

// (past the grid's axes: one query a wave)
static bool too_many(const QueryArgs& a) {
  return a.B * (a.heads / a.group) > 65535 || int64_t{a.T} * a.group > int64_t{65535} * kTileRows;
}

bool tiles_paged_try(const QueryArgs& a, const PagedArgs& p, int dtype, int* status) {
  if (p.pages < 1 || p.columns < 1) return false;
  const PagedRows rows{p, a.T, a.D};
  const int64_t capacity = p.columns * p.block, seen = p.window ? p.window + a.T - 1 : capacity;
  const int64_t tokens = seen < capacity ? seen : capacity;
  if (too_many(a)) return false;
  const int wide = rows_of_16(a.q, a.qs, dtype == KK_F16 ? 2 : 4);
  const char* who = "cache_attention";
  *status = dtype == KK_F16 ? launch_tiles<__half, PagedRows, kPaged>(a, rows, tokens, wide, who)
                            : launch_tiles<float, PagedRows, kPaged>(a, rows, tokens, wide, who);
  return true;
}

bool tiles_dense_try(const QueryArgs& a, const DenseArgs& d, int dtype, int* status) {
  if (d.S < 1 || too_many(a)) return false;
  const int size = dtype == KK_F16 ? 2 : 4;
  const int wide = a.D % 8 == 0 && d.ks[3] == 1 && d.vs[3] == 1 && rows_of_16(a.q, a.qs, size) &&
                   rows_of_16(d.k, d.ks, size) && rows_of_16(d.v, d.vs, size);
  const char* who = "cross_attention";
  *status = dtype == KK_F16
                ? launch_tiles<__half, DenseRows<__half>, kHalf>(a, DenseRows<__half>{d}, d.S, wide, who)
                : launch_tiles<float, DenseRows<float>, kFloat>(a, DenseRows<float>{d}, d.S, wide, who);
  return true;
}

}  // namespace kk
