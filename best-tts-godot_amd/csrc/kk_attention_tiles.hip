// Attention of many queries (a chunk of new tokens, the frames of an utterance)
// over a paged cache of 8-bit codes or an encoder's states.
#include "kk_attention.h"

namespace kk {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kTileThreads = 256;
constexpr int kTileRows = 128;  // queries of a block: 32 a wave
constexpr int kPutRows = 64;    // of them put out at a time
constexpr int kLeastTiles = 2;    // of tokens, of a block that shares them
constexpr float kSlack = 7.0f;

struct TileCut {
  int splits;          // blocks that share the tokens of a tile of queries
  int tiles;           // of kTileRows queries in a sequence and key head
  int64_t rows;        // queries of a sequence and key head: T * group
  // of each tile of queries, where splits > 1: the parts that it has, and those
  // parts' sums [kTileRows][D], maxima and sums of powers [kTileRows]
  int* parts;
  float* part;
};
constexpr int64_t part_floats(int D) { return int64_t{kTileRows} * (D + 2); }

// Where the tile kernel's operands come from.
enum Source { kPaged, kHalf, kFloat };

// LDS of a block, in bytes: keys [TT][pitch], values [32 DT][pitch] (a copy for each
// part of a split value), of dense rows what is added to their scores (0, or -inf
// where none is seen); later the sums.
constexpr int key_pitch(int DT) { return 64 * DT + 16; }
constexpr int value_pitch(int TT) { return 2 * TT + 16; }
constexpr int tile_bytes(int SRC, int DT, int TT) {
  return (TT * key_pitch(DT) + 32 * DT * value_pitch(TT)) * (SRC == kFloat ? 3 : 1) + (SRC == kPaged ? 0 : TT * 4);
}

// The larger of, or the sum of, the values of lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// Two values as the sum of two halves each.
__device__ __forceinline__ void split2(float x, float y, h2* hi, h2* lo) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  *hi = __builtin_convertvector((f2{x, y}), h2);
  *lo = __builtin_convertvector((f2{x - static_cast<float>((*hi)[0]), y - static_cast<float>((*hi)[1])}), h2);
}

// Two values as the sums of three bf16 each, exactly (a part's rest is exact in
// fp32): word p holds both values' parts p.  Of a value that is not finite, or
// too large for bf16, the second part is NaN.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&word)[3]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    const b2 v = __builtin_convertvector((f2{x, y}), b2);
    word[p] = __builtin_bit_cast(uint32_t, v);
    if (p == 2) break;
    x -= __uint_as_float(word[p] << 16);
    y -= __uint_as_float(word[p] & 0xffff0000u);
  }
}

// c + a b of 32x32x16: of halves, or of bf16 parts.
template <int SRC>
__device__ __forceinline__ f16v product(h8 a, h8 b, f16v c) {
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  if constexpr (SRC == kFloat)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// c + the products of a's and b's parts, the small ones first; those below the
// last part of a value (2^-24) are left out.
template <int SRC, int PA, int PB>
__device__ __forceinline__ f16v product_of_parts(const h8 (&a)[PA], const h8 (&b)[PB], f16v c) {
  constexpr int kMost = (PA > PB ? PA : PB) - 1;
#pragma unroll
  for (int order = kMost; order >= 0; --order)
#pragma unroll
    for (int i = PA - 1; i >= 0; --i)
      if (order - i >= 0 && order - i < PB) c = product<SRC>(a[i], b[order - i], c);
  return c;
}

// Eight values as fragments of their three parts.
__device__ __forceinline__ void split3(const float (&x)[8], h8 (&to)[3]) {
  u4 part[3];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    uint32_t word[3];
    split3(x[i], x[i + 1], word);
#pragma unroll
    for (int p = 0; p < 3; ++p) part[p][i / 2] = word[p];
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) to[p] = __builtin_bit_cast(h8, part[p]);
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
// 8-bit codes and fp16 values are exact as halves.  fp32 queries over pages are the
// sum of two, after a power of two for each row that brings its largest to 2^14,
// which keeps 22 bits.  fp32 queries over fp32 states, states and weights are sums of three
// bf16 each, exactly, with fp32's exponents: no row shares a power of two with
// another, or a value with its row, so that each keeps its own bits (values below
// 2^-110 those that fp32's normal numbers hold); of nine products the three of
// 2^-24 and less are left out.  Over pages, a weight carries
// its page's scale, over a power of two of the largest such product that the query
// has met: by what it weighs, not by what it sees, so that a page of large scale
// without weight takes no bits from the others.  Weights of fp16 queries are rounded
// to fp16 (half a step of the output's type; in two halves the chunk below takes 315
// us).  They are 2^8 times as large, so that one below 2^-22 of the largest keeps
// 2^-33 of that: over states, an error below half of fp16's smallest step for
// values up to 256.
//
// Bound by the vector units beside the products: 32 x 64 scores a wave take some
// 300 vector instructions for their softmax against 32 (fp16, 128 values) or 96
// (fp32, 64) products, bringing a tile 120 (codes), 30 (fp16) or 220 (fp32) a
// wave.  2 x 1531 queries of 32 heads of 128 over up to 4099 cached tokens: 255
// us, 455 TFLOP/s; 2 x 3000 over 1500 fp16 states: 220 us, 669 TFLOP/s; 2 x 3380
// of 12 heads of 64 over up to 509 fp32 states: 73 us (67 to 69 in two halves beside the
// block's largest row, which lost rows that a query weighs beside a large one that
// it does not; heads of 80 and 96 take a tenth less than so, of 128 a twentieth).  64 tokens a tile: keys and
// values of 128 take 36 KB, so that two blocks a CU overlap one's loads with the
// other's products; 256 queries a block, for half the loads, gave 256 and 86 us.
//
// A state that is not finite poisons the sums of all queries here (0 times it is
// NaN) where only queries that see it should be: a block whose sums are not finite
// marks its part, and its queries are formed one by one.
template <typename T, class Rows, int SRC, int DT, int TT, bool WIDE>
__global__ void __launch_bounds__(kTileThreads, WIDE && DT <= (SRC == kFloat ? 2 : sizeof(T) == 4 ? 3 : 4) ? 2 : 1)
    attention_tile_kernel(QueryArgs a, Rows rows, TileCut cut) {
  constexpr int PQ = SRC == kFloat ? 3 : sizeof(T) == 4 ? 2 : 1, PK = SRC == kFloat ? 3 : 1, PW = PQ;  // parts
  constexpr int KS = 2 * DT, NS = TT / 32, G = TT / 16;
  constexpr int KP = key_pitch(DT), VP = value_pitch(TT);
  constexpr bool kAhead = SRC != kFloat || DT <= 4;  // (fp32 heads past 128 values leave no registers for it)
  extern __shared__ __attribute__((aligned(16))) char tile_lds[];
  char* lds_k = tile_lds;
  char* lds_v = lds_k + PK * TT * KP;
  float* key_bias = reinterpret_cast<float*>(lds_v + PK * 32 * DT * VP);

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
  each = each < kLeastTiles ? kLeastTiles : each;
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
    if constexpr (PQ == 1) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 16 * s + 8 * hf;
        if constexpr (WIDE) {
          const u4 v = *reinterpret_cast<const u4*>(q + (d < D ? d : 0));
          qf[s][0] = __builtin_bit_cast(h8, d < D ? v : u4{0, 0, 0, 0});
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const T v = q[d + i < D ? d + i : 0];
            qf[s][0][i] = d + i < D ? __builtin_bit_cast(_Float16, v) : static_cast<_Float16>(0.0f);
          }
        }
      }
    } else {
      float x[KS][8], top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 16 * s + 8 * hf;
        if constexpr (WIDE) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const f4 v = *reinterpret_cast<const f4*>(q + (d < D ? d : 0) + 4 * w);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[s][4 * w + i] = d < D ? v[i] : 0.0f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = to_f32(q[d + i < D ? d + i : 0]);
            x[s][i] = d + i < D ? v : 0.0f;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, __builtin_fabsf(x[s][i]));
      }
      if constexpr (SRC == kFloat) {
#pragma unroll
        for (int s = 0; s < KS; ++s) split3(x[s], qf[s]);
      } else {
        top = max_halves(top);
        const int up = 14 + 127 - static_cast<int>(__float_as_uint(top) >> 23);
        cq = ldexpf(a.scale, -up);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            h2 y0, y1;
            split2(ldexpf(x[s][i], up), ldexpf(x[s][i + 1], up), &y0, &y1);
            qf[s][0][i] = y0[0];
            qf[s][0][i + 1] = y0[1];
            qf[s][PQ - 1][i] = y1[0];
            qf[s][PQ - 1][i + 1] = y1[1];
          }
      }
    }
  }

  // ---- from memory: a tile in registers, one tile ahead
  // token tk of 32 lies in row 8 j + 4 h + r, where its score comes out in
  // register 4 j + r of half h: tokens 16 (j / 2) + 8 h + 4 (j % 2) + r
  auto row_of = [](int tk) { return (tk & ~31) | (tk & 16) | (tk & 4) << 1 | (tk & 8) >> 1 | (tk & 3); };
  constexpr int kKeyUnits = SRC == kPaged ? TT * 2 * DT : TT * 4 * DT;  // 16 codes, or 8 values
  constexpr int kVD = SRC == kHalf ? 8 : 4;                             // values of 4 tokens, or 16 codes of a row
  constexpr int kValueUnits = SRC == kPaged ? 32 * DT * G : TT / 4 * (32 * DT / kVD);
  constexpr int UK = (kKeyUnits + kTileThreads - 1) / kTileThreads;
  constexpr int UV = (kValueUnits + kTileThreads - 1) / kTileThreads;
  u4 ck[SRC == kFloat ? 2 * UK : UK], cv[SRC == kPaged ? UV : 4 * UV];
  // (threads past the last unit do it again; values past a head's are whatever
  // lies at its start: against zeros of q, or in rows that are not put out)
  auto key_unit = [&](int i) {
    const int u = tid + kTileThreads * i;
    return kKeyUnits % kTileThreads == 0 || u < kKeyUnits ? u : kKeyUnits - 1;
  };
  auto value_unit = [&](int i) {
    const int u = tid + kTileThreads * i;
    return kValueUnits % kTileThreads == 0 || u < kValueUnits ? u : kValueUnits - 1;
  };
  // dense: eight or four lanes next to each other read a token's values, the
  // next ones the next four tokens'
  auto value_d = [&](int u) { return kVD * (u % (32 / kVD) + 32 / kVD * (u / (32 / kVD * (TT / 4)))); };
  auto value_tokens = [&](int u) { return u / (32 / kVD) % (TT / 4) * 4; };

  // paged: the table's entry (a tile before its codes) and, with its codes, the
  // scales of 16 tokens, of group lane % G
  int entry = 0, page1 = -1;
  float ks1 = 0.0f, vs1 = 0.0f;
  // dense: bit j: any of the block's queries may see token j
  uint64_t word = 0;
  bool sees1 = false;  // whether token `lane` of the tile after may be seen

  auto find_entry = [&](int64_t t0) {
    if constexpr (SRC == kPaged) {
      const int64_t column = (t0 + 16 * (lane % G)) >> __builtin_ctz(rows.a.block);
      entry = rows.a.table[b * rows.a.table_stride + (column < rows.a.columns ? column : rows.a.columns - 1)];
    } else {
      const auto& p = rows.a;
      const int64_t t = t0 + lane;
      sees1 = t < hi && lane < TT;
      if (p.mask && (p.ms[1] == 0 || a.T == 1))  // (past the end: the last, without effect)
        sees1 = (p.mask[b * p.ms[0] + (t < p.S ? t : p.S - 1) * p.ms[2]] != 0) & sees1;
    }
  };
  auto fetch = [&](int64_t t0) {
    if constexpr (SRC == kPaged) {
      const auto& p = rows.a;
      const int64_t t = t0 + 16 * (lane % G);
      page1 = t < hi && t >> __builtin_ctz(p.block) < p.columns && entry < p.pages ? entry : -1;
      const int pages = page1 < 0 ? 0 : page1;  // (page 0's codes, without weight)
      const int64_t sc = int64_t{pages} * p.heads + h, page_bytes = int64_t{p.block} * D;
      ks1 = p.k_scale[sc];
      vs1 = p.v_scale[sc];
      if (p.block >= TT) {
        const int64_t at_page = (int64_t{__builtin_amdgcn_readfirstlane(pages)} * p.heads + h) * page_bytes;
        const int in_page = static_cast<int>(t0 & (p.block - 1));
        const int8_t* k = p.k + at_page + in_page * D;
        const int8_t* v = p.v + at_page + in_page;
#pragma unroll
        for (int i = 0; i < UK; ++i) {
          const int u = key_unit(i), tk = u / (2 * DT), c = 16 * (u % (2 * DT));
          ck[i] = *reinterpret_cast<const u4*>(k + (tk * D + (c < D ? c : 0)));
        }
#pragma unroll
        for (int i = 0; i < UV; ++i) {
          const int u = value_unit(i), d = u / G, g = u % G;
          cv[i] = *reinterpret_cast<const u4*>(v + ((d < D ? d : 0) * p.block + 16 * g));
        }
      } else {
#pragma unroll
        for (int i = 0; i < UK; ++i) {
          const int u = key_unit(i), tk = u / (2 * DT), c = 16 * (u % (2 * DT));
          const int64_t at_page = (int64_t{__shfl(pages, tk / 16, 64)} * p.heads + h) * page_bytes;
          ck[i] = *reinterpret_cast<const u4*>(p.k + at_page + (static_cast<int>((t0 + tk) & (p.block - 1)) * D +
                                                                (c < D ? c : 0)));
        }
#pragma unroll
        for (int i = 0; i < UV; ++i) {
          const int u = value_unit(i), d = u / G, g = u % G;
          const int64_t at_page = (int64_t{__shfl(pages, g, 64)} * p.heads + h) * page_bytes;
          cv[i] = *reinterpret_cast<const u4*>(p.v + at_page + ((d < D ? d : 0) * p.block +
                                                                static_cast<int>((t0 + 16 * g) & (p.block - 1))));
        }
      }
    } else {
      using S = std::conditional_t<SRC == kHalf, __half, float>;
      const auto& p = rows.a;
      word = __ballot(sees1);
      if (word == 0) return;
      // a token that no query of the block may see is not read: in its place,
      // without weight, the first that some do
      const int visible = __builtin_ctzll(word);
      const S* k = static_cast<const S*>(p.k) + b * p.ks[0] + h * p.ks[2] + t0 * p.ks[1];
      const S* v = static_cast<const S*>(p.v) + b * p.vs[0] + h * p.vs[2] + t0 * p.vs[1];
      constexpr int W = SRC == kFloat ? 2 : 1;
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < UK; ++i) {
          const int u = key_unit(i), tk = u / (4 * DT), d = 8 * (u % (4 * DT));
          const S* from = k + (word >> tk & 1 ? tk : visible) * p.ks[1] + (d < D ? d : 0);
#pragma unroll
          for (int w = 0; w < W; ++w) ck[W * i + w] = *reinterpret_cast<const u4*>(from + 4 * w);
        }
#pragma unroll
        for (int i = 0; i < UV; ++i) {
          const int u = value_unit(i), d = value_d(u), tk = value_tokens(u);
          const uint32_t there = static_cast<uint32_t>(word >> tk);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            cv[4 * i + j] = *reinterpret_cast<const u4*>(v + (there >> j & 1 ? tk + j : visible) * p.vs[1] +
                                                         (d < D ? d : 0));
        }
      } else {
        auto bits = [](S x) -> uint32_t {
          if constexpr (SRC == kFloat)
            return __float_as_uint(x);
          else
            return __half_as_ushort(x);
        };
#pragma unroll
        for (int i = 0; i < UK; ++i) {
          const int u = key_unit(i), tk = u / (4 * DT), d = 8 * (u % (4 * DT));
          u4 w[2];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t x = d + e < D ? bits(k[(word >> tk & 1 ? tk : visible) * p.ks[1] + d + e]) : 0u;
            if constexpr (SRC == kFloat)
              w[e / 4][e % 4] = x;
            else
              w[0][e / 2] = e % 2 ? w[0][e / 2] | x << 16 : x;
          }
#pragma unroll
          for (int e = 0; e < W; ++e) ck[W * i + e] = w[e];
        }
#pragma unroll
        for (int i = 0; i < UV; ++i) {
          const int u = value_unit(i), d = value_d(u), tk = value_tokens(u);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            u4 w;
#pragma unroll
            for (int e = 0; e < kVD; ++e) {
              const uint32_t x = d + e < D ? bits(v[(word >> (tk + j) & 1 ? tk + j : visible) * p.vs[1] + d + e]) : 0u;
              if constexpr (SRC == kFloat)
                w[e % 4] = x;
              else
                w[e / 2] = e % 2 ? w[e / 2] | x << 16 : x;
            }
            cv[4 * i + j] = w;
          }
        }
      }
    }
  };
  float m = -3.4028235e38f, l = 0.0f;
  // paged: log2 of the largest weight times page scale that the query has met (a
  // whole number, as m is there; kLeastSize below m at the least), and 2^(m - mv + 8)
  float mv = -3.4028235e38f, size = 256.0f;

  auto stage = [&]() {
    if constexpr (SRC == kPaged) {
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = key_unit(i), tk = u / (2 * DT), c = u % (2 * DT);
        h8* to = reinterpret_cast<h8*>(lds_k + row_of(tk) * KP + 32 * c);
        to[0] = codes_h8(ck[i][0], ck[i][1]);
        to[1] = codes_h8(ck[i][2], ck[i][3]);
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = value_unit(i), d = u / G, g = u % G;
        h8* to = reinterpret_cast<h8*>(lds_v + d * VP + 32 * g);
        to[0] = codes_h8(cv[i][0], cv[i][1]);
        to[1] = codes_h8(cv[i][2], cv[i][3]);
      }
      return;
    }
    if (tid < TT) key_bias[tid] = word >> tid & 1 ? 0.0f : -INFINITY;
    if constexpr (SRC == kHalf) {
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = key_unit(i), tk = u / (4 * DT), c = u % (4 * DT);
        *reinterpret_cast<u4*>(lds_k + row_of(tk) * KP + 16 * c) = ck[i];
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = value_unit(i), d = value_d(u), tk = value_tokens(u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // one value of four tokens
          const uint32_t sel = e % 2 ? 0x07060302u : 0x05040100u;
          typedef uint32_t u2 __attribute__((ext_vector_type(2)));
          const u2 w = {__builtin_amdgcn_perm(cv[(4 * i + 1) % (4 * UV)][e / 2], cv[4 * i % (4 * UV)][e / 2], sel),
                        __builtin_amdgcn_perm(cv[(4 * i + 3) % (4 * UV)][e / 2], cv[(4 * i + 2) % (4 * UV)][e / 2], sel)};
          *reinterpret_cast<u2*>(lds_v + (d + e) * VP + 2 * tk) = w;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < UK; ++i) {
        const int u = key_unit(i), tk = u / (4 * DT), c = u % (4 * DT);
        float x[8];
        h8 part[3];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(ck[(2 * i + e / 4) % (2 * UK)][e % 4]);
        split3(x, part);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *reinterpret_cast<h8*>(lds_k + (p * TT + row_of(tk)) * KP + 16 * c) = part[p];
      }
#pragma unroll
      for (int i = 0; i < UV; ++i) {
        const int u = value_unit(i), d = value_d(u), tk = value_tokens(u);
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // one value of four tokens
          u2 part[3];
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            uint32_t word[3];
            split3(__uint_as_float(cv[(4 * i + j) % (4 * UV)][e]),
                   __uint_as_float(cv[(4 * i + j + 1) % (4 * UV)][e]), word);
#pragma unroll
            for (int p = 0; p < 3; ++p) part[p][j / 2] = word[p];
          }
#pragma unroll
          for (int p = 0; p < 3; ++p) *reinterpret_cast<u2*>(lds_v + (p * 32 * DT + d + e) * VP + 2 * tk) = part[p];
        }
      }
    }
  };

  f16v acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
  // bounds of what the wave's queries see: some of [from, upto), all of [all_from, all_upto)
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
  const bool by_query = rows_masked_by_query(rows, a);
  if (wave * 32 >= count) upto = from = 0;  // (no queries: the wave only helps to bring tiles)

  if (kAhead && lo < hi) {
    find_entry(lo);
    fetch(lo);
    find_entry(lo + TT);
  }
  for (int64_t t0 = lo; t0 < hi; t0 += TT) {
    if (!kAhead) {
      find_entry(t0);
      fetch(t0);
    }
    const bool empty = SRC != kPaged && word == 0;  // the same in all waves
    __syncthreads();  // the tile before is read
    if (!empty) stage();
    const int page = page1;
    const float ks = ks1, vs = page < 0 ? 0.0f : vs1;
    if (kAhead && t0 + TT < hi) {
      fetch(t0 + TT);
      find_entry(t0 + 2 * TT);
    }
    __syncthreads();
    if (empty || t0 >= upto || t0 + TT <= from) continue;
    // what the lane's query sees of its tokens 32 j + 16 k + 8 hf + e: bit 16 j + 8 k + e
    uint32_t seen = 0, groups = 0;  // (groups: bit g: some of tokens 16 g .. 16 g + 15)
    bool tested = t0 < all_from || t0 + TT > all_upto || by_query;
    bool poisoned = false;
    if constexpr (SRC == kPaged) {
      poisoned = __any((__float_as_uint(vs) & 0x7f800000u) == 0x7f800000u);
      tested = tested || poisoned || !__all(page >= 0);
    }
    if (tested) {
      const int64_t below = qs.lo - t0, past = qs.hi - t0;
      const int lo32 = below < 0 ? 0 : below > TT ? TT : static_cast<int>(below);
      const int hi32 = past < 0 ? 0 : past > TT ? TT : static_cast<int>(past);
      uint64_t w = hi32 > lo32 ? ~uint64_t{0} >> (64 - (hi32 - lo32)) << lo32 : 0;  // by token
      if constexpr (SRC == kPaged) {
        const uint64_t pages = __ballot(page >= 0);
#pragma unroll
        for (int g = 0; g < G; ++g)
          if (!(pages >> g & 1)) w &= ~(uint64_t{0xffff} << (16 * g));
      } else {
        w = query_mask(rows, a, b, qt, t0, TT, w);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) groups |= (w >> (16 * g) & 0xffff ? 1u : 0u) << g;
      w >>= 8 * hf;
#pragma unroll
      for (int s = 0; s < 2 * NS; ++s) seen |= (static_cast<uint32_t>(w >> (16 * s)) & 0xffu) << (8 * s);
    }

    float by[G], vg[G], ev[G];  // of a group's tokens: score by, page scale, and its log2, rounded up
    float largest = -INFINITY;  // of the tile's ev
    if constexpr (SRC == kPaged) {
      const uint32_t bits = __float_as_uint(__builtin_fabsf(vs));
      const bool finite = bits < 0x7f800000u;
      const float lane_v = finite ? vs : 0.0f;
      const float lane_e = finite && bits ? static_cast<float>(static_cast<int>(bits >> 23) - 126) : -INFINITY;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        by[g] = cq * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), g));
        vg[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lane_v), g));
        ev[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lane_e), g));
        largest = fmaxf(largest, ev[g]);
      }
      if (poisoned && (groups & static_cast<uint32_t>(__ballot(!finite)))) l = NAN;  // (lane g is of group g)
    }
    {
      // fragments of keys or values are read a batch ahead of their products
      constexpr int KB = DT > 4 || PK > 1 ? 1 : 2, BATCHES = KS / KB;
      constexpr int VB = DT > 4 || DT % 2 || PK > 1 ? 1 : 2, VBATCHES = DT / VB;
      h8 kf[2][KB][PK], vf[2][VB][PK];
      auto read_keys = [&](int j, int batch, h8 (&to)[KB][PK]) {
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
          for (int part = 0; part < PK; ++part)
            to[k][part] = *reinterpret_cast<const h8*>(lds_k + (part * TT + 32 * j + n) * KP + 32 * (batch * KB + k) + 16 * hf);
      };
      auto read_values = [&](int step, int batch, h8 (&to)[VB][PK]) {
#pragma unroll
        for (int i = 0; i < VB; ++i)
#pragma unroll
          for (int part = 0; part < PK; ++part)
            to[i][part] = *reinterpret_cast<const h8*>(lds_v + (part * 32 * DT + 32 * (batch * VB + i) + n) * VP + 32 * step + 16 * hf);
      };
      read_keys(0, 0, kf[0]);
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        f16v s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
        for (int batch = 0; batch < BATCHES; ++batch) {
          const int now = (j * BATCHES + batch) % 2;
          if (batch + 1 < BATCHES)
            read_keys(j, batch + 1, kf[now ^ 1]);
          else
            read_values(2 * j, 0, vf[0]);
#pragma unroll
          for (int k = 0; k < KB; ++k) s = product_of_parts<SRC>(kf[now][k], qf[batch * KB + k], s);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int tk = 32 * j + 16 * (c / 2) + 8 * hf + 4 * (c % 2);
          if constexpr (SRC == kPaged) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * c + e] *= by[(2 * j + c / 2) % G];
          } else {
            const f4 bias = *reinterpret_cast<const f4*>(key_bias + tk);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * c + e] = __builtin_fmaf(s[4 * c + e], cq, bias[e]);
          }
        }
        if (tested) {
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = seen >> (16 * j + e) & 1 ? s[e] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        top = max_halves(top);
        // m follows a row's maximum only where that is kSlack above it: weights are
        // 2^(x - m + 8) <= 2^15 (fp32: 2^(x - m - kSlack)), and few tiles scale the sums
        // again; so does mv
        if constexpr (SRC == kPaged) {
          if (__any(top > fminf(m, mv - largest) + kSlack)) {  // (as if the largest score had the largest scale)
            float early = s[0], late = s[8];
#pragma unroll
            for (int e = 1; e < 8; ++e) {
              early = fmaxf(early, s[e]);
              late = fmaxf(late, s[8 + e]);
            }
            const float sized = fmaxf(early + ev[2 * j % G], late + ev[(2 * j + 1) % G]);
            top = fmaxf(ceilf(top), m);
            const float most = fmaxf(fmaxf(ceilf(max_halves(sized)), top - kLeastSize), mv);
            const float keep = __builtin_amdgcn_exp2f(mv - most);
            l *= __builtin_amdgcn_exp2f(m - top);
            m = top;
            mv = most;
            size = __builtin_amdgcn_exp2f(m - mv + 8.0f);
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[i][e] *= keep;
          }
        } else if (__any(top > m + kSlack)) {
          top = fmaxf(top, m);
          const float keep = __builtin_amdgcn_exp2f(m - top);
          m = top;
          l *= keep;
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][e] *= keep;
        }
        const float less = SRC == kPaged ? m : SRC == kHalf ? m - 8.0f : m + kSlack;
        h8 pf[2][PW];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            w[e] = __builtin_amdgcn_exp2f(s[8 * k + e] - less);
            l += w[e];
          }
          if constexpr (SRC == kPaged) {
            const float vw = sized_by(vg[(2 * j + k) % G], size);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] *= vw;
          }
          if constexpr (SRC == kFloat) {
            split3(w, pf[k]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              h2 p0, p1;
              split2(w[e], w[e + 1], &p0, &p1);
              pf[k][0][e] = p0[0];
              pf[k][0][e + 1] = p0[1];
              if constexpr (PW == 2) {
                pf[k][PW - 1][e] = p1[0];
                pf[k][PW - 1][e + 1] = p1[1];
              }
            }
          }
        }
#pragma unroll
        for (int step = 0; step < 2 * VBATCHES; ++step) {
          const int k = step / VBATCHES, batch = step % VBATCHES;
          if (step + 1 < 2 * VBATCHES)
            read_values(2 * j + (step + 1) / VBATCHES, (step + 1) % VBATCHES, vf[(step + 1) % 2]);
          else if (j + 1 < NS)
            read_keys(j + 1, 0, kf[(j + 1) * BATCHES % 2]);
#pragma unroll
          for (int i = 0; i < VB; ++i)
            acc[batch * VB + i] = product_of_parts<SRC>(vf[step % 2][i], pf[k], acc[batch * VB + i]);
        }
      }
    }
  }

  // the sums by rows, half of them at a time, in LDS
  bool marked = false;
  if constexpr (SRC != kPaged) {
    float any = l * 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) any = __builtin_fmaf(acc[i][e], 0.0f, any);
    marked = any != any;
  }
  marked = __syncthreads_or(marked);
  const int pitch = D + 4;
  float* sums = reinterpret_cast<float*>(tile_lds);
  float* wm = sums + kPutRows * pitch;
  float* wl = wm + kPutRows;
  l = sum_halves(l);
  const float scale = SRC == kPaged ? __builtin_amdgcn_exp2f(mv - m - 8.0f) : 1.0f;
  const int64_t pair = at.z * static_cast<int64_t>(cut.tiles) + tile;
  if (cut.splits > 1 && chunk == 0 && tid == 0) cut.parts[pair] = chunks;
  if (chunks > 1) {
    float* to = cut.part + (pair * cut.splits + chunk) * part_floats(D);
    const int r = wave * 32 + n;
    if (r < count) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int d = 32 * i + 8 * c + 4 * hf;
          const f4 v = f4{acc[i][4 * c], acc[i][4 * c + 1], acc[i][4 * c + 2], acc[i][4 * c + 3]} * scale;
          if (D % 4 == 0) {
            if (d < D) *reinterpret_cast<f4*>(to + r * D + d) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + e < D) to[r * D + d + e] = v[e];
          }
        }
      if (hf == 0) {
        to[kTileRows * D + r] = marked ? NAN : m;
        to[kTileRows * D + kTileRows + r] = l;
      }
    }
    return;
  }
  for (int part = 0; part * kPutRows < count; ++part) {
    const int r = wave * 32 + n - part * kPutRows, here = count - part * kPutRows < kPutRows ? count - part * kPutRows : kPutRows;
    __syncthreads();
    if (r >= 0 && r < here) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int d = 32 * i + 8 * c + 4 * hf;
          const f4 v = f4{acc[i][4 * c], acc[i][4 * c + 1], acc[i][4 * c + 2], acc[i][4 * c + 3]} * scale;
          if (D % 4 == 0) {
            if (d < D) *reinterpret_cast<f4*>(sums + r * pitch + d) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + e < D) sums[r * pitch + d + e] = v[e];
          }
        }
      if (hf == 0) {
        wm[r] = marked ? NAN : m;
        wl[r] = l;
      }
    }
    __syncthreads();
    const Part out{b, h, here, 0, 1, first + part * kPutRows, nullptr, 0, nullptr};
    const bool out_is_there = put_rows<T, kTileThreads>(a, out, sums, pitch, wm, wl, nullptr);
    if constexpr (SRC != kPaged) {  // (no page marks a part)
      if (out_is_there) continue;
      __syncthreads();
      for (int i = wave; i < here; i += kTileThreads / 64) {
        const int64_t at_row = out.first + i;
        one_query<T>(a, rows, b, at_row / a.group, h * a.group + static_cast<int>(at_row % a.group), sums + wave * kMaxHead);
      }
    }
  }
}

// Joins the parts of queries whose tokens were shared by several blocks, a wave a
// query: weights 2^(m_i - max) / sum_i l_i 2^(m_i - max), a lane a part.  A launch
// of its own, so that parts go by ordinary stores and many CUs join them (2 x 100
// queries of 28 heads over up to 2000 tokens: 35 us with it, 101 where the last
// block of a tile joins its parts).
template <typename T, class Rows>
__global__ void __launch_bounds__(kTileThreads) join_parts_kernel(QueryArgs a, Rows rows, TileCut cut) {
  __shared__ float qv[kTileThreads / 64][kMaxHead];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, D = a.D;
  constexpr int kRows = kTileThreads / 64;
  const int64_t unit = blockIdx.x / (kTileRows / kRows);
  const int r = blockIdx.x % (kTileRows / kRows) * kRows + wave;
  const int64_t row = unit % cut.tiles * kTileRows + r, pair = unit / cut.tiles;
  const int parts = cut.parts[unit];
  if (row >= cut.rows || parts <= 1) return;
  const int heads = a.heads / a.group;
  const int64_t b = pair / heads, t = row / a.group;
  const int head = static_cast<int>(pair % heads) * a.group + static_cast<int>(row % a.group);
  const float* from = cut.part + unit * cut.splits * part_floats(D);
  const float* ml = from + kTileRows * D + r;
  const float m = lane < parts ? ml[lane * part_floats(D)] : -INFINITY;
  const float l = lane < parts ? ml[lane * part_floats(D) + kTileRows] : 0.0f;
  if (!std::is_same<Rows, PagedRows>::value && __any(m != m)) {
    one_query<T>(a, rows, b, t, head, qv[wave]);
    return;
  }
  const float w = exp2f(m - wave_max_dpp(m)), sum = wave_sum_dpp(w * l);
  const float by = sum != 0.0f ? w / sum : 0.0f;
  T* y = static_cast<T*>(a.y) + b * a.ys[0] + t * a.ys[1] + head * a.ys[2];
  for (int d = lane; d < D; d += 64) {
    float v = 0.0f;
    for (int i = 0; i < parts; ++i)
      v = __builtin_fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(by), i)),
                         from[i * part_floats(D) + r * D + d], v);
    from_f32(y[d], v);
  }
}

template <typename T, class Rows, int SRC, int DT, int TT, bool WIDE>
static int launch_tiles(const QueryArgs& a, const Rows& rows, int64_t tokens, const char* who) {
  const int64_t queries = int64_t{a.T} * a.group, pairs = a.B * (a.heads / a.group);
  const int64_t tiles = ceil_div(queries, kTileRows);
  TileCut cut{};
  cut.rows = queries;
  // where there are fewer blocks than two a CU, the tokens are cut, into parts
  // of two tiles at least (100 fp32 queries of 12 heads of 128 over 1400 states: 31
  // us; in parts of four tiles 83)
  const int64_t blocks = pairs * tiles, head = (blocks * 4 + 15) / 16 * 16;
  int64_t splits = ceil_div(2 * ctx().num_cus, blocks);
  const int64_t room = (static_cast<int64_t>(kScratchBytes) - head) / 4 / part_floats(a.D) / blocks;
  const int64_t parts = ceil_div(tokens, kLeastTiles * TT);
  splits = splits < parts ? splits : parts;
  splits = splits < kMaxChunks ? splits : kMaxChunks;
  splits = splits < room ? splits : room;
  if (splits < 1) splits = 1;
  cut.parts = static_cast<int*>(ctx().scratch);
  cut.part = reinterpret_cast<float*>(static_cast<char*>(ctx().scratch) + head);
  cut.splits = static_cast<int>(splits);
  cut.tiles = static_cast<int>(tiles);
  const dim3 grid(static_cast<unsigned>(splits), static_cast<unsigned>(tiles), static_cast<unsigned>(pairs));
  KK_TRY(check_xcd_grid(grid, who));
  int64_t bytes = (int64_t{kPutRows} * (a.D + 4) + 2 * kPutRows) * 4;
  if (bytes < tile_bytes(SRC, DT, TT)) bytes = tile_bytes(SRC, DT, TT);
  if (bytes < 4 * kMaxHead * 4) bytes = 4 * kMaxHead * 4;
  if (bytes > 65536) KK_TRY(allow_large_lds(reinterpret_cast<const void*>(attention_tile_kernel<T, Rows, SRC, DT, TT, WIDE>)));
  KK_LAUNCH((attention_tile_kernel<T, Rows, SRC, DT, TT, WIDE>), grid, dim3(kTileThreads), static_cast<unsigned>(bytes),
            ctx().stream, a, rows, cut);
  KK_TRY(check_launch("attention_tile_kernel"));
  if (splits == 1) return KK_OK;
  KK_LAUNCH((join_parts_kernel<T, Rows>), dim3(static_cast<unsigned>(blocks * (kTileRows / (kTileThreads / 64)))),
            dim3(kTileThreads), 0, ctx().stream, a, rows, cut);
  return check_launch("join_parts_kernel");
}

// WIDE: rows of q, and of dense keys and values, take 16-byte accesses.
template <typename T, class Rows, int SRC, bool WIDE>
static int launch_tiles(const QueryArgs& a, const Rows& rows, int64_t tokens, const char* who) {
  return a.D <= 64    ? launch_tiles<T, Rows, SRC, 2, 64, WIDE>(a, rows, tokens, who)
         : a.D <= 96  ? launch_tiles<T, Rows, SRC, 3, 64, WIDE>(a, rows, tokens, who)
         : a.D <= 128 ? launch_tiles<T, Rows, SRC, 4, 64, WIDE>(a, rows, tokens, who)
                      : launch_tiles<T, Rows, SRC, 8, 32, WIDE>(a, rows, tokens, who);
}

template <typename T, class Rows, int SRC>
static int launch_tiles(const QueryArgs& a, const Rows& rows, int64_t tokens, bool wide, const char* who) {
  return wide ? launch_tiles<T, Rows, SRC, true>(a, rows, tokens, who)
              : launch_tiles<T, Rows, SRC, false>(a, rows, tokens, who);
}

// (past the grid's axes: one query a wave)
static bool too_many(const QueryArgs& a) {
  return a.B * (a.heads / a.group) > 65535 || int64_t{a.T} * a.group > int64_t{65535} * kTileRows;
}

bool tiles_paged_try(const QueryArgs& a, const PagedArgs& p, int dtype, int* status) {
  if (p.pages < 1 || p.columns < 1) return false;
  const PagedRows rows{p, a.T, a.D};
  const int64_t capacity = p.columns * p.block;
  const int64_t seen = p.window && p.window < capacity ? p.window + a.T - 1 : capacity;
  const int64_t tokens = seen < capacity ? seen : capacity;
  if (too_many(a)) return false;
  const bool wide = rows_of_16(a.q, a.qs, dtype == KK_F16 ? 2 : 4);
  const char* who = "cache_attention";
  *status = dtype == KK_F16 ? launch_tiles<__half, PagedRows, kPaged>(a, rows, tokens, wide, who)
                            : launch_tiles<float, PagedRows, kPaged>(a, rows, tokens, wide, who);
  return true;
}

bool tiles_dense_try(const QueryArgs& a, const DenseArgs& d, int dtype, int* status) {
  if (d.S < 1 || too_many(a)) return false;
  const int size = dtype == KK_F16 ? 2 : 4;
  const bool wide = a.D % 8 == 0 && d.ks[3] == 1 && d.vs[3] == 1 && rows_of_16(a.q, a.qs, size) &&
                   rows_of_16(d.k, d.ks, size) && rows_of_16(d.v, d.vs, size);
  const char* who = "cross_attention";
  *status = dtype == KK_F16
                ? launch_tiles<__half, DenseRows<__half>, kHalf>(a, DenseRows<__half>{d}, d.S, wide, who)
                : launch_tiles<float, DenseRows<float>, kFloat>(a, DenseRows<float>{d}, d.S, wide, who);
  return true;
}

}  // namespace kk
