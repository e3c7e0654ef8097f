// Attention of few queries over an encoder's states: a step of single tokens.
#include "kk_attention.h"

namespace kk {

constexpr int kStateThreads = 256;
constexpr int kStateWaves = kStateThreads / 64;

// The sum over LANES neighbouring lanes, in each of them: pairs, quads, eights,
// sixteens by lane moves, then by exchange of rows and of halves.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_move<0xB1, 0xF>(v, 0.0f);
  v += dpp_move<0x4E, 0xF>(v, 0.0f);
  v += dpp_move<0x141, 0xF>(v, 0.0f);
  if constexpr (LANES >= 16) v += dpp_move<0x140, 0xF>(v, 0.0f);
  if constexpr (LANES >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (LANES >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}

// out = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m) for at most R queries of a
// key head: bound by the states' way from memory, with a product and a sum for
// each value and query, so the vector units carry it, in fp32 throughout.  A
// token lies over LANES lanes of 16 bytes, U times 64 / LANES tokens are a
// wave's step, and the next step's are loaded while it works.  Each group of
// LANES lanes keeps a maximum, sum and outputs of its own tokens; they are joined
// at the end.  32 sequences of 1500 to 2999 states: 93 us for 12 heads of 64 in
// fp32 (4.7 TB/s of the 6.2 that reading alone reaches; 193 us in tiles for the
// matrix cores, which bring states to halves for one query in 128), 71 us for 8
// key heads of 128 under 32 query heads in fp16 (4.1 TB/s).
template <typename T, int LANES, int R, int U>
__global__ void __launch_bounds__(kStateThreads, 2) few_states_kernel(QueryArgs a, DenseRows<T> rows, Cut cut) {
  constexpr int VEC = 16 / sizeof(T), TOK = 64 / LANES, STEP = TOK * U;
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  extern __shared__ __attribute__((aligned(16))) float lds[];
  Unit u;
  if (!find_unit(rows, cut, &u)) return;
  const DenseArgs& p = rows.a;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int D = a.D, count = static_cast<int>(cut.rows), tok = lane / LANES;
  const int d = lane % LANES * VEC, d0 = d < D ? d : 0;  // (lanes past the head: its start, against zeros of q)

  u4 q[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = r < count ? r : count - 1, t = row / a.group, head = u.h * a.group + row % a.group;
    const T* at = static_cast<const T*>(a.q) + u.b * a.qs[0] + t * a.qs[1] + head * a.qs[2] + d0;
    q[r] = *reinterpret_cast<const u4*>(at);
    if (d >= D) q[r] = u4{0, 0, 0, 0};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) q[r][e] = __float_as_uint(__uint_as_float(q[r][e]) * a.scale);
    }
  }
  const T* kb = static_cast<const T*>(p.k) + u.b * p.ks[0] + u.h * p.ks[2] + d0;
  const T* vb = static_cast<const T*>(p.v) + u.b * p.vs[0] + u.h * p.vs[2] + d0;
  const uint8_t* mask = p.mask ? p.mask + u.b * p.ms[0] : nullptr;

  u4 k1[U], v1[U];
  uint8_t see1[U];
  auto load = [&](int64_t j0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t j = j0 + i * TOK + tok, at = j < u.hi ? j : u.hi - 1;
      k1[i] = *reinterpret_cast<const u4*>(kb + at * p.ks[1]);
      v1[i] = *reinterpret_cast<const u4*>(vb + at * p.vs[1]);
      see1[i] = mask ? mask[at * p.ms[2]] : 1;
    }
  };
  float acc[R][VEC], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -3.4028235e38f;
    l[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[r][e] = 0.0f;
  }
  const int64_t first = u.lo + wave * STEP;
  if (first < u.hi) load(first);
  for (int64_t j0 = first; j0 < u.hi; j0 += kStateWaves * STEP) {
    u4 k[U], v[U];
    bool sees[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      sees[i] = j0 + i * TOK + tok < u.hi && see1[i] != 0;
      k[i] = k1[i];
      v[i] = sees[i] ? v1[i] : u4{0, 0, 0, 0};
    }
    if (j0 + kStateWaves * STEP < u.hi) load(j0 + kStateWaves * STEP);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[U], top = m[r];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4)
            x = __builtin_fmaf(__uint_as_float(q[r][e]), __uint_as_float(k[i][e]), x);
          else
            x = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, uint32_t{q[r][e]}),
                                       __builtin_bit_cast(h2, uint32_t{k[i][e]}), x, false);
        }
        x = lanes_sum<LANES>(x);
        if constexpr (sizeof(T) == 2) x *= a.scale;
        s[i] = sees[i] ? x : -INFINITY;
        top = fmaxf(top, s[i]);
      }
      const float keep = __builtin_amdgcn_exp2f(m[r] - top);
      m[r] = top;
      l[r] *= keep;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[r][e] *= keep;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float w = __builtin_amdgcn_exp2f(s[i] - top);
        l[r] += w;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float x;
          if constexpr (sizeof(T) == 4) {
            x = __uint_as_float(v[i][e % 4]);
          } else {
            const h2 pair = __builtin_bit_cast(h2, uint32_t{v[i][e / 2]});
            x = static_cast<float>(pair[e % 2]);
          }
          acc[r][e] = __builtin_fmaf(w, x, acc[r][e]);
        }
      }
    }
  }

  // the groups of a wave, then the waves in LDS
  const int pitch = (D + 7) / 4 * 4;
  float* wm = lds;                            // [waves][R], then [R] the block's
  float* wl = wm + (kStateWaves + 1) * R;
  float* sums = wl + (kStateWaves + 1) * R;   // [waves][R][pitch]
  sums += (4 - 2 * (kStateWaves + 1) * R % 4) % 4;
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int off = LANES; off < 64; off <<= 1) {
      const float mo = __shfl_xor(m[r], off, 64), top = fmaxf(m[r], mo), keep = __builtin_amdgcn_exp2f(m[r] - top);
      m[r] = top;
      l[r] *= keep;
      l[r] += __shfl_xor(l[r], off, 64);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        acc[r][e] *= keep;
        acc[r][e] += __shfl_xor(acc[r][e], off, 64);
      }
    }
    if (lane == 0) {
      wm[wave * R + r] = m[r];
      wl[wave * R + r] = l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = wm[r], sum = 0.0f;
    for (int w = 1; w < kStateWaves; ++w) top = fmaxf(top, wm[w * R + r]);
    for (int w = 0; w < kStateWaves; ++w) sum += wl[w * R + r] * exp2f(wm[w * R + r] - top);
    if (threadIdx.x == 0) {
      wm[kStateWaves * R + r] = top;
      wl[kStateWaves * R + r] = sum;
    }
    const float by = exp2f(m[r] - top);
    if (tok == 0 && d < D) {
#pragma unroll
      for (int e = 0; e < VEC; e += 4)
        *reinterpret_cast<f4*>(sums + (wave * R + r) * pitch + d + e) =
            f4{acc[r][e], acc[r][e + 1], acc[r][e + 2], acc[r][e + 3]} * by;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * D; i += kStateThreads) {
    float* at = sums + (i / D) * pitch + i % D;
    float x = at[0];
    for (int w = 1; w < kStateWaves; ++w) x += at[w * R * pitch];
    at[0] = x;
  }
  __syncthreads();
  const int64_t slot = int64_t{count} * (D + 2);
  const Part part{u.b, u.h, count, u.chunk, u.chunks, 0, cut.part + u.slot * slot, slot * cut.heads,
                  cut.arrived + u.b * cut.heads + u.h};
  put_rows<T, kStateThreads>(a, part, sums, pitch, wm + kStateWaves * R, wl + kStateWaves * R, sums + R * pitch);
}

template <typename T, int LANES, int R>
static int launch_states(const QueryArgs& a, const DenseRows<T>& rows, int64_t queries) {
  constexpr int U = R > 4 ? 2 : 4;  // (eight queries' sums leave registers for two tokens a lane in flight)
  // chunks of four steps at least, of one where each takes eight queries' products
  // (7 queries over 700 states: 33 us in chunks of 8 steps, 25 in 4, 22 in 1)
  Cut cut;
  int64_t blocks;
  KK_TRY(plan_cut(a.B, a.heads / a.group, queries, a.D, rows.a.S, R > 4 ? 1 : 4, int64_t{8} * ctx().num_cus, &cut, &blocks,
                  "cross_attention"));
  // the waves' sums; then, beside the first's, the chunks' weights
  const int pitch = (a.D + 7) / 4 * 4;
  const size_t sums = size_t{kStateWaves} * R * pitch, joined = size_t{R} * (pitch + 2 * kMaxChunks);
  const size_t bytes = 4 * (2 * (kStateWaves + 1) * R + 4 + (sums > joined ? sums : joined));
  KK_LAUNCH((few_states_kernel<T, LANES, R, U>), dim3(static_cast<unsigned>(blocks)), dim3(kStateThreads), bytes,
            ctx().stream, a, rows, cut);
  return check_launch("few_states_kernel");
}

template <typename T, int LANES>
static int launch_states(const QueryArgs& a, const DenseRows<T>& rows, int64_t queries) {
  return queries == 1   ? launch_states<T, LANES, 1>(a, rows, queries)
         : queries <= 2 ? launch_states<T, LANES, 2>(a, rows, queries)
         : queries <= 4 ? launch_states<T, LANES, 4>(a, rows, queries)
                        : launch_states<T, LANES, 8>(a, rows, queries);
}

template <typename T>
static int launch_states(const QueryArgs& a, const DenseRows<T>& rows, int64_t queries) {
  const int lanes = a.D * static_cast<int>(sizeof(T)) / 16;
  if (lanes <= 8) return launch_states<T, 8>(a, rows, queries);
  if (lanes <= 16) return launch_states<T, 16>(a, rows, queries);
  if constexpr (sizeof(T) == 4)
    if (lanes > 32) return launch_states<T, 64>(a, rows, queries);
  return launch_states<T, 32>(a, rows, queries);
}

bool few_dense_try(const QueryArgs& a, const DenseArgs& d, int dtype, int* status) {
  const int64_t queries = int64_t{a.T} * a.group;
  const int size = dtype == KK_F16 ? 2 : 4;
  // up to eight queries of a key head, as long as they see the same states and
  // a head's values take 16-byte accesses
  if (queries > 8 || d.S < 1 || a.D * size % 16 || (a.D > 1 && (d.ks[3] != 1 || d.vs[3] != 1)) ||
      !rows_of_16(a.q, a.qs, size) || !rows_of_16(d.k, d.ks, size) || !rows_of_16(d.v, d.vs, size) ||
      (d.mask && d.ms[1] != 0 && a.T > 1))
    return false;
  *status = dtype == KK_F16 ? launch_states<__half>(a, DenseRows<__half>{d}, queries)
                            : launch_states<float>(a, DenseRows<float>{d}, queries);
  return true;
}

}  // namespace kk
