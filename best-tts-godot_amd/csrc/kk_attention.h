// What the attention kernels share: their operands, what a query sees, the cut
// of long sequences over blocks and the join of the parts.
#pragma once

#include "kk_decode.h"

namespace kk {

constexpr int kMaxHead = 256;
// Weights over pages are kept beside 2^mv, mv = max log2(weight's power of two
// times its page's scale), but not below 2^-kLeastSize of the largest power of two
// (values whose scale is below that may lose bits).
constexpr float kLeastSize = 100.0f;
// The product of a page's scale and the power of two that its weights are kept
// by; past the largest value those weights are zero, and stay so.
__device__ __forceinline__ float sized_by(float scale, float by) {
  return __builtin_amdgcn_fmed3f(scale * by, -3.4028235e38f, 3.4028235e38f);
}

// Queries and outputs: [B, T, heads, D], group query heads a key head.
struct QueryArgs {
  const void* q;
  void* y;
  int64_t qs[3], ys[3];
  int64_t B;
  int T, heads, group, D;
  float scale;  // times log2 e: the softmax is formed from powers of two
};

// Keys and values of one piece each: [B, S, key heads, D].
struct DenseArgs {
  const void *k, *v;
  int64_t ks[4], vs[4];
  int64_t S;
  const void* lengths;
  int lengths_dt;
  int64_t lengths_st;
  const uint8_t* mask;
  int64_t ms[3];
};

struct PagedArgs {
  const int8_t *k, *v;
  const float *k_scale, *v_scale;
  const int32_t* table;
  int64_t table_stride, pages, columns;
  const void *lengths, *counts;
  int lengths_dt, counts_dt;
  int64_t lengths_st, counts_st, window;
  int heads, block;
};

// What the query t of sequence b sees, and the score of one token.
template <typename T>
struct DenseRows {
  DenseArgs a;
  __device__ Seen seen(int64_t b, int64_t) const {
    int64_t n = a.S;
    if (a.lengths) {
      const int64_t l = load_index(a.lengths, a.lengths_dt, b * a.lengths_st);
      n = l < 0 ? 0 : (l < n ? l : n);
    }
    return Seen{0, n};
  }
  __device__ Seen span(int64_t b) const { return seen(b, 0); }  // of all its queries
  __device__ bool sees(int64_t b, int64_t t, int64_t j) const {
    return !a.mask || a.mask[b * a.ms[0] + t * a.ms[1] + j * a.ms[2]] != 0;
  }
  __device__ float key(int64_t b, int h, int64_t j, int d) const {
    return to_f32(static_cast<const T*>(a.k)[b * a.ks[0] + j * a.ks[1] + h * a.ks[2] + d * a.ks[3]]);
  }
  __device__ float value(int64_t b, int h, int64_t j, int d) const {
    return to_f32(static_cast<const T*>(a.v)[b * a.vs[0] + j * a.vs[1] + h * a.vs[2] + d * a.vs[3]]);
  }
};

struct PagedRows {
  PagedArgs a;
  int T, D;
  __device__ int64_t count(int64_t b) const {  // of b's queries that are there
    if (!a.counts) return T;
    const int64_t c = load_index(a.counts, a.counts_dt, b * a.counts_st);
    return c < 0 ? 0 : (c < T ? c : T);
  }
  __device__ Seen span(int64_t b) const {  // of all its queries
    const int64_t n = count(b);
    return Seen{seen(b, 0).lo, n ? seen(b, n - 1).hi : 0};
  }
  __device__ Seen seen(int64_t b, int64_t t) const {
    const int64_t n = count(b);
    const int64_t len = load_index(a.lengths, a.lengths_dt, b * a.lengths_st);
    const int64_t place = (len < 0 ? 0 : len) - n + t;
    return seen_tokens(t < n ? place : -1, a.window, a.columns * a.block);
  }
  __device__ int64_t page(int64_t b, int64_t j) const {
    const int64_t p = a.table[b * a.table_stride + j / a.block];
    return p < a.pages ? p : -1;
  }
  __device__ bool sees(int64_t b, int64_t, int64_t j) const { return page(b, j) >= 0; }
  __device__ float key(int64_t b, int h, int64_t j, int d) const {
    const int64_t p = page(b, j) * a.heads + h;
    return static_cast<float>(a.k[(p * a.block + j % a.block) * D + d]) * a.k_scale[p];
  }
  __device__ float value(int64_t b, int h, int64_t j, int d) const {
    const int64_t p = page(b, j) * a.heads + h;
    return static_cast<float>(a.v[(p * D + d) * a.block + j % a.block]) * a.v_scale[p];
  }
};

// Eight codes as halves, exactly: a byte with its sign turned over is the low
// half of 1024 + 128 + code, from which a packed sum takes 1152.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
__device__ __forceinline__ h8 codes_h8(uint32_t lo, uint32_t hi) {
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

// One wave a query: a lane scores one of 64 tokens, then owns every 64th
// value of the output.  Right for every size, stride and type; qv is the
// wave's own, kMaxHead floats of LDS.
template <typename T, class Rows>
__device__ __forceinline__ void one_query(const QueryArgs& a, const Rows& rows, int64_t b, int64_t t, int head, float* qv) {
  const int lane = threadIdx.x % 64, h = head / a.group;
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + t * a.qs[1] + head * a.qs[2];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int d = lane; d < a.D; d += 64) qv[d] = to_f32(q[d]);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const Seen w = rows.seen(b, t);
  float m = -INFINITY, l = 0.0f, acc[kMaxHead / 64] = {};
  for (int64_t j0 = w.lo; j0 < w.hi; j0 += 64) {
    const int64_t j = j0 + lane;
    const bool sees = j < w.hi && rows.sees(b, t, j);
    float s = 0.0f;
    if (sees)
      for (int d = 0; d < a.D; ++d) s = __builtin_fmaf(qv[d], rows.key(b, h, j, d), s);
    s = sees ? s * a.scale : -INFINITY;
    const float next = fmaxf(fmaxf(m, wave_max(s)), -3.4028235e38f);
    const float keep = exp2f(m - next), p = exp2f(s - next);
    m = next;
    l = l * keep + wave_sum(p);
#pragma unroll
    for (int i = 0; i < kMaxHead / 64; ++i) acc[i] *= keep;
    uint64_t live = __ballot(sees);
    while (live) {
      const int e = __builtin_ctzll(live);
      live &= live - 1;
      const float pe = __shfl(p, e, 64);
#pragma unroll
      for (int i = 0; i < kMaxHead / 64; ++i)
        if (lane + 64 * i < a.D) acc[i] = __builtin_fmaf(pe, rows.value(b, h, j0 + e, lane + 64 * i), acc[i]);
    }
  }
  T* y = static_cast<T*>(a.y) + b * a.ys[0] + t * a.ys[1] + head * a.ys[2];
#pragma unroll
  for (int i = 0; i < kMaxHead / 64; ++i)
    if (lane + 64 * i < a.D) from_f32(y[lane + 64 * i], l != 0.0f ? acc[i] / l : 0.0f);
}

// ---------------------------------------------- few queries, many tokens
// A step reads a whole cache for a few queries: sequences are cut into chunks
// so that every CU has some.  How long they are is known on the device only,
// so the blocks find their chunk there: with n_b steps of kStep tokens in
// sequence b, a chunk is c = max(least, ceil(sum n_b / units)) steps, one and
// the same for all, so that ragged batches load the CUs evenly: `units` blocks
// for each CU to have a few, or, once their chunks would pass kLongChunk steps,
// `most`, which even out what some take longer.  At most most + B chunks come
// of that, times the key heads: the grid.  (24 sequences of up to 8000 tokens,
// 4 key heads of 96: 54 us in chunks of 8 steps, 49 in 16; 12 heads of 96: 104
// us with two blocks a CU, 97 with four.)
struct Cut {
  int64_t B;
  int heads;           // key heads
  int64_t units, most; // chunks to aim for, for each head: of ordinary calls, of long ones
  int64_t least;       // steps of a chunk at least
  int64_t rows;        // queries of a key head: T * group
  float* part;         // a slot of rows * (D + 2) floats a block
  int* arrived;        // a counter for each sequence and head, zero between launches
};

struct Unit {
  int64_t b, lo, hi;   // tokens of the chunk; lo a multiple of kStep
  int h, chunk, chunks;
  int64_t slot;        // of the sequence's first chunk and this head; the next chunk's is `heads` later
};

__device__ __forceinline__ int64_t uniform(int64_t v) {  // the same in all lanes: in scalar registers
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>(uint64_t{hi} << 32 | lo);
}

// This block's chunk (the same in every wave); false where it has none.
template <class Rows>
__device__ __forceinline__ bool find_unit(const Rows& rows, const Cut& cut, Unit* u) {
  const int lane = threadIdx.x % 64;
  const int64_t id = blockIdx.x / cut.heads;
  u->h = static_cast<int>(blockIdx.x % cut.heads);
  auto steps_of = [&](int64_t b) -> int64_t {
    if (b >= cut.B) return 0;
    const Seen s = rows.span(b);
    return ceil_div(s.hi - (s.lo / kStep) * kStep, kStep);
  };
  const int64_t mine = steps_of(lane);
  int64_t total = mine;
  for (int64_t b = 64 + lane; b < cut.B; b += 64) total += steps_of(b);
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  const int64_t c = chunk_size(total, cut.units, cut.most, cut.least);
  int64_t before = 0;
  for (int64_t b0 = 0; b0 < cut.B; b0 += 64) {
    const int64_t b = b0 + lane, n = b0 ? steps_of(b) : mine;
    const int64_t each = chunk_steps(n, c), chunks = b >= cut.B ? 0 : chunk_count(n, c);
    int64_t upto = chunks;
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t o = __shfl_up(upto, off, 64);
      if (lane >= off) upto += o;
    }
    const uint64_t past = __ballot(before + upto > id);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int64_t first = before + __shfl(upto - chunks, at, 64);
      u->b = b0 + at;
      u->chunks = static_cast<int>(uniform(__shfl(chunks, at, 64)));
      u->chunk = static_cast<int>(uniform(id - first));
      u->slot = uniform(first) * cut.heads + u->h;
      const Seen s = rows.span(u->b);
      const int64_t lo = (s.lo / kStep) * kStep, size = __shfl(each, at, 64) * kStep;
      u->lo = uniform(lo + u->chunk * size);
      u->hi = uniform(u->lo + size < s.hi ? u->lo + size : s.hi);
      return true;
    }
    before += __shfl(upto, 63, 64);
  }
  return false;
}

// Chunks and grid for `most` tokens a sequence at the most and `aim` blocks;
// *blocks the grid.
// Where scratch or counters do not hold a slot for each, sequences stay whole.
inline int plan_cut(int64_t B, int heads, int64_t rows, int D, int64_t most, int64_t least, int64_t aim, Cut* cut,
                    int64_t* blocks, const char* who) {
  const int64_t slots = static_cast<int64_t>(kScratchBytes / 4) / (rows * (D + 2)) / heads;
  cut->B = B;
  cut->heads = heads;
  cut->rows = rows;
  cut->least = least;
  cut->units = ceil_div(aim, heads);
  cut->most = ceil_div(8 * ctx().num_cus, heads);
  if (cut->most < cut->units) cut->most = cut->units;
  cut->part = static_cast<float*>(ctx().scratch);
  cut->arrived = ctx().row_counters;
  int64_t n = grid_chunks(B, most, cut->most, least);
  if (n > slots) {
    cut->most = slots - B;
    if (cut->units > cut->most) cut->units = cut->most;
    n = slots;
  }
  if (cut->units < 1 || B * heads > kRowCounters) {
    cut->units = cut->most = 1;
    cut->least = int64_t{1} << 40;
    n = B;
  }
  if (n * heads > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many sequences and heads", who);
  *blocks = n * heads;
  return KK_OK;
}

// What a block puts out: `rows` queries of key head h of sequence b from `first`
// on, over one of `chunks` parts of their tokens; slots of rows * (D + 2) floats
// from `slots` on, `next` apart, and the parts' counter.
struct Part {
  int64_t b;
  int h, rows, chunk, chunks;
  int64_t first;
  float* slots;
  int64_t next;
  int* arrived;
};

// The block's sums of its queries, `pitch` floats apart in LDS (acc, not yet
// divided; m[r] and l[r] a row's maximum and sum of powers of two), to the
// output, or to the block's slot and, by the block that comes last of a row's,
// joined from there: always in the chunks' order.  The order of slot and
// counter is that of the row reductions: stores that write through to where
// all XCDs read, a wait for them, then the count; no whole cache is written
// back.  Called by all threads, after a barrier; `weights` holds
// 2 * chunks * rows floats.  False, with nothing put out, where there is one part
// and its first maximum is NaN: the caller has marked it as not to be used.
template <typename T, int THREADS>
__device__ __forceinline__ bool put_rows(const QueryArgs& a, const Part& u, const float* acc, int pitch,
                                         const float* m, const float* l, float* weights) {
  const int rows = u.rows, D = a.D;
  auto out = [&](int r, int d, float v) {
    const int64_t row = u.first + r, t = row / a.group, head = u.h * a.group + row % a.group;
    from_f32(static_cast<T*>(a.y)[u.b * a.ys[0] + t * a.ys[1] + head * a.ys[2] + d], v);
  };
  __shared__ int last;  // of a row's blocks to arrive
  if (u.chunks == 1) {
    if (m[0] != m[0]) return false;
    if (D % 4 == 0) {
      const int D4 = D / 4;
      for (int i = threadIdx.x; i < rows * D4; i += THREADS) {
        const int r = i / D4, d = 4 * (i - r * D4);
        const float by = l[r] != 0.0f ? 1.0f / l[r] : 0.0f;
        const f4 v = *reinterpret_cast<const f4*>(acc + r * pitch + d) * by;
        const int64_t row = u.first + r, t = row / a.group, head = u.h * a.group + row % a.group;
        T* y = static_cast<T*>(a.y) + u.b * a.ys[0] + t * a.ys[1] + head * a.ys[2] + d;
        T o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) from_f32(o[e], v[e]);
        __builtin_memcpy(y, o, sizeof o);
      }
      return true;
    }
    for (int i = threadIdx.x; i < rows * D; i += THREADS) {
      const int r = i / D, d = i - r * D;
      out(r, d, l[r] != 0.0f ? acc[r * pitch + d] / l[r] : 0.0f);
    }
    return true;
  }
  auto put = [&](float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  auto get = [&](const float* p) {
    return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  float* mine = u.slots + u.chunk * u.next;
  for (int i = threadIdx.x; i < rows * D; i += THREADS) {
    const int r = i / D, d = i - r * D;
    put(mine + i, acc[r * pitch + d]);
  }
  for (int r = threadIdx.x; r < rows; r += THREADS) {
    put(mine + rows * D + r, m[r]);
    put(mine + rows * D + rows + r, l[r]);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(u.arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == u.chunks - 1;
  __syncthreads();
  if (!last) return true;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  if (threadIdx.x == 0) __hip_atomic_store(u.arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // weights[i][r] = 2^(m_i - max) / sum_i l_i 2^(m_i - max), from all parts' m and
  // l at once (one after the other, each would wait its whole way)
  float* sums = weights + u.chunks * rows;
  for (int i = threadIdx.x; i < u.chunks * rows; i += THREADS) {
    const float* at = u.slots + (i / rows) * u.next + rows * D + i % rows;
    weights[i] = get(at);
    sums[i] = get(at + rows);
  }
  __syncthreads();
  for (int r = threadIdx.x / 64; r < rows; r += THREADS / 64) {  // a wave a row, a lane a part
    const int i = threadIdx.x % 64;
    const float mi = i < u.chunks ? weights[i * rows + r] : -INFINITY;
    const float w = exp2f(mi - wave_max_dpp(mi));
    const float sum = wave_sum_dpp(i < u.chunks ? w * sums[i * rows + r] : 0.0f);
    if (i < u.chunks) weights[i * rows + r] = sum != 0.0f ? w / sum : 0.0f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += THREADS) {
    const int r = i / D, d = i - r * D;
    float sum = 0.0f;
    auto some = [&](int j0, auto batch) {  // (past the last part: it again, without weight)
      constexpr int N = decltype(batch)::value;
      float x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = get(u.slots + (j0 + j < u.chunks ? j0 + j : u.chunks - 1) * u.next + i);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j0 + j < u.chunks) sum = __builtin_fmaf(weights[(j0 + j) * rows + r], x[j], sum);
    };
    if (u.chunks <= 4) {
      some(0, std::integral_constant<int, 4>{});
    } else {
      for (int j0 = 0; j0 < u.chunks; j0 += 16) some(j0, std::integral_constant<int, 16>{});
    }
    out(r, d, sum);
  }
  return true;
}

// ------------------------------------------------------- many queries
constexpr int kTileThreads = 256;
constexpr int kTileRows = 128;  // queries of a block: 32 a wave
struct TileCut {
  int splits;          // blocks that share the tokens of a tile of queries
  int tiles;           // of kTileRows queries in a sequence and key head
  int64_t rows;        // queries of a sequence and key head: T * group
  int row_waves;       // waves of a block that have queries of their own (over 4-bit codes)
  // of each tile of queries, where splits > 1: the parts that it has, and those
  // parts' sums [kTileRows][D], maxima and sums of powers [kTileRows]
  int* parts;
  float* part;
};
constexpr int64_t part_floats(int D) { return int64_t{kTileRows} * (D + 2); }

// The larger of, or the sum of, the values of lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
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
  if (!std::is_base_of<PagedRows, Rows>::value && __any(m != m)) {  // (no page marks a part)
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

// How many blocks share the tokens of each of `blocks` tiles of queries that see
// at most `tokens`, in parts of `least` tokens at the least: where there are fewer
// blocks than `wanted` (two a CU: 100 fp32 queries of 12 heads of 128 over 1400 states: 31 us; in
// parts of four tiles 83).
inline void plan_parts(int64_t blocks, int64_t tokens, int64_t least, int D, int64_t wanted, TileCut* cut) {
  const int64_t head = (blocks * 4 + 15) / 16 * 16;
  int64_t splits = ceil_div(wanted, blocks);
  const int64_t room = (static_cast<int64_t>(kScratchBytes) - head) / 4 / part_floats(D) / blocks;
  const int64_t parts = ceil_div(tokens, least);
  splits = splits < parts ? splits : parts;
  splits = splits < kMaxChunks ? splits : kMaxChunks;
  splits = splits < room ? splits : room;
  cut->splits = static_cast<int>(splits < 1 ? 1 : splits);
  cut->parts = static_cast<int*>(ctx().scratch);
  cut->part = reinterpret_cast<float*>(static_cast<char*>(ctx().scratch) + head);
}

// Whether rows of an operand start at multiples of 16 bytes.
inline bool rows_of_16(const void* p, const int64_t* strides, int size) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] * size % 16) return false;
  return true;
}

// Entry points of the kernels; false where a call is not theirs.
bool few_paged_try(const QueryArgs& a, const PagedArgs& p, int dtype, int* status);
bool few_dense_try(const QueryArgs& a, const DenseArgs& d, int dtype, int* status);
bool tiles_paged_try(const QueryArgs& a, const PagedArgs& p, int dtype, int* status);
bool tiles_dense_try(const QueryArgs& a, const DenseArgs& d, int dtype, int* status);

}  // namespace kk
