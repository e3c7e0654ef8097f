// A token drawn from each row of logits with a given number, after temperature,
// top-k, top-p and min-p.
//
// The tokens in order (larger logits first, equal ones by index) weigh w = 2^-y,
// y = (max - x) log2(e) / temperature.  Each of the three limits keeps a first part
// of them, and the token drawn is the first whose running sum passes u times what
// is kept, so that all four are one search: the first token in order whose running
// count or sum reaches a target.  A row is not sorted for it.  Its y are counted
// into bins of one width, which also sum the weights; only the tokens of the bins
// that a target can fall into (some hundred of 131072) are put in order.
//
// A token next to a border must not fall on the other side of it by rounding, and
// sums must not hang on the order of atomics: y is formed in 64 bits, and within a
// bin of at most 2^-5 a weight is 2^-(lower edge) (1 - d), d a whole number of
// 2^-34ths from a Taylor series in 64 bits, so a bin's sum is exact in whole
// numbers, with its count in one 64-bit atomic of LDS.
#include "kk_decode.h"

namespace kk {

constexpr double kFarthest = 64.0;  // past 2^-64 a weight counts as none (a row of 2^17 sums them to 2^-47)
constexpr int kOnes = 34;           // a weight within its bin: 2^34 - d
constexpr int kDefShift = 46;       // a bin: (tokens << 46) + sum of d, both exact up to 2^17 tokens
constexpr int kMostTokens = 1 << 17;
constexpr int kCandidates = 2048;
constexpr int kDrawThreads = 256;
// A row in one block: short ones in 256 threads and 512 bins, others in 1024 and
// 2048 (a row of 1025 tokens: 9.4 us against 12.3).
constexpr int kShortRow = 4096;
// Longer ones in blocks of kSlice tokens, in four launches: their largest and
// smallest logits; their bins, which the last block of a row sums up and asks; their
// candidates; and a block a row that draws from those.  64 rows of 131072: 5.8, 27, 12
// and 7.3 us in the kernels, 51 in a recorded call; the row is read three times from caches
// (34 MB), and what takes the time are the steps one after another: a bin's atomic a
// token, the sums over 2048 bins, the searches.
constexpr int kSlice = 16384;
constexpr int kMostSlices = kMostTokens / kSlice;
constexpr int kWide = 2048;         // bins of these, and of rows in one block past kShortRow

// The bins that the limits and the drawn number can fall into, as far as the bins'
// sums say, and what is known beforehand.
struct Asked {
  int64_t k;       // tokens kept by top-k; live where all are
  double p, m, u;  // p >= 1, m <= 0: no limit
  double far;      // largest y kept by min-p
  int bin[6];      // of k; first and last of p; of m; first and last of u (-1: none)
};

struct SampleArgs {
  const void* x;
  int64_t xs, V, B;
  const float *u, *temperature, *top_p, *min_p;
  const void* top_k;
  int k_dt;
  int64_t u_st, t_st, k_st, p_st, m_st;
  int32_t* tokens;
  float* logs;      // or NULL
  int slices;       // blocks of a row
  // of rows over several blocks, [B] each:
  float2* range;    // [slices] largest and smallest
  uint64_t* cells;  // [slices][kWide + 1] bins
  double* mass;     // [kWide + 1] what comes before a bin
  int* count;       // [kWide + 2]
  Asked* asked;
  uint64_t* found;  // [kCandidates]
  int* counters;    // [2]: blocks that arrived, and candidates; zero between calls
};

// What a row's numbers ask for.
struct RowRule {
  float top;       // its largest logit
  double c;        // log2(e) / temperature
  double inv, width;
  bool greedy;
};

template <typename T>
__device__ __forceinline__ float as_logit(T v) {
  const float x = to_f32(v);
  return x != x ? -INFINITY : x + 0.0f;  // (-0 is 0)
}
template <typename T>
__device__ __forceinline__ float logit(const SampleArgs& a, int64_t b, int64_t i) {
  return as_logit(static_cast<const T*>(a.x)[b * a.xs + i]);
}
// f(logit, token) for the tokens [lo, hi) of row b, 16 bytes a load and two loads
// a thread in flight.
template <int THREADS, typename T, class F>
__device__ __forceinline__ void each_logit(const SampleArgs& a, int64_t b, int64_t lo, int64_t hi, F f) {
  constexpr int VEC = 16 / sizeof(T), U = 2;
  struct __attribute__((packed, aligned(sizeof(T)))) Some {
    T v[VEC];
  };
  const T* x = static_cast<const T*>(a.x) + b * a.xs;
  for (int64_t i0 = lo + threadIdx.x * VEC; i0 < hi; i0 += THREADS * VEC * U) {
    Some v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t i = i0 + k * (THREADS * VEC);
      if (i + VEC <= hi) v[k] = *reinterpret_cast<const Some*>(x + i);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t i = i0 + k * (THREADS * VEC);
      if (i + VEC <= hi) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(as_logit(v[k].v[e]), i + e);
      } else {
        for (int64_t e = i; e < hi; ++e) f(as_logit(x[e]), e);
      }
    }
  }
}
// Larger logits have smaller keys.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t w = __float_as_uint(x);
  return w >> 31 ? w : ~w & 0x7fffffffu;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k : ~k & 0x7fffffffu); }

__device__ __forceinline__ double far_of(const RowRule& r, float x) {
  return x == r.top ? 0.0 : (static_cast<double>(r.top) - static_cast<double>(x)) * r.c;
}
template <int BINS>
__device__ __forceinline__ int bin_of(const RowRule& r, double y) {
  if (!(y < kFarthest)) return BINS;
  const double b = y * r.inv;
  return b < BINS - 1 ? static_cast<int>(b) : BINS - 1;
}
// 2^34 (1 - 2^-t), t = y - lower edge, by its series, t <= 64 / BINS, to the term
// below 2^-36.
template <int BINS>
__device__ __forceinline__ uint32_t deficit(const RowRule& r, double y, int bin) {
  constexpr double kLn2 = 0.69314718055994530942, kUnit = static_cast<double>(int64_t{1} << kOnes);
  constexpr double k1 = kUnit * kLn2, k2 = -k1 * kLn2 / 2, k3 = -k2 * kLn2 / 3, k4 = -k3 * kLn2 / 4, k5 = -k4 * kLn2 / 5,
                   k6 = -k5 * kLn2 / 6, k7 = -k6 * kLn2 / 7;
  double t = fma(-static_cast<double>(bin), r.width, y);
  t = t > 0.0 ? t : 0.0;
  double d = k5;
  if constexpr (BINS < kWide) d = fma(fma(k7, t, k6), t, k5);
  d = fma(d, t, k4);
  d = fma(d, t, k3);
  d = fma(d, t, k2);
  d = fma(d, t, k1);
  return static_cast<uint32_t>(fma(d, t, 0.5));
}
__device__ __forceinline__ double edge_weight(const RowRule& r, int bin) { return exp2(-static_cast<double>(bin) * r.width); }

template <int BINS>
__device__ __forceinline__ RowRule rule_of(const SampleArgs& a, int64_t b, float top, float least) {
  RowRule r;
  const float t = a.temperature ? a.temperature[b * a.t_st] : 1.0f;
  r.top = top;
  r.greedy = !(t > 0.0f);
  r.c = r.greedy ? 0.0 : 1.44269504088896340736 / static_cast<double>(t);
  const double all = far_of(r, least);
  const double span = all < kFarthest ? all : kFarthest;
  r.inv = span > 0.0 ? BINS / span : 0.0;
  r.width = span / BINS;
  if (!(r.inv < 1e300)) r.inv = r.width = 0.0;
  return r;
}

template <int BINS>
struct SampleShared {
  uint64_t cells[(BINS > kCandidates ? BINS : kCandidates) + 1];  // bins' counts and sums; then the candidates
  uint64_t sums[kCandidates];     // running sums of the candidates' 2^34 - d
  double mass[BINS + 1];          // before a bin
  int count[BINS + 2];
  uint16_t bin[kCandidates];
  uint64_t part[16];
  double dpart[16];
  int n, at, last;
  double value;
};

// ------------------------------------------------------------ over a block
template <int THREADS, typename T>
__device__ __forceinline__ T block_scan(T v, T* part, T* all) {  // up to and including this thread
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (int off = 1; off < 64; off <<= 1) {
    const T o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  T before = 0, sum = 0;
  for (int i = 0; i < THREADS / 64; ++i) {
    if (i == wave) before = sum;
    sum += part[i];
  }
  *all = sum;
  return v + before;
}

// The largest and smallest of the threads' values.
template <int THREADS>
__device__ __forceinline__ float2 block_range(float top, float least, double* part) {
  top = wave_max_dpp(top);
  least = -wave_max_dpp(-least);
  float2* p = reinterpret_cast<float2*>(part);
  __syncthreads();
  if (threadIdx.x % 64 == 0) p[threadIdx.x / 64] = make_float2(top, least);
  __syncthreads();
  for (int i = 0; i < THREADS / 64; ++i) {
    top = fmaxf(top, p[i].x);
    least = fminf(least, p[i].y);
  }
  return make_float2(top, least);
}
// The largest and smallest logit of tokens [lo, hi) that are not -inf.
template <int THREADS, typename T>
__device__ __forceinline__ float2 find_range(const SampleArgs& a, int64_t b, int64_t lo, int64_t hi, double* part) {
  float top = -INFINITY, least = INFINITY;
  each_logit<THREADS, T>(a, b, lo, hi, [&](float x, int64_t) {
    top = fmaxf(top, x);
    least = fminf(least, x == -INFINITY ? INFINITY : x);
  });
  return block_range<THREADS>(top, least, part);
}

template <int THREADS, int BINS, typename T>
__device__ __forceinline__ void fill_bins(const SampleArgs& a, int64_t b, int64_t lo, int64_t hi, const RowRule& r,
                                          uint64_t* cells) {
  for (int i = threadIdx.x; i <= BINS; i += THREADS) cells[i] = 0;
  __syncthreads();
  each_logit<THREADS, T>(a, b, lo, hi, [&](float x, int64_t) {
    if (x == -INFINITY) return;
    const double y = far_of(r, x);
    const int bin = bin_of<BINS>(r, y);
    const uint64_t one = (uint64_t{1} << kDefShift) + (bin < BINS ? deficit<BINS>(r, y, bin) : 0u);
    atomicAdd(reinterpret_cast<unsigned long long*>(&cells[bin]), static_cast<unsigned long long>(one));
  });
  __syncthreads();
}

// From the bins' counts and sums of d, what comes before each bin: tokens, and
// weight.  get(bin, &n, &d).
template <int THREADS, int BINS, class Get>
__device__ __forceinline__ void sum_bins(const RowRule& r, SampleShared<BINS>& s, Get get) {
  constexpr int EACH = BINS / THREADS;
  int64_t n[EACH], tokens = 0, all;
  double m[EACH], weight = 0.0, total;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int bin = threadIdx.x * EACH + i;
    uint64_t d;
    get(bin, &n[i], &d);
    const int64_t ones = (n[i] << kOnes) - static_cast<int64_t>(d);
    m[i] = n[i] ? edge_weight(r, bin) * (static_cast<double>(ones) * (1.0 / (int64_t{1} << kOnes))) : 0.0;
    tokens += n[i];
    weight += m[i];
  }
  int64_t n_far = 0;
  if (threadIdx.x == THREADS - 1) {
    uint64_t d;
    get(BINS, &n_far, &d);
  }
  tokens = block_scan<THREADS, int64_t>(tokens, reinterpret_cast<int64_t*>(s.part), &all) - tokens;
  weight = block_scan<THREADS, double>(weight, s.dpart, &total) - weight;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int bin = threadIdx.x * EACH + i;
    s.count[bin] = static_cast<int>(tokens);
    s.mass[bin] = weight;
    tokens += n[i];
    weight += m[i];
  }
  if (threadIdx.x == THREADS - 1) {
    s.count[BINS] = static_cast<int>(tokens);
    s.mass[BINS] = weight;
    s.count[BINS + 1] = static_cast<int>(tokens + n_far);
  }
  __syncthreads();
}

// The first bin whose end fulfils `reaches`, which later ends then do too; the last
// one where none does.  Each wave finds it for itself in two looks at 64 ends.
template <int BINS, class Reaches>
__device__ __forceinline__ int first_bin(Reaches reaches) {
  constexpr int EACH = BINS / 64;
  const int lane = threadIdx.x % 64;
  const uint64_t rough = __ballot(reaches((lane + 1) * EACH));
  if (!rough) return BINS - 1;
  const int from = static_cast<int>(__builtin_ctzll(rough)) * EACH;
  return from + static_cast<int>(__builtin_ctzll(__ballot(lane >= EACH - 1 || reaches(from + lane + 1))));
}

template <int BINS>
__device__ __forceinline__ Asked ask(const SampleArgs& a, int64_t b, const RowRule& r, SampleShared<BINS>& s) {
  Asked q;
  const int64_t live = s.count[BINS + 1];
  int64_t k = a.top_k ? load_index(a.top_k, a.k_dt, b * a.k_st) : 0;
  q.k = k > 0 && k < live ? k : live;
  const float p = a.top_p ? a.top_p[b * a.p_st] : 1.0f, m = a.min_p ? a.min_p[b * a.m_st] : 0.0f, u = a.u[b * a.u_st];
  q.p = p < 1.0f ? (p > 0.0f ? p : 0.0) : 1.0;
  q.m = m > 0.0f ? (m < 1.0f ? m : 1.0) : 0.0;
  q.u = u > 0.0f ? (u < 0x1.fffffep-1f ? u : 0x1.fffffep-1f) : 0.0;
  constexpr double kLess = 1.0 - 1e-12, kMore = 1.0 + 1e-12;
  double lo = s.mass[BINS], hi = lo;
  for (int i = 0; i < 6; ++i) q.bin[i] = -1;
  // (k within the far tokens, which weigh nothing, cuts nothing off)
  if (q.k < live && q.k <= s.count[BINS]) {
    const int64_t want = q.k;
    q.bin[0] = first_bin<BINS>([&](int i) { return s.count[i] >= want; });
    lo = s.mass[q.bin[0]];
    hi = s.mass[q.bin[0] + 1];
  }
  if (q.p < 1.0) {
    const double t0 = q.p * lo * kLess, t1 = q.p * hi * kMore;
    q.bin[1] = first_bin<BINS>([&](int i) { return s.mass[i] >= t0; });
    q.bin[2] = first_bin<BINS>([&](int i) { return s.mass[i] >= t1; });
    const double end = s.mass[q.bin[2] + 1];
    lo = s.mass[q.bin[1]];
    hi = end < hi ? end : hi;
  }
  q.far = INFINITY;
  if (q.m > 0.0) {
    q.far = -log2(q.m);
    const int bin = bin_of<BINS>(r, q.far);
    if (bin < BINS) {
      q.bin[3] = bin;
      lo = s.mass[bin] < lo ? s.mass[bin] : lo;
      hi = s.mass[bin + 1] < hi ? s.mass[bin + 1] : hi;
    }
  }
  const double t0 = q.u * lo * kLess, t1 = q.u * hi * kMore;
  q.bin[4] = first_bin<BINS>([&](int i) { return s.mass[i] > t0; });
  q.bin[5] = first_bin<BINS>([&](int i) { return s.mass[i] > t1; });
  return q;
}

__device__ __forceinline__ bool wanted(const Asked& q, int bin) {
  return bin == q.bin[0] || bin == q.bin[3] || (bin >= q.bin[1] && bin <= q.bin[2]) || (bin >= q.bin[4] && bin <= q.bin[5]);
}

__device__ __forceinline__ void put_token(const SampleArgs& a, int64_t b, int64_t token, double y, double kept) {
  a.tokens[b] = static_cast<int32_t>(token);
  if (a.logs) a.logs[b] = static_cast<float>(-y * 0.69314718055994530942 - log(kept));
}

// The token from the `n` candidates in s.cells: all tokens of the wanted bins.  By
// the first kDrawThreads threads alone; the others have left (some hundred
// candidates: fewer waves wait for each other).
template <int BINS>
__device__ __forceinline__ void draw_from(const SampleArgs& a, int64_t b, const RowRule& r, const Asked& q,
                                          SampleShared<BINS>& s, const double* mass, const int* count, int n) {
  constexpr int THREADS = kDrawThreads;
  int size = 64;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += THREADS) s.cells[i] = ~uint64_t{0};
  __syncthreads();
  for (int run = 2; run <= size; run *= 2)
    for (int step = run / 2; step > 0; step /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += THREADS) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const uint64_t x = s.cells[lo], y = s.cells[hi];
        if ((x > y) == ((lo & run) == 0)) {
          s.cells[lo] = y;
          s.cells[hi] = x;
        }
      }
      // steps up to 64 stay within a wave's 128 cells, and a wave's LDS accesses in order
      const int next = step > 1 ? step / 2 : run;
      if (step > 64 || next > 64)
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  __syncthreads();
  // running sums of 2^34 - d over all candidates
  constexpr int EACH = kCandidates / THREADS;
  uint64_t ones[EACH], mine = 0, all;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = threadIdx.x * EACH + i;
    ones[i] = 0;
    if (at < n) {
      const double y = far_of(r, of_key(static_cast<uint32_t>(s.cells[at] >> 32)));
      const int bin = bin_of<BINS>(r, y);
      s.bin[at] = static_cast<uint16_t>(bin);
      ones[i] = (uint64_t{1} << kOnes) - deficit<BINS>(r, y, bin);
    }
    mine += ones[i];
  }
  mine = block_scan<THREADS, uint64_t>(mine, s.part, &all) - mine;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = threadIdx.x * EACH + i;
    mine += ones[i];
    if (at < n) s.sums[at] = mine;
  }
  if (threadIdx.x == 0) s.at = n;
  __syncthreads();
  // of candidate `at`: tokens up to and including it, and their weight
  auto upto = [&](int at, int64_t* rank) {
    const int bin = s.bin[at];
    int lo = 0, hi = at;  // the bin's first candidate
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (s.bin[mid] < bin)
        lo = mid + 1;
      else
        hi = mid;
    }
    *rank = count[bin] + (at - lo) + 1;
    const uint64_t in_bin = s.sums[at] - (lo ? s.sums[lo - 1] : 0);
    return mass[bin] + edge_weight(r, bin) * (static_cast<double>(in_bin) * (1.0 / (int64_t{1} << kOnes)));
  };
  double run[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = threadIdx.x + i * THREADS;
    int64_t rank = 0;
    run[i] = at < n ? upto(at, &rank) : 0.0;
    if (at < n && q.bin[0] >= 0 && rank == q.k) s.value = run[i];
  }
  __syncthreads();
  double kept = q.bin[0] >= 0 ? s.value : mass[BINS];
  // the first candidate whose running weight fulfils `reaches`
  auto first = [&](auto reaches) {
    __syncthreads();
    if (threadIdx.x == 0) s.at = n - 1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = threadIdx.x + i * THREADS;
      if (at < n && reaches(run[i], at)) atomicMin(&s.at, at);
    }
    __syncthreads();
    return s.at;
  };
  auto weight_of = [&](int at) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (threadIdx.x + i * THREADS == at) s.value = run[i];
    __syncthreads();
    return s.value;
  };
  if (q.p < 1.0) {
    const double want = q.p * kept;
    const double end = weight_of(first([&](double w, int at) { return s.bin[at] >= q.bin[1] && w >= want; }));
    kept = end < kept ? end : kept;
  }
  if (q.bin[3] >= 0) {
    // the last of its bin that is kept, or what comes before the bin
    const int cut = first([&](double, int at) {
      return s.bin[at] > q.bin[3] || (s.bin[at] == q.bin[3] && far_of(r, of_key(static_cast<uint32_t>(s.cells[at] >> 32))) > q.far);
    });
    const bool none = s.bin[cut] < q.bin[3] ||
                      (s.bin[cut] == q.bin[3] && !(far_of(r, of_key(static_cast<uint32_t>(s.cells[cut] >> 32))) > q.far));
    const int last = none ? cut : cut - 1;  // (the last candidate of all where none is cut off)
    double end = mass[q.bin[3]];
    if (last >= 0 && s.bin[last] == q.bin[3]) end = weight_of(last);
    kept = end < kept ? end : kept;
  }
  const double want = q.u * kept;
  const int drawn = first([&](double w, int at) { return s.bin[at] >= q.bin[4] && w > want; });
  if (threadIdx.x == 0) {
    const uint64_t c = s.cells[drawn];
    put_token(a, b, static_cast<int64_t>(c & 0xffffffffu), far_of(r, of_key(static_cast<uint32_t>(c >> 32))), kept);
  }
}

// The same where the wanted bins hold more tokens than there is room for: for each
// target in turn its bin, then the keys of the bin's tokens digit by digit, each over the
// whole row, then which of the equal ones.  That is so for many equal logits, and where
// a finite logit far below the others (a mask of -1e4, or of the type's lowest value)
// makes bins 2^-5 of a power of two wide and most of the others lie in a few of them: of
// 131072 with a deviation of 0.5, 330 to 540 us for 64 rows, against 65 to 85 with a mask of
// -inf; with a deviation of 3 as fast as with it.
template <int THREADS, int BINS, typename T>
__device__ __forceinline__ void draw_slowly(const SampleArgs& a, int64_t b, const RowRule& r, const Asked& q,
                                            SampleShared<BINS>& s) {
  constexpr double kUnit = 1.0 / (int64_t{1} << kOnes);
  uint64_t* const n = s.cells;  // of a digit: tokens, then their 2^34 - d
  double kept = s.mass[BINS];
#pragma unroll 1
  for (int target = 0; target < 3; ++target) {  // top-k, top-p, the drawn token
    if (target == 0 && q.bin[0] < 0) continue;
    if (target == 1 && !(q.p < 1.0)) continue;
    if (target == 2 && q.bin[3] >= 0) {  // min-p
      uint64_t ones = 0, all;
      for (int64_t i = threadIdx.x; i < a.V; i += THREADS) {
        const float x = logit<T>(a, b, i);
        if (x == -INFINITY) continue;
        const double y = far_of(r, x);
        if (bin_of<BINS>(r, y) == q.bin[3] && !(y > q.far)) ones += (uint64_t{1} << kOnes) - deficit<BINS>(r, y, q.bin[3]);
      }
      block_scan<THREADS, uint64_t>(ones, s.part, &all);
      const double end = s.mass[q.bin[3]] + edge_weight(r, q.bin[3]) * (static_cast<double>(all) * kUnit);
      kept = end < kept ? end : kept;
    }
    const double want = target == 1 ? q.p * kept : q.u * kept;
    auto reaches = [&](int64_t tokens, double w) {
      return target == 0 ? tokens >= q.k : target == 1 ? w >= want : w > want;
    };
    const int bin = first_bin<BINS>([&](int i) { return reaches(s.count[i], s.mass[i]); });
    const double before = s.mass[bin], by = edge_weight(r, bin);
    auto weight = [&](uint64_t ones) { return before + by * (static_cast<double>(ones) * kUnit); };
    uint32_t key = 0;
    int64_t rank = s.count[bin], here = 0;  // tokens before the key, and its own
    uint64_t sum = 0;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = threadIdx.x; i < 512; i += THREADS) n[i] = 0;
      __syncthreads();
      for (int64_t i = threadIdx.x; i < a.V; i += THREADS) {
        const float x = logit<T>(a, b, i);
        if (x == -INFINITY) continue;
        const uint32_t k = key_of(x);
        if (shift < 24 && (k ^ key) >> (shift + 8)) continue;
        const double y = far_of(r, x);
        if (bin_of<BINS>(r, y) != bin) continue;
        const int digit = k >> shift & 255u;
        atomicAdd(reinterpret_cast<unsigned long long*>(&n[digit]), 1ull);
        atomicAdd(reinterpret_cast<unsigned long long*>(&n[256 + digit]),
                  static_cast<unsigned long long>((uint64_t{1} << kOnes) - deficit<BINS>(r, y, bin)));
      }
      __syncthreads();
      int digit = 0, last = 0;
      for (; digit < 256; ++digit) {  // (all threads alike)
        if (!n[digit]) continue;
        last = digit;
        if (reaches(rank + static_cast<int64_t>(n[digit]), weight(sum + n[256 + digit]))) break;
        rank += n[digit];
        sum += n[256 + digit];
      }
      if (digit == 256) {  // none does, by a rounding: the last
        digit = last;
        rank -= n[last];
        sum -= n[256 + last];
      }
      key |= static_cast<uint32_t>(digit) << shift;
      here = n[digit];
    }
    // which of the equal ones
    const float x = of_key(key);
    const double y = far_of(r, x);
    const uint64_t each = (uint64_t{1} << kOnes) - deficit<BINS>(r, y, bin);
    int64_t lo = 1, hi = here;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (reaches(rank + mid, weight(sum + each * mid)))
        hi = mid;
      else
        lo = mid + 1;
    }
    if (target < 2) {
      const double end = weight(sum + each * lo);
      kept = end < kept ? end : kept;
      continue;
    }
    // its place: each thread counts a piece of the row
    const int64_t piece = ceil_div(a.V, THREADS), i0 = threadIdx.x * piece, i1 = i0 + piece < a.V ? i0 + piece : a.V;
    int64_t mine = 0, all;
    for (int64_t i = i0; i < i1; ++i) mine += logit<T>(a, b, i) == x;
    const int64_t to = block_scan<THREADS, int64_t>(mine, reinterpret_cast<int64_t*>(s.part), &all);
    if (lo <= to - mine || lo > to) continue;
    lo -= to - mine;
    for (int64_t i = i0; i < i1; ++i)
      if (logit<T>(a, b, i) == x && --lo == 0) put_token(a, b, i, y, kept);
  }
}

// From n <= 64 E candidates by their order, without sorting them: for each the block
// counts and sums those of its bin before it (THREADS / 64 E threads each), then one
// wave looks.
template <int THREADS, int E, int BINS>
__device__ __forceinline__ void draw_few(const SampleArgs& a, int64_t b, const RowRule& r, const Asked& q, SampleShared<BINS>& s,
                                         const uint64_t* cells, const double* mass, const int* count, int n) {
  constexpr int SLOTS = 64 * E, EACH = THREADS / SLOTS;
  uint64_t* const all = s.sums;
  uint64_t* const weights = s.sums + SLOTS;
  double* const runs = reinterpret_cast<double*>(s.sums + 2 * SLOTS);
  int* const ranks = reinterpret_cast<int*>(s.sums + 3 * SLOTS);
  const int slot = threadIdx.x / EACH, part = threadIdx.x % EACH;
  const uint64_t its = slot < n ? cells[slot] : ~uint64_t{0};
  const double its_y = slot < n ? far_of(r, of_key(static_cast<uint32_t>(its >> 32))) : 0.0;
  const int its_bin = slot < n ? bin_of<BINS>(r, its_y) : BINS;
  uint64_t in_bin = slot < n && part == 0 ? (uint64_t{1} << kOnes) - deficit<BINS>(r, its_y, its_bin) : 0;
  int before = 0;
  if (part == 0) {
    all[slot] = its;
    weights[slot] = in_bin;
    s.bin[slot] = static_cast<uint16_t>(its_bin);
  }
  const double bin_mass = mass[its_bin], bin_weight = edge_weight(r, its_bin);
  const int bin_count = count[its_bin];
  __syncthreads();
  for (int i = part; i < n; i += EACH) {
    const bool less = all[i] < its && s.bin[i] == its_bin;
    in_bin += less ? weights[i] : 0;
    before += less;
  }
#pragma unroll
  for (int off = EACH / 2; off > 0; off >>= 1) {
    in_bin += __shfl_xor(in_bin, off, 64);
    before += __shfl_xor(before, off, 64);
  }
  if (part == 0) {
    runs[slot] = bin_mass + bin_weight * (static_cast<double>(in_bin) * (1.0 / (int64_t{1} << kOnes)));
    ranks[slot] = bin_count + before + 1;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  uint64_t cell[E];
  double y[E], run[E];
  int bin[E], rank[E];
  bool mine[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = lane + 64 * e;
    mine[e] = at < n;
    cell[e] = all[at];
    bin[e] = s.bin[at];
    run[e] = runs[at];
    rank[e] = ranks[at];
    y[e] = mine[e] ? far_of(r, of_key(static_cast<uint32_t>(cell[e] >> 32))) : 0.0;
  }
  // the first and the last cell of those that `fulfil` (~0 and 0: none)
  auto first = [&](auto fulfils) {
    uint64_t best = ~uint64_t{0};
#pragma unroll
    for (int e = 0; e < E; ++e) best = mine[e] && fulfils(e) && cell[e] < best ? cell[e] : best;
    for (int off = 32; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor(best, off, 64);
      best = o < best ? o : best;
    }
    return best;
  };
  auto last = [&](auto fulfils) {
    uint64_t best = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) best = mine[e] && fulfils(e) && cell[e] > best ? cell[e] : best;
    for (int off = 32; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor(best, off, 64);
      best = o > best ? o : best;
    }
    return best;
  };
  auto run_of = [&](uint64_t best) {
    double w = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t at = __ballot(mine[e] && cell[e] == best);
      if (at) w = __shfl(run[e], static_cast<int>(__builtin_ctzll(at)), 64);
    }
    return w;
  };
  double kept = mass[BINS];
  if (q.bin[0] >= 0) kept = run_of(first([&](int e) { return rank[e] >= q.k && bin[e] >= q.bin[0]; }));
  if (q.p < 1.0) {
    const double want = q.p * kept;
    uint64_t at = first([&](int e) { return bin[e] >= q.bin[1] && run[e] >= want; });
    if (at == ~uint64_t{0}) at = last([&](int e) { return bin[e] <= q.bin[2]; });
    const double end = run_of(at);
    kept = end < kept ? end : kept;
  }
  if (q.bin[3] >= 0) {
    const uint64_t at = last([&](int e) { return bin[e] == q.bin[3] && !(y[e] > q.far); });
    const double end = at == 0 ? mass[q.bin[3]] : run_of(at);
    kept = end < kept ? end : kept;
  }
  const double want = q.u * kept;
  uint64_t at = first([&](int e) { return bin[e] >= q.bin[4] && run[e] > want; });
  if (at == ~uint64_t{0}) at = last([&](int e) { return bin[e] <= q.bin[5]; });
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (mine[e] && cell[e] == at) put_token(a, b, static_cast<int64_t>(at & 0xffffffffu), y[e], kept);
}

// The token from the wanted bins' n tokens, of which up to kCandidates are in `cells`.
template <int THREADS, int BINS, typename T>
__device__ __forceinline__ void draw(const SampleArgs& a, int64_t b, const RowRule& r, const Asked& q, SampleShared<BINS>& s,
                                     const uint64_t* cells, const double* mass, const int* count, int n) {
  if (n <= 64) return draw_few<THREADS, 1>(a, b, r, q, s, cells, mass, count, n);
  if (n <= 128) return draw_few<THREADS, 2>(a, b, r, q, s, cells, mass, count, n);
  if (n <= kCandidates) {
    if (threadIdx.x >= kDrawThreads) return;
    if (cells != s.cells)
      for (int i = threadIdx.x; i < n; i += kDrawThreads) s.cells[i] = cells[i];
    draw_from(a, b, r, q, s, mass, count, n);
    return;
  }
  if (mass != s.mass) {
    for (int i = threadIdx.x; i <= BINS + 1; i += THREADS) {
      if (i <= BINS) s.mass[i] = mass[i];
      s.count[i] = count[i];
    }
    __syncthreads();
  }
  draw_slowly<THREADS, BINS, T>(a, b, r, q, s);
}

// Rows of which nothing is left, and rows whose largest logit is taken; false
// where there is more to do.
template <int THREADS, typename T>
__device__ __forceinline__ bool draw_simply(const SampleArgs& a, int64_t b, const RowRule& r, int* first) {
  if (r.top == -INFINITY) {
    if (threadIdx.x == 0) {
      a.tokens[b] = -1;
      if (a.logs) a.logs[b] = -INFINITY;
    }
    return true;
  }
  if (!r.greedy) return false;
  if (threadIdx.x == 0) *first = 0x7fffffff;
  __syncthreads();
  int at = 0x7fffffff;
  each_logit<THREADS, T>(a, b, 0, a.V, [&](float x, int64_t i) {
    if (x == r.top && i < at) at = static_cast<int>(i);
  });
  if (at != 0x7fffffff) atomicMin(first, at);
  __syncthreads();
  if (threadIdx.x == 0) {
    a.tokens[b] = *first;
    if (a.logs) a.logs[b] = 0.0f;
  }
  return true;
}

// f(cell) for the tokens [lo, hi) of wanted bins: those between a logit a little
// beyond the wanted bins' ends are looked at in 64 bits.
template <int THREADS, int BINS, typename T, class F>
__device__ __forceinline__ void each_candidate(const SampleArgs& a, int64_t b, int64_t lo, int64_t hi, const RowRule& r,
                                               const Asked& q, F f) {
  int least = BINS, most = -1;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    if (q.bin[i] < 0) continue;
    least = q.bin[i] < least ? q.bin[i] : least;
    most = q.bin[i] > most ? q.bin[i] : most;
  }
  // y in [least width, (most + 1) width]: x = top - y / c, a bin and 2^-20 of the size wider
  const double by = r.c > 0.0 ? 1.0 / r.c : 0.0, slack = (fabs(static_cast<double>(r.top)) + kFarthest * by) * 0x1p-20;
  const bool all = !(r.c > 0.0) || !(slack < 1e30) || r.inv == 0.0;
  const float high = all ? INFINITY : static_cast<float>(r.top - (least - 1) * r.width * by + slack);
  const float low = all || most >= BINS - 1 ? -INFINITY : static_cast<float>(r.top - (most + 2) * r.width * by - slack);
  each_logit<THREADS, T>(a, b, lo, hi, [&](float x, int64_t i) {
    if (x == -INFINITY || x < low || x > high) return;
    if (wanted(q, bin_of<BINS>(r, far_of(r, x)))) f(uint64_t{key_of(x)} << 32 | static_cast<uint32_t>(i));
  });
}

// A block a row: short rows, in one launch.
template <int THREADS, int BINS, typename T>
__global__ void __launch_bounds__(THREADS) sample_row_kernel(SampleArgs a) {
  __shared__ SampleShared<BINS> s;
  const int64_t b = blockIdx.x;
  const float2 range = find_range<THREADS, T>(a, b, 0, a.V, s.dpart);
  const RowRule r = rule_of<BINS>(a, b, range.x, range.y);
  if (draw_simply<THREADS, T>(a, b, r, &s.at)) return;
  fill_bins<THREADS, BINS, T>(a, b, 0, a.V, r, s.cells);
  sum_bins<THREADS>(r, s, [&](int bin, int64_t* n, uint64_t* d) {
    const uint64_t w = s.cells[bin];
    *n = static_cast<int64_t>(w >> kDefShift);
    *d = w & ((uint64_t{1} << kDefShift) - 1);
  });
  const Asked q = ask(a, b, r, s);
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  each_candidate<THREADS, BINS, T>(a, b, 0, a.V, r, q, [&](uint64_t cell) {
    const int at = atomicAdd(&s.n, 1);
    if (at < kCandidates) s.cells[at] = cell;
  });
  __syncthreads();
  draw<THREADS, BINS, T>(a, b, r, q, s, s.cells, s.mass, s.count, s.n);
}

// ------------------------------------------------- a row over several blocks
// What blocks hand to the last of their row goes past the caches of their XCD, both
// ways, and is there before the block is counted: no cache is written back or
// emptied for it (an acquire of the whole GPU's scope took the last block 8 to 20 us).
template <typename T>
__device__ __forceinline__ void put_shared(T* p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ T get_shared(const T* p) {
  return __hip_atomic_load(const_cast<T*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool arrives_last(int* arrived, int blocks, int* last) {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (threadIdx.x == 0) {
    *last = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == blocks - 1;
    if (*last) put_shared(arrived, 0);
  }
  __syncthreads();
  return *last;
}

// Two blocks share a CU where bins are counted, with 512 threads (26 us for 64 rows of
// 131072); blocks of 1024 run one by one (35 us).
constexpr int kSliceThreads = 1024, kBinThreads = 512;

__device__ __forceinline__ void slice_of(const SampleArgs& a, int64_t* lo, int64_t* hi) {
  const int64_t each = ceil_div(ceil_div(a.V, a.slices), 64) * 64;
  *lo = blockIdx.x * each;
  *hi = *lo + each < a.V ? *lo + each : a.V;
}

template <typename T>
__global__ void __launch_bounds__(kSliceThreads) sample_range_kernel(SampleArgs a) {
  __shared__ double part[16];
  int64_t lo, hi;
  slice_of(a, &lo, &hi);
  const int64_t b = blockIdx.y;
  const float2 range = find_range<kSliceThreads, T>(a, b, lo, hi, part);
  if (threadIdx.x == 0) a.range[b * a.slices + blockIdx.x] = range;
}

__device__ __forceinline__ RowRule row_rule(const SampleArgs& a, int64_t b) {
  float2 r[kMostSlices];  // (all on their way together)
#pragma unroll
  for (int i = 0; i < kMostSlices; ++i) r[i] = a.range[b * a.slices + (i < a.slices ? i : 0)];
#pragma unroll
  for (int i = 1; i < kMostSlices; ++i) r[0] = make_float2(fmaxf(r[0].x, r[i].x), fminf(r[0].y, r[i].y));
  return rule_of<kWide>(a, b, r[0].x, r[0].y);
}

template <typename T>
__global__ void __launch_bounds__(kBinThreads) sample_bins_kernel(SampleArgs a) {
  __shared__ SampleShared<kWide> s;
  const int64_t b = blockIdx.y;
  const RowRule r = row_rule(a, b);
  if (r.greedy || r.top == -INFINITY) return;
  int64_t lo, hi;
  slice_of(a, &lo, &hi);
  fill_bins<kBinThreads, kWide, T>(a, b, lo, hi, r, s.cells);
  uint64_t* cells = a.cells + b * a.slices * (kWide + 1);
  for (int i = threadIdx.x; i <= kWide; i += kBinThreads) put_shared(cells + blockIdx.x * (kWide + 1) + i, s.cells[i]);
  if (!arrives_last(a.counters + 2 * b, a.slices, &s.last)) return;
  sum_bins<kBinThreads>(r, s, [&](int bin, int64_t* n, uint64_t* d) {
    *n = 0;
    *d = 0;
    uint64_t w[kMostSlices];  // (all on their way together)
#pragma unroll
    for (int i = 0; i < kMostSlices; ++i) w[i] = get_shared(cells + (i < a.slices ? i : 0) * (kWide + 1) + bin);
#pragma unroll
    for (int i = 0; i < kMostSlices; ++i) {
      if (i >= a.slices) continue;
      *n += static_cast<int64_t>(w[i] >> kDefShift);
      *d += w[i] & ((uint64_t{1} << kDefShift) - 1);
    }
  });
  for (int i = threadIdx.x; i <= kWide + 1; i += kBinThreads) {
    if (i <= kWide) a.mass[b * (kWide + 1) + i] = s.mass[i];
    a.count[b * (kWide + 2) + i] = s.count[i];
  }
  const Asked q = ask(a, b, r, s);
  if (threadIdx.x == 0) a.asked[b] = q;
}

template <typename T>
__global__ void __launch_bounds__(kSliceThreads) sample_find_kernel(SampleArgs a) {
  __shared__ uint64_t cells[kCandidates];
  __shared__ int found, first;
  const int64_t b = blockIdx.y;
  const RowRule r = row_rule(a, b);
  if (r.top == -INFINITY) return;
  int64_t lo, hi;
  slice_of(a, &lo, &hi);
  int* counter = a.counters + 2 * b + 1;
  if (r.greedy) {  // the first of the largest: the most tokens behind it
    int behind = 0;
    each_logit<kSliceThreads, T>(a, b, lo, hi, [&](float x, int64_t i) {
      if (x == r.top && static_cast<int>(a.V - i) > behind) behind = static_cast<int>(a.V - i);
    });
    if (behind) atomicMax(counter, behind);
    return;
  }
  const Asked q = a.asked[b];
  // the block's own together first, then a place for them among the row's
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  each_candidate<kSliceThreads, kWide, T>(a, b, lo, hi, r, q, [&](uint64_t cell) {
    const int at = atomicAdd(&found, 1);
    if (at < kCandidates) cells[at] = cell;
  });
  __syncthreads();
  if (threadIdx.x == 0 && found) first = atomicAdd(counter, found);
  __syncthreads();
  for (int i = threadIdx.x; i < found && first + i < kCandidates; i += kSliceThreads)
    a.found[b * kCandidates + first + i] = cells[i];
}

template <typename T>
__global__ void __launch_bounds__(kSliceThreads) sample_draw_kernel(SampleArgs a) {
  __shared__ SampleShared<kWide> s;
  const int64_t b = blockIdx.x;
  const int n = a.counters[2 * b + 1];
  const RowRule r = row_rule(a, b);
  __syncthreads();  // (all have read it)
  if (threadIdx.x == 0) a.counters[2 * b + 1] = 0;
  if (r.top == -INFINITY || r.greedy) {
    if (threadIdx.x) return;
    a.tokens[b] = r.top == -INFINITY ? -1 : static_cast<int32_t>(a.V - n);
    if (a.logs) a.logs[b] = r.top == -INFINITY ? -INFINITY : 0.0f;
    return;
  }
  draw<kSliceThreads, kWide, T>(a, b, r, a.asked[b], s, a.found + b * kCandidates, a.mass + b * (kWide + 1),
                                a.count + b * (kWide + 2), n);
}

template <typename T>
static int launch_sample(SampleArgs& a) {
  if (a.B > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "sample: too many rows");
  const dim3 rows(static_cast<unsigned>(a.B));
  if (a.V <= kShortRow) {
    KK_LAUNCH((sample_row_kernel<256, 512, T>), rows, dim3(256), 0, ctx().stream, a);
    return check_launch("sample_row_kernel");
  }
  // as many blocks a row as scratch has room for their bins, and counters
  const int64_t fixed = (kWide + 1) * 8 + (kWide + 2) * 4 + kCandidates * 8 + sizeof(Asked) + 16;
  const int64_t room = (static_cast<int64_t>(kScratchBytes) / a.B - fixed) / ((kWide + 1) * 8 + 8);
  int64_t slices = ceil_div(a.V, kSlice);
  slices = slices < room ? slices : room;
  if (slices < 2 || 2 * a.B > kRowCounters) {
    KK_LAUNCH((sample_row_kernel<1024, kWide, T>), rows, dim3(1024), 0, ctx().stream, a);
    return check_launch("sample_row_kernel");
  }
  a.slices = static_cast<int>(slices);
  char* at = static_cast<char*>(ctx().scratch);
  a.cells = reinterpret_cast<uint64_t*>(at);
  at += a.B * slices * (kWide + 1) * 8;
  a.mass = reinterpret_cast<double*>(at);
  at += a.B * (kWide + 1) * 8;
  a.found = reinterpret_cast<uint64_t*>(at);
  at += a.B * kCandidates * 8;
  a.range = reinterpret_cast<float2*>(at);
  at += a.B * slices * 8;
  a.asked = reinterpret_cast<Asked*>(at);
  at += a.B * sizeof(Asked);
  a.count = reinterpret_cast<int*>(at);
  a.counters = ctx().row_counters;
  const dim3 grid(static_cast<unsigned>(slices), static_cast<unsigned>(a.B));
  KK_LAUNCH(sample_range_kernel<T>, grid, dim3(kSliceThreads), 0, ctx().stream, a);
  KK_LAUNCH(sample_bins_kernel<T>, grid, dim3(kBinThreads), 0, ctx().stream, a);
  KK_LAUNCH(sample_find_kernel<T>, grid, dim3(kSliceThreads), 0, ctx().stream, a);
  KK_LAUNCH(sample_draw_kernel<T>, rows, dim3(kSliceThreads), 0, ctx().stream, a);
  return check_launch("sample_draw_kernel");
}

}  // namespace kk

using namespace kk;

extern "C" {

int kk_sample(const kk_tensor* tokens, const kk_tensor* logs, const kk_tensor* logits, const kk_tensor* uniforms,
              const kk_tensor* temperature, const kk_tensor* top_k, const kk_tensor* top_p, const kk_tensor* min_p) {
  const char* who = "sample";
  KK_TRY(check_tensor(logits, "logits"));
  if (!is_float(logits->dtype) || logits->rank != 2)
    return set_error(KK_E_ARG, "%s: logits must be f32 or f16 [rows, tokens]", who);
  SampleArgs a{};
  a.B = logits->shape[0];
  a.V = logits->shape[1];
  if (a.V > 1 && a.B > 0 && logits->strides[1] != 1)
    return set_error(KK_E_ARG, "%s: a row of logits must lie in one piece", who);
  KK_TRY(check_tensor(tokens, "tokens"));
  if (tokens->dtype != KK_I32 || tokens->rank != 1 || tokens->shape[0] != a.B || !is_contiguous(tokens))
    return set_error(KK_E_ARG, "%s: tokens must be int32, one a row, in one piece", who);
  if (logs) {
    KK_TRY(check_tensor(logs, "logs"));
    if (logs->dtype != KK_F32 || logs->rank != 1 || logs->shape[0] != a.B || !is_contiguous(logs))
      return set_error(KK_E_ARG, "%s: logs must be f32, one a row, in one piece", who);
  }
  KK_TRY(check_per_row(uniforms, "uniforms", a.B, false, who));
  const kk_tensor* of[3] = {temperature, top_p, min_p};
  const char* names[3] = {"temperature", "top_p", "min_p"};
  const float** to[3] = {&a.temperature, &a.top_p, &a.min_p};
  int64_t* strides[3] = {&a.t_st, &a.p_st, &a.m_st};
  for (int i = 0; i < 3; ++i) {
    if (!of[i]) continue;
    KK_TRY(check_per_row(of[i], names[i], a.B, false, who));
    *to[i] = static_cast<const float*>(of[i]->data);
    *strides[i] = row_stride(of[i]);
  }
  if (top_k) {
    KK_TRY(check_per_row(top_k, "top_k", a.B, true, who));
    a.top_k = top_k->data;
    a.k_dt = top_k->dtype;
    a.k_st = row_stride(top_k);
  }
  if (a.V < 1 || a.V > kMostTokens)
    return set_error(KK_E_UNSUPPORTED, "%s: rows of %lld tokens (1 to %d)", who, static_cast<long long>(a.V), kMostTokens);
  KK_TRY(require_ready());
  if (a.B == 0) return KK_OK;
  a.x = logits->data;
  a.xs = a.B > 1 ? logits->strides[0] : 0;
  a.u = static_cast<const float*>(uniforms->data);
  a.u_st = row_stride(uniforms);
  a.tokens = static_cast<int32_t*>(tokens->data);
  a.logs = logs ? static_cast<float*>(logs->data) : nullptr;
  return logits->dtype == KK_F16 ? launch_sample<__half>(a) : launch_sample<float>(a);
}

}  // extern "C"
