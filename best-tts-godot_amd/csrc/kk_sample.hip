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

constexpr int kBins = 2048;
constexpr double kFarthest = 64.0;  // past 2^-64 a weight counts as none (a row of 2^23 sums them to 2^-41)
constexpr int kOnes = 34;           // a weight within its bin: 2^34 - d
constexpr int kDefShift = 46;       // a bin: (tokens << 46) + sum of d, both exact up to 2^17 tokens
constexpr int kSliceMost = 1 << 17;
constexpr int kCandidates = 2048;
constexpr int kRangeThreads = 1024;

struct SampleArgs {
  const void* x;
  int x_dt;
  int64_t xs, V, B;
  const float *u, *temperature, *top_p, *min_p;
  const void* top_k;
  int k_dt;
  int64_t u_st, t_st, k_st, p_st, m_st;
  int32_t* tokens;
  float* logs;       // or NULL
  int64_t slice;     // tokens of a block, and blocks of a row
  int slices;
  float2* range;     // [B][slices] largest and smallest
  uint64_t* hist;    // [B][slices][kBins + 1]
  uint64_t* found;   // [B][kCandidates]
  int* counters;     // [B][2]: candidates, blocks that arrived; zero between launches
};

// What a row's numbers ask for.
struct RowRule {
  float top;       // its largest logit
  double c;        // log2(e) / temperature
  double inv, width;
  bool greedy;
};

__device__ __forceinline__ float logit(const SampleArgs& a, int64_t b, int64_t i) {
  const int64_t at = b * a.xs + i;
  const float v = a.x_dt == KK_F16 ? __half2float(static_cast<const __half*>(a.x)[at]) : static_cast<const float*>(a.x)[at];
  return v != v ? -INFINITY : v + 0.0f;  // (-0 is 0)
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
__device__ __forceinline__ int bin_of(const RowRule& r, double y) {
  if (!(y < kFarthest)) return kBins;
  const double b = y * r.inv;
  return b < kBins - 1 ? static_cast<int>(b) : kBins - 1;
}
// 2^34 (1 - 2^-(y - lower edge)): 1 - e^-z by its series, z <= 2^-5 ln 2, to 2^-34.
__device__ __forceinline__ uint32_t deficit(const RowRule& r, double y, int bin) {
  double z = fma(-static_cast<double>(bin), r.width, y) * 0.69314718055994530942;
  z = z > 0.0 ? z : 0.0;
  const double d = z * fma(-z, fma(-z, fma(-z, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0);
  return static_cast<uint32_t>(fma(d, static_cast<double>(int64_t{1} << kOnes), 0.5));
}
__device__ __forceinline__ double edge_weight(const RowRule& r, int bin) { return exp2(-static_cast<double>(bin) * r.width); }

__device__ __forceinline__ RowRule rule_of(const SampleArgs& a, int64_t b, float top, float least) {
  RowRule r;
  const float t = a.temperature ? a.temperature[b * a.t_st] : 1.0f;
  r.top = top;
  r.greedy = !(t > 0.0f);
  r.c = r.greedy ? 0.0 : 1.44269504088896340736 / static_cast<double>(t);
  const double all = far_of(r, least);
  const double span = all < kFarthest ? all : kFarthest;
  r.inv = span > 0.0 ? kBins / span : 0.0;
  r.width = span / kBins;
  if (!(r.inv < 1e300)) r.inv = r.width = 0.0;
  return r;
}

template <int THREADS>
struct SampleShared {
  uint64_t cells[kCandidates + 1];  // bins' counts and sums; then the candidates
  uint64_t sums[kCandidates];       // running sums of the candidates' 2^34 - d
  double mass[kBins + 1];           // before a bin
  int count[kBins + 2];
  uint16_t bin[kCandidates];
  uint64_t part[THREADS / 64];
  double dpart[THREADS / 64];
  int range[7];
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

// The largest and smallest logit of tokens [lo, hi) that are not -inf.
template <int THREADS>
__device__ __forceinline__ float2 find_range(const SampleArgs& a, int64_t b, int64_t lo, int64_t hi, double* part) {
  float top = -INFINITY, least = INFINITY;
  for (int64_t i = lo + threadIdx.x; i < hi; i += THREADS) {
    const float x = logit(a, b, i);
    top = fmaxf(top, x);
    least = fminf(least, x == -INFINITY ? INFINITY : x);
  }
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

template <int THREADS>
__device__ __forceinline__ void fill_bins(const SampleArgs& a, int64_t b, int64_t lo, int64_t hi, const RowRule& r,
                                          uint64_t* cells) {
  for (int i = threadIdx.x; i <= kBins; i += THREADS) cells[i] = 0;
  __syncthreads();
  for (int64_t i = lo + threadIdx.x; i < hi; i += THREADS) {
    const float x = logit(a, b, i);
    if (x == -INFINITY) continue;
    const double y = far_of(r, x);
    const int bin = bin_of(r, y);
    const uint64_t one = (uint64_t{1} << kDefShift) + (bin < kBins ? deficit(r, y, bin) : 0u);
    atomicAdd(reinterpret_cast<unsigned long long*>(&cells[bin]), static_cast<unsigned long long>(one));
  }
  __syncthreads();
}

// From the bins' counts and sums of d, what comes before each bin: tokens, and
// weight.  get(bin, &n, &d).
template <int THREADS, class Get>
__device__ __forceinline__ void sum_bins(const RowRule& r, SampleShared<THREADS>& s, Get get) {
  constexpr int EACH = kBins / THREADS;
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
    int64_t n_far;
    uint64_t d;
    get(kBins, &n_far, &d);
    s.count[kBins] = static_cast<int>(tokens);
    s.mass[kBins] = weight;
    s.count[kBins + 1] = static_cast<int>(tokens + n_far);
  }
  __syncthreads();
}

// The first bin that fulfils `reaches` of what comes before its end; the last one
// where none does.
template <int THREADS, class Reaches>
__device__ __forceinline__ int first_bin(SampleShared<THREADS>& s, int slot, Reaches reaches) {
  if (threadIdx.x == 0) s.range[slot] = kBins - 1;
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += THREADS)
    if (reaches(b + 1) && (b == 0 || !reaches(b))) atomicMin(&s.range[slot], b);
  __syncthreads();
  return s.range[slot];
}

// The bins that the limits and the drawn number can fall into, as far as the bins'
// sums say, and what is known beforehand.
struct Asked {
  int64_t k;       // tokens kept by top-k; live where all are
  double p, m, u;  // p >= 1, m <= 0: no limit
  double far;      // largest y kept by min-p
  int bin[7];      // of k; first and last of p; of m; first and last of u (-1: none)
};

template <int THREADS>
__device__ __forceinline__ Asked ask(const SampleArgs& a, int64_t b, const RowRule& r, SampleShared<THREADS>& s) {
  Asked q;
  const int64_t live = s.count[kBins + 1];
  int64_t k = a.top_k ? load_index(a.top_k, a.k_dt, b * a.k_st) : 0;
  q.k = k > 0 && k < live ? k : live;
  const float p = a.top_p ? a.top_p[b * a.p_st] : 1.0f, m = a.min_p ? a.min_p[b * a.m_st] : 0.0f, u = a.u[b * a.u_st];
  q.p = p < 1.0f ? (p > 0.0f ? p : 0.0) : 1.0;
  q.m = m > 0.0f ? (m < 1.0f ? m : 1.0) : 0.0;
  q.u = u > 0.0f ? (u < 0x1.fffffep-1f ? u : 0x1.fffffep-1f) : 0.0;
  constexpr double kLess = 1.0 - 1e-12, kMore = 1.0 + 1e-12;
  double lo = s.mass[kBins], hi = lo;
  for (int i = 0; i < 7; ++i) q.bin[i] = -1;
  // (k within the far tokens, which weigh nothing, cuts nothing off)
  if (q.k < live && q.k <= s.count[kBins]) {
    const int64_t want = q.k;
    q.bin[0] = first_bin(s, 0, [&](int i) { return s.count[i] >= want; });
    lo = s.mass[q.bin[0]];
    hi = s.mass[q.bin[0] + 1];
  }
  if (q.p < 1.0) {
    const double t0 = q.p * lo * kLess, t1 = q.p * hi * kMore;
    q.bin[1] = first_bin(s, 1, [&](int i) { return s.mass[i] >= t0; });
    q.bin[2] = first_bin(s, 2, [&](int i) { return s.mass[i] >= t1; });
    const double end = s.mass[q.bin[2] + 1];
    lo = s.mass[q.bin[1]];
    hi = end < hi ? end : hi;
  }
  q.far = INFINITY;
  if (q.m > 0.0) {
    q.far = -log2(q.m);
    const int bin = bin_of(r, q.far);
    if (bin < kBins) {
      q.bin[3] = bin;
      lo = s.mass[bin] < lo ? s.mass[bin] : lo;
      hi = s.mass[bin + 1] < hi ? s.mass[bin + 1] : hi;
    }
  }
  const double t0 = q.u * lo * kLess, t1 = q.u * hi * kMore;
  q.bin[4] = first_bin(s, 4, [&](int i) { return s.mass[i] > t0; });
  q.bin[5] = first_bin(s, 5, [&](int i) { return s.mass[i] > t1; });
  return q;
}

__device__ __forceinline__ bool wanted(const Asked& q, int bin) {
  return bin == q.bin[0] || bin == q.bin[3] || (bin >= q.bin[1] && bin <= q.bin[2]) || (bin >= q.bin[4] && bin <= q.bin[5]);
}

__device__ __forceinline__ void put_token(const SampleArgs& a, int64_t b, int64_t token, double y, double kept) {
  a.tokens[b] = static_cast<int32_t>(token);
  if (a.logs) a.logs[b] = static_cast<float>(-y * 0.69314718055994530942 - log(kept));
}

// The token from the `n` candidates in s.cells: all tokens of the wanted bins.
template <int THREADS>
__device__ __forceinline__ void draw_from(const SampleArgs& a, int64_t b, const RowRule& r, const Asked& q,
                                          SampleShared<THREADS>& s, int n) {
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
      __syncthreads();
    }
  // running sums of 2^34 - d over all candidates
  constexpr int EACH = kCandidates / THREADS;
  uint64_t ones[EACH], mine = 0, all;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = threadIdx.x * EACH + i;
    ones[i] = 0;
    if (at < n) {
      const double y = far_of(r, of_key(static_cast<uint32_t>(s.cells[at] >> 32)));
      const int bin = bin_of(r, y);
      s.bin[at] = static_cast<uint16_t>(bin);
      ones[i] = (uint64_t{1} << kOnes) - deficit(r, y, bin);
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
    *rank = s.count[bin] + (at - lo) + 1;
    const uint64_t in_bin = s.sums[at] - (lo ? s.sums[lo - 1] : 0);
    return s.mass[bin] + edge_weight(r, bin) * (static_cast<double>(in_bin) * (1.0 / (int64_t{1} << kOnes)));
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
  double kept = q.bin[0] >= 0 ? s.value : s.mass[kBins];
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
    double end = s.mass[q.bin[3]];
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

// The same where the wanted bins hold more tokens than there is room for (many
// equal logits): for each target in turn its bin, then the keys of the bin's
// tokens digit by digit, each over the whole row, then which of the equal ones.
template <int THREADS>
__device__ __forceinline__ void draw_slowly(const SampleArgs& a, int64_t b, const RowRule& r, const Asked& q,
                                            SampleShared<THREADS>& s) {
  constexpr double kUnit = 1.0 / (int64_t{1} << kOnes);
  uint64_t* const n = s.cells;  // of a digit: tokens, then their 2^34 - d
  double kept = s.mass[kBins];
#pragma unroll 1
  for (int target = 0; target < 3; ++target) {  // top-k, top-p, the drawn token
    if (target == 0 && q.bin[0] < 0) continue;
    if (target == 1 && !(q.p < 1.0)) continue;
    if (target == 2 && q.bin[3] >= 0) {  // min-p
      uint64_t ones = 0, all;
      for (int64_t i = threadIdx.x; i < a.V; i += THREADS) {
        const float x = logit(a, b, i);
        if (x == -INFINITY) continue;
        const double y = far_of(r, x);
        if (bin_of(r, y) == q.bin[3] && !(y > q.far)) ones += (uint64_t{1} << kOnes) - deficit(r, y, q.bin[3]);
      }
      block_scan<THREADS, uint64_t>(ones, s.part, &all);
      const double end = s.mass[q.bin[3]] + edge_weight(r, q.bin[3]) * (static_cast<double>(all) * kUnit);
      kept = end < kept ? end : kept;
    }
    const double want = target == 1 ? q.p * kept : q.u * kept;
    auto reaches = [&](int64_t tokens, double w) {
      return target == 0 ? tokens >= q.k : target == 1 ? w >= want : w > want;
    };
    const int bin = first_bin(s, 6, [&](int i) { return reaches(s.count[i], s.mass[i]); });
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
        const float x = logit(a, b, i);
        if (x == -INFINITY) continue;
        const uint32_t k = key_of(x);
        if (shift < 24 && (k ^ key) >> (shift + 8)) continue;
        const double y = far_of(r, x);
        if (bin_of(r, y) != bin) continue;
        const int digit = k >> shift & 255u;
        atomicAdd(reinterpret_cast<unsigned long long*>(&n[digit]), 1ull);
        atomicAdd(reinterpret_cast<unsigned long long*>(&n[256 + digit]),
                  static_cast<unsigned long long>((uint64_t{1} << kOnes) - deficit(r, y, bin)));
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
    const uint64_t each = (uint64_t{1} << kOnes) - deficit(r, y, bin);
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
    for (int64_t i = i0; i < i1; ++i) mine += logit(a, b, i) == x;
    const int64_t to = block_scan<THREADS, int64_t>(mine, reinterpret_cast<int64_t*>(s.part), &all);
    if (lo <= to - mine || lo > to) continue;
    lo -= to - mine;
    for (int64_t i = i0; i < i1; ++i)
      if (logit(a, b, i) == x && --lo == 0) put_token(a, b, i, y, kept);
  }
}

// Rows of which nothing is left, and rows whose largest logit is taken; false
// where there is more to do.
template <int THREADS>
__device__ __forceinline__ bool draw_simply(const SampleArgs& a, int64_t b, const RowRule& r, SampleShared<THREADS>& s) {
  if (r.top == -INFINITY) {
    if (threadIdx.x == 0) {
      a.tokens[b] = -1;
      if (a.logs) a.logs[b] = -INFINITY;
    }
    return true;
  }
  if (!r.greedy) return false;
  if (threadIdx.x == 0) s.at = 0x7fffffff;
  __syncthreads();
  int at = 0x7fffffff;
  for (int64_t i = threadIdx.x; i < a.V; i += THREADS)
    if (logit(a, b, i) == r.top) {
      at = static_cast<int>(i);
      break;
    }
  if (at != 0x7fffffff) atomicMin(&s.at, at);
  __syncthreads();
  if (threadIdx.x == 0) {
    a.tokens[b] = s.at;
    if (a.logs) a.logs[b] = 0.0f;
  }
  return true;
}

// A block a row: short rows, in one launch.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) sample_row_kernel(SampleArgs a) {
  __shared__ SampleShared<THREADS> s;
  const int64_t b = blockIdx.x;
  const float2 range = find_range<THREADS>(a, b, 0, a.V, s.dpart);
  const RowRule r = rule_of(a, b, range.x, range.y);
  if (draw_simply(a, b, r, s)) return;
  fill_bins<THREADS>(a, b, 0, a.V, r, s.cells);
  sum_bins<THREADS>(r, s, [&](int bin, int64_t* n, uint64_t* d) {
    const uint64_t w = s.cells[bin];
    *n = static_cast<int64_t>(w >> kDefShift);
    *d = w & ((uint64_t{1} << kDefShift) - 1);
  });
  const Asked q = ask(a, b, r, s);
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.V; i += THREADS) {
    const float x = logit(a, b, i);
    if (x == -INFINITY || !wanted(q, bin_of(r, far_of(r, x)))) continue;
    const int at = atomicAdd(&s.n, 1);
    if (at < kCandidates) s.cells[at] = uint64_t{key_of(x)} << 32 | static_cast<uint32_t>(i);
  }
  __syncthreads();
  const int n = s.n;
  if (n <= kCandidates)
    draw_from(a, b, r, q, s, n);
  else
    draw_slowly(a, b, r, q, s);
}

static int launch_rows(const SampleArgs& a) {
  if (a.B > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "sample: too many rows");
  const dim3 grid(static_cast<unsigned>(a.B));
  if (a.V <= 4096)
    KK_LAUNCH(sample_row_kernel<256>, grid, dim3(256), 0, ctx().stream, a);
  else
    KK_LAUNCH(sample_row_kernel<1024>, grid, dim3(1024), 0, ctx().stream, a);
  return check_launch("sample_row_kernel");
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
  if (a.V < 1 || a.V > kSliceMost)
    return set_error(KK_E_UNSUPPORTED, "%s: rows of %lld tokens (1 to %d)", who, static_cast<long long>(a.V), kSliceMost);
  KK_TRY(require_ready());
  if (a.B == 0) return KK_OK;
  a.x = logits->data;
  a.x_dt = logits->dtype;
  a.xs = a.B > 1 ? logits->strides[0] : 0;
  a.u = static_cast<const float*>(uniforms->data);
  a.u_st = row_stride(uniforms);
  a.tokens = static_cast<int32_t*>(tokens->data);
  a.logs = logs ? static_cast<float*>(logs->data) : nullptr;
  return launch_rows(a);
}

}  // extern "C"
