// Pages of a cache given to sequences and taken back, and the slots of their
// tokens: the whole numbers that a server's step begins with.  Bound by their
// launch (single tokens) or by the slots' bytes (prompts).
#include "kk_decode.h"

namespace kk {

struct PlanArgs {
  int32_t* table;
  int64_t table_stride, columns;
  int64_t* slots;
  int64_t slots_st;
  int32_t* positions;
  int64_t positions_st;
  int32_t *lengths, *granted;   // [B]
  const void *starts, *counts;  // counts NULL: T each
  int starts_dt, counts_dt;
  int64_t starts_st, counts_st;
  const int32_t* free;
  int64_t F;
  const int32_t* used;
  int32_t* used_out;  // may be `used`
  int64_t B;
  int T, shift;       // pages of 2^shift tokens
  int rows;           // sequences of a block
  int chunk;          // tokens of a sequence and block
  int* arrived;       // of the grid's blocks; zero between launches
};

constexpr int kPlanThreads = 256;

// What sequence b asks for: `need` pages behind the `have` that it has.  None
// where its start or its end is not within the table.
struct Wish {
  int64_t start, have, need;
  int count;
};
__device__ __forceinline__ Wish wish_of(const PlanArgs& a, int64_t b) {
  Wish w{0, 0, 0, 0};
  if (b >= a.B) return w;
  const int64_t capacity = a.columns << a.shift, start = load_index(a.starts, a.starts_dt, b * a.starts_st);
  if (start < 0 || start > capacity) return w;
  int64_t count = a.counts ? load_index(a.counts, a.counts_dt, b * a.counts_st) : a.T;
  count = count < 0 ? 0 : count < a.T ? count : a.T;
  if (start + count > capacity) count = 0;
  const int64_t past = (int64_t{1} << a.shift) - 1;
  w.start = start;
  w.have = (start + past) >> a.shift;
  w.need = ((start + count + past) >> a.shift) - w.have;
  w.count = static_cast<int>(count);
  return w;
}

// Sum over the block's threads up to and including this one; *all of all of them.
__device__ __forceinline__ int64_t scan_block(int64_t v, int64_t* all, int64_t* part) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  int64_t before = 0, sum = 0;
  for (int i = 0; i < waves; ++i) {
    if (i == wave) before = sum;
    sum += part[i];
  }
  *all = sum;
  return v + before;
}

// A block has `rows` sequences (one, cut into chunks of its tokens, where T is
// long).  Each block forms by itself the sum of what the sequences before its own
// ask for: B / 256 loads a thread, against a launch of its own for them.
__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(PlanArgs a) {
  __shared__ int64_t part[kPlanThreads / 64], s_start[kPlanThreads], s_first[kPlanThreads];
  __shared__ int s_have[kPlanThreads], s_granted[kPlanThreads], s_need[kPlanThreads], s_last;
  const int tid = threadIdx.x;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * a.rows;
  const int here = static_cast<int>(a.B - row0 < a.rows ? a.B - row0 : a.rows);
  int64_t used = *a.used, all;
  used = used < 0 ? 0 : used < a.F ? used : a.F;
  const int64_t left = a.F - used;
  int64_t before = 0;
  for (int64_t b = tid; b < row0; b += kPlanThreads) before += wish_of(a, b).need;
  if (row0) {
    scan_block(before, &all, part);
    before = all;
  }
  const Wish w = wish_of(a, tid < here ? row0 + tid : a.B);
  const int64_t upto = before + scan_block(w.need, &all, part);
  const bool served = w.need == 0 || upto <= left;
  if (tid < here) {
    s_start[tid] = w.start;
    s_have[tid] = static_cast<int>(w.have);
    s_need[tid] = served ? static_cast<int>(w.need) : 0;
    s_granted[tid] = served ? w.count : 0;
    s_first[tid] = used + upto - w.need;
    if (blockIdx.x == 0) {
      a.lengths[row0 + tid] = static_cast<int32_t>(w.start + (served ? w.count : 0));
      a.granted[row0 + tid] = served ? w.count : 0;
    }
  }
  __syncthreads();
  // the table's new entries: of a sequence's first chunk, a sequence a wave
  if (blockIdx.x == 0)
    for (int r = tid / 64; r < here; r += kPlanThreads / 64)
      for (int i = tid % 64; i < s_need[r]; i += 64)
        a.table[(row0 + r) * a.table_stride + s_have[r] + i] = a.free[s_first[r] + i];
  const int t0 = static_cast<int>(blockIdx.x) * a.chunk, tokens = a.T - t0 < a.chunk ? a.T - t0 : a.chunk;
  for (int i = tid; i < here * tokens; i += kPlanThreads) {
    const int r = a.rows == 1 ? 0 : i / tokens, t = t0 + (i - r * tokens);
    int64_t slot = -1;
    int32_t place = -1;
    if (t < s_granted[r]) {
      const int64_t p = s_start[r] + t, column = p >> a.shift;
      const int page = column < s_have[r] ? a.table[(row0 + r) * a.table_stride + column]
                                          : a.free[s_first[r] + (column - s_have[r])];
      place = static_cast<int32_t>(p);
      if (page >= 0) slot = (int64_t{page} << a.shift) + (p & ((int64_t{1} << a.shift) - 1));
    }
    a.slots[(row0 + r) * a.slots_st + t] = slot;
    a.positions[(row0 + r) * a.positions_st + t] = place;
  }
  // how many pages are given out in all: by the block that comes last, when all
  // have read how many were
  int64_t taken = served && w.need ? upto : 0;
  if (gridDim.x * gridDim.y > 1) {
    __syncthreads();
    if (tid == 0)
      s_last = __hip_atomic_fetch_add(a.arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               static_cast<int>(gridDim.x * gridDim.y) - 1;
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) __hip_atomic_store(a.arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    taken = before = 0;
    for (int64_t b0 = 0; b0 < a.B; b0 += kPlanThreads) {
      const int64_t need = wish_of(a, b0 + tid).need, to = before + scan_block(need, &all, part);
      if (need && to <= left) taken = to;
      before += all;
    }
  }
  for (int off = 32; off > 0; off >>= 1) {
    const int64_t o = __shfl_xor(taken, off, 64);
    taken = o > taken ? o : taken;
  }
  __syncthreads();
  if (tid % 64 == 0) part[tid / 64] = taken;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kPlanThreads / 64; ++i) taken = part[i] > taken ? part[i] : taken;
    *a.used_out = static_cast<int32_t>(used + taken);
  }
}

struct ReleaseArgs {
  int32_t* table;
  int64_t table_stride, columns;
  const void* lengths;
  int lengths_dt;
  int64_t lengths_st;
  const uint8_t* ended;
  int64_t ended_st;
  int32_t* free;
  int64_t F;
  int32_t* used;
  int64_t B;
  int shift;
};

constexpr int kReleaseThreads = 1024;

// One block: first how many pages come back, then they, in the order of
// sequences and columns, in front of those that are free.  Of 1024 sequences at a
// time it lists the ended ones, and takes the columns of each 1024 at a time: two passes and
// a scan for each ended sequence, 2 us (one of 32: 6.7 us; 64 of 256 pages: 144).
__global__ void __launch_bounds__(kReleaseThreads) release_pages_kernel(ReleaseArgs a) {
  __shared__ int64_t part[kReleaseThreads / 64];
  __shared__ int s_row[kReleaseThreads], s_pages[kReleaseThreads];
  const int tid = threadIdx.x;
  const int64_t given = *a.used < 0 ? 0 : *a.used < a.F ? *a.used : a.F;
  int64_t all = 0, back = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t mine = 0, at = given - back;  // (pass 1)
    for (int64_t b0 = 0; b0 < a.B; b0 += kReleaseThreads) {
      const int64_t b = b0 + tid;
      int64_t n = 0;
      if (b < a.B && a.ended[b * a.ended_st]) {
        n = load_index(a.lengths, a.lengths_dt, b * a.lengths_st);
        n = n < 0 ? 0 : n;
        n = n > a.columns << a.shift ? a.columns : (n + (int64_t{1} << a.shift) - 1) >> a.shift;
      }
      const int place = static_cast<int>(scan_block(n > 0, &all, part)) - 1, listed = static_cast<int>(all);
      if (n > 0) {
        s_row[place] = tid;
        s_pages[place] = static_cast<int>(n);
      }
      __syncthreads();
      for (int e = 0; e < listed; ++e) {
        int32_t* row = a.table + (b0 + s_row[e]) * a.table_stride;
        for (int c0 = 0; c0 < s_pages[e]; c0 += kReleaseThreads) {
          const int c = c0 + tid;
          const int32_t page = c < s_pages[e] ? row[c] : -1;
          if (pass == 0) {
            mine += page >= 0;
            continue;
          }
          const int64_t to = at + scan_block(page >= 0, &all, part) - 1;
          if (page >= 0 && to < given) a.free[to] = page;
          if (c < s_pages[e]) row[c] = -1;
          at += all;
        }
      }
    }
    if (pass == 0) {
      scan_block(mine, &all, part);
      back = all < given ? all : given;
    }
  }
  if (tid == 0) *a.used = static_cast<int32_t>(given - back);
}

static int check_ints(const kk_tensor* t, const char* name, int dtype, int64_t n, const char* who) {
  KK_TRY(check_tensor(t, name));
  if (t->dtype != dtype || t->rank != 1 || (n >= 0 && t->shape[0] != n) || !is_contiguous(t))
    return set_error(KK_E_ARG, "%s: %s must be int32 of one axis in one piece%s", who, name,
                     n == 1 ? ", one value" : n >= 0 ? ", a value a sequence" : "");
  return KK_OK;
}

// Whether a tensor in one piece and one of one axis share memory.
static bool shared(const kk_tensor* piece, const kk_tensor* axis) {
  if (numel(piece) == 0 || numel(axis) == 0) return false;
  const int64_t size = dtype_size(axis->dtype), n = axis->shape[0];
  int64_t step = n > 1 ? axis->strides[0] * size : 0;
  int64_t first = reinterpret_cast<int64_t>(axis->data);
  const int64_t lo = reinterpret_cast<int64_t>(piece->data), hi = lo + numel(piece) * dtype_size(piece->dtype);
  if (step < 0) {  // from its other end
    first += (n - 1) * step;
    step = -step;
  }
  // its first value that ends behind the piece's start
  const int64_t i = first + size > lo ? 0 : step ? (lo - size - first) / step + 1 : n;
  return i < n && first + i * step < hi;
}

static int check_table(const kk_tensor* table, int64_t block, int64_t* stride, int* shift, const char* who) {
  KK_TRY(check_tensor(table, "table"));
  if (table->dtype != KK_I32 || table->rank != 2)
    return set_error(KK_E_ARG, "%s: table must be int32 [sequences, pages]", who);
  KK_TRY(check_writable(table, "table", who));
  if (table->shape[1] > 1 && table->shape[0] > 0 && table->strides[1] != 1)
    return set_error(KK_E_ARG, "%s: a row of table must lie in one piece", who);
  if (block != 16 && block != 32 && block != 64 && block != 128 && block != 256)
    return set_error(KK_E_UNSUPPORTED, "%s: pages of %lld tokens (16, 32, 64, 128 or 256)", who,
                     static_cast<long long>(block));
  if (table->shape[1] > 0x7fffffff / block)
    return set_error(KK_E_UNSUPPORTED, "%s: a table of %lld columns", who, static_cast<long long>(table->shape[1]));
  *stride = table->shape[0] > 1 ? table->strides[0] : 0;
  *shift = __builtin_ctzll(static_cast<unsigned long long>(block));
  return KK_OK;
}

}  // namespace kk

using namespace kk;

extern "C" {

int kk_plan_pages(const kk_tensor* table, const kk_tensor* slots, const kk_tensor* positions,
                  const kk_tensor* lengths, const kk_tensor* granted, const kk_tensor* used_out,
                  const kk_tensor* starts, const kk_tensor* counts, const kk_tensor* free, const kk_tensor* used,
                  int64_t block) {
  const char* who = "plan_pages";
  PlanArgs a{};
  KK_TRY(check_table(table, block, &a.table_stride, &a.shift, who));
  a.B = table->shape[0];
  const kk_tensor* outs[2] = {slots, positions};
  const char* names[2] = {"slots", "positions"};
  for (int i = 0; i < 2; ++i) {
    KK_TRY(check_tensor(outs[i], names[i]));
    if (outs[i]->dtype != (i ? KK_I32 : KK_I64) || outs[i]->rank != 2 || outs[i]->shape[0] != a.B ||
        outs[i]->shape[1] != slots->shape[1] ||
        (numel(outs[i]) > 0 && outs[i]->shape[1] > 1 && outs[i]->strides[1] != 1))
      return set_error(KK_E_ARG, "%s: %s must be %s [sequences, tokens], rows in one piece", who, names[i],
                       i ? "int32" : "int64");
    KK_TRY(check_writable(outs[i], names[i], who));
  }
  KK_TRY(check_ints(lengths, "lengths", KK_I32, a.B, who));
  KK_TRY(check_ints(granted, "granted", KK_I32, a.B, who));
  KK_TRY(check_per_row(starts, "starts", a.B, true, who));
  if (counts) KK_TRY(check_per_row(counts, "counts", a.B, true, who));
  KK_TRY(check_ints(free, "free", KK_I32, -1, who));
  KK_TRY(check_ints(used, "used", KK_I32, 1, who));
  KK_TRY(check_ints(used_out, "used_out", KK_I32, 1, who));
  // (a block reads the starts and counts of sequences that another may have answered already)
  const kk_tensor* read[4] = {starts, counts, free, used};
  for (const kk_tensor* t : read)
    if (t && (shared(lengths, t) || shared(granted, t)))
      return set_error(KK_E_ARG, "%s: lengths and granted must not be starts or counts, nor lie in them, free or used", who);
  if (shared(lengths, granted)) return set_error(KK_E_ARG, "%s: lengths and granted must not share memory", who);
  if (slots->shape[1] > (1 << 30) || free->shape[0] > 0x7fffffff || a.B > (1 << 30))
    return set_error(KK_E_UNSUPPORTED, "%s: too many tokens, sequences or pages", who);
  KK_TRY(require_ready());
  a.table = static_cast<int32_t*>(table->data);
  a.columns = table->shape[1];
  a.slots = static_cast<int64_t*>(slots->data);
  a.slots_st = slots->strides[0];
  a.positions = static_cast<int32_t*>(positions->data);
  a.positions_st = positions->strides[0];
  a.lengths = static_cast<int32_t*>(lengths->data);
  a.granted = static_cast<int32_t*>(granted->data);
  a.starts = starts->data;
  a.starts_dt = starts->dtype;
  a.starts_st = row_stride(starts);
  if (counts) {
    a.counts = counts->data;
    a.counts_dt = counts->dtype;
    a.counts_st = row_stride(counts);
  }
  a.free = static_cast<const int32_t*>(free->data);
  a.F = free->shape[0];
  a.used = static_cast<const int32_t*>(used->data);
  a.used_out = static_cast<int32_t*>(used_out->data);
  a.T = static_cast<int>(slots->shape[1]);
  a.arrived = ctx().row_counters;
  // 2048 tokens a block: whole sequences, 256 at the most, or a part of one
  constexpr int kTokens = 2048;
  const int64_t fit = a.T ? kTokens / a.T : kPlanThreads;
  a.rows = static_cast<int>(fit < 1 ? 1 : fit < kPlanThreads ? fit : kPlanThreads);
  a.chunk = a.rows > 1 || a.T < 1 ? (a.T < 1 ? 1 : a.T) : kTokens;
  const int64_t x = a.T ? ceil_div(a.T, a.chunk) : 1, y = a.B ? ceil_div(a.B, a.rows) : 1;
  if (y > 65535 || x * y > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many sequences", who);
  KK_LAUNCH(plan_pages_kernel, dim3(static_cast<unsigned>(x), static_cast<unsigned>(y)), dim3(kPlanThreads), 0,
            ctx().stream, a);
  return check_launch("plan_pages_kernel");
}

int kk_release_pages(const kk_tensor* table, const kk_tensor* lengths, const kk_tensor* ended, const kk_tensor* free,
                     const kk_tensor* used, int64_t block) {
  const char* who = "release_pages";
  ReleaseArgs a{};
  KK_TRY(check_table(table, block, &a.table_stride, &a.shift, who));
  a.B = table->shape[0];
  KK_TRY(check_per_row(lengths, "lengths", a.B, true, who));
  KK_TRY(check_tensor(ended, "ended"));
  if ((ended->dtype != KK_BOOL && ended->dtype != KK_U8) || ended->rank != 1 || ended->shape[0] != a.B)
    return set_error(KK_E_ARG, "%s: ended must be bool, a value a sequence", who);
  KK_TRY(check_ints(free, "free", KK_I32, -1, who));
  KK_TRY(check_ints(used, "used", KK_I32, 1, who));
  if (free->shape[0] > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many pages", who);
  KK_TRY(require_ready());
  if (a.B == 0) return KK_OK;
  a.table = static_cast<int32_t*>(table->data);
  a.columns = table->shape[1];
  a.lengths = lengths->data;
  a.lengths_dt = lengths->dtype;
  a.lengths_st = row_stride(lengths);
  a.ended = static_cast<const uint8_t*>(ended->data);
  a.ended_st = ended->strides[0];
  a.free = static_cast<int32_t*>(free->data);
  a.F = free->shape[0];
  a.used = static_cast<int32_t*>(used->data);
  KK_LAUNCH(release_pages_kernel, dim3(1), dim3(kReleaseThreads), 0, ctx().stream, a);
  return check_launch("release_pages_kernel");
}

}  // extern "C"
