// Attention of a token decoder: over a paged cache of 8-bit codes, and over
// an encoder's states.
#include "kk_attention4.h"

namespace kk {

constexpr int kRowWaves = 4;

template <typename T, class Rows>
__global__ void __launch_bounds__(kRowWaves * 64) attention_row_kernel(QueryArgs a, Rows rows, int64_t queries) {
  __shared__ float qv[kRowWaves][kMaxHead];
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kRowWaves + threadIdx.x / 64;
  if (at >= queries) return;  // (no barrier below)
  one_query<T>(a, rows, at / a.heads / a.T, at / a.heads % a.T, static_cast<int>(at % a.heads), qv[threadIdx.x / 64]);
}

template <typename T, class Rows>
static int launch_rows(const QueryArgs& a, const Rows& rows) {
  const int64_t queries = a.B * a.T * a.heads, blocks = ceil_div(queries, kRowWaves);
  if (blocks > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "attention: too many queries");
  KK_LAUNCH((attention_row_kernel<T, Rows>), dim3(static_cast<unsigned>(blocks)), dim3(kRowWaves * 64), 0,
            ctx().stream, a, rows, queries);
  return check_launch("attention_row_kernel");
}

static int check_queries(const kk_tensor* out, const kk_tensor* q, int64_t key_heads, int64_t D, float scale,
                         QueryArgs* a, const char* who) {
  KK_TRY(check_heads(q, "q", who));
  KK_TRY(check_heads(out, "out", who));
  KK_TRY(check_writable(out, "out", who));
  if (out->dtype != q->dtype) return set_error(KK_E_ARG, "%s: out must have q's dtype", who);
  for (int i = 0; i < 4; ++i)
    if (out->shape[i] != q->shape[i]) return set_error(KK_E_ARG, "%s: out must have q's shape", who);
  if (q->shape[3] != D)
    return set_error(KK_E_ARG, "%s: queries of %lld values over keys of %lld", who,
                     static_cast<long long>(q->shape[3]), static_cast<long long>(D));
  if (key_heads < 1 || q->shape[2] % key_heads)
    return set_error(KK_E_ARG, "%s: %lld query heads are not a multiple of %lld key heads", who,
                     static_cast<long long>(q->shape[2]), static_cast<long long>(key_heads));
  if (q->shape[1] > 0x7fffffff || q->shape[2] > 65535)
    return set_error(KK_E_UNSUPPORTED, "%s: too many queries", who);
  if (!(scale == scale) || scale == INFINITY || scale == -INFINITY)
    return set_error(KK_E_ARG, "%s: scale must be finite", who);
  a->q = q->data;
  a->y = out->data;
  for (int i = 0; i < 3; ++i) {
    a->qs[i] = q->strides[i];
    a->ys[i] = out->strides[i];
  }
  a->B = q->shape[0];
  a->T = static_cast<int>(q->shape[1]);
  a->heads = static_cast<int>(q->shape[2]);
  a->group = static_cast<int>(q->shape[2] / key_heads);
  a->D = static_cast<int>(D);
  a->scale = scale * 0x1.715476p+0f;
  return KK_OK;
}

// What an attention over a paged cache takes of its table, lengths and counts.
static int check_places(const kk_tensor* table, const kk_tensor* lengths, const kk_tensor* counts, int64_t window,
                        const CacheShape& c, int64_t B, PagedArgs* p, const char* who) {
  if (table->shape[0] != B) return set_error(KK_E_ARG, "%s: table must have a row a sequence", who);
  KK_TRY(check_per_row(lengths, "lengths", B, true, who));
  if (counts) KK_TRY(check_per_row(counts, "counts", B, true, who));
  if (window < 0) return set_error(KK_E_ARG, "%s: window must not be negative", who);
  p->table = static_cast<const int32_t*>(table->data);
  p->table_stride = c.table_stride;
  p->pages = c.pages;
  p->columns = c.columns;
  p->lengths = lengths->data;
  p->lengths_dt = lengths->dtype;
  p->lengths_st = row_stride(lengths);
  if (counts) {
    p->counts = counts->data;
    p->counts_dt = counts->dtype;
    p->counts_st = row_stride(counts);
  }
  p->window = window;
  p->heads = static_cast<int>(c.heads);
  p->block = static_cast<int>(c.block);
  return KK_OK;
}

}  // namespace kk

using namespace kk;

extern "C" {

int kk_cache_attention(const kk_tensor* out, const kk_tensor* q, const kk_tensor* k_codes,
                       const kk_tensor* k_scales, const kk_tensor* v_codes, const kk_tensor* v_scales,
                       const kk_tensor* table, const kk_tensor* lengths, const kk_tensor* counts, float scale,
                       int64_t window) {
  const char* who = "cache_attention";
  CacheShape c;
  KK_TRY(check_cache(k_codes, k_scales, v_codes, v_scales, table, &c, who));
  QueryArgs a{};
  KK_TRY(check_queries(out, q, c.heads, c.D, scale, &a, who));
  PagedArgs p{};
  KK_TRY(check_places(table, lengths, counts, window, c, a.B, &p, who));
  p.k = static_cast<const int8_t*>(k_codes->data);
  p.v = static_cast<const int8_t*>(v_codes->data);
  p.k_scale = static_cast<const float*>(k_scales->data);
  p.v_scale = static_cast<const float*>(v_scales->data);
  KK_TRY(require_ready());
  if (a.B * a.T * a.heads == 0) return KK_OK;
  int status = KK_OK;
  if (few_paged_try(a, p, q->dtype, &status) || tiles_paged_try(a, p, q->dtype, &status)) return status;
  const PagedRows rows{p, a.T, a.D};
  return q->dtype == KK_F16 ? launch_rows<__half>(a, rows) : launch_rows<float>(a, rows);
}

int kk_cache4_attention(const kk_tensor* out, const kk_tensor* q, const kk_tensor* k_codes,
                        const kk_tensor* k_scales, const kk_tensor* v_codes, const kk_tensor* v_scales,
                        const kk_tensor* table, const kk_tensor* lengths, const kk_tensor* counts, float scale,
                        int64_t window) {
  const char* who = "cache4_attention";
  CacheShape c;
  KK_TRY(check_codes4(k_codes, k_scales, v_codes, v_scales, &c, who));
  KK_TRY(check_cache_table(table, &c, who));
  QueryArgs a{};
  KK_TRY(check_queries(out, q, c.heads, c.D, scale, &a, who));
  Paged4Rows rows{};
  KK_TRY(check_places(table, lengths, counts, window, c, a.B, &rows.a, who));
  rows.T = a.T;
  rows.D = a.D;
  rows.k = static_cast<const uint8_t*>(k_codes->data);
  rows.v = static_cast<const uint8_t*>(v_codes->data);
  rows.k_scale = static_cast<const uint32_t*>(k_scales->data);
  rows.v_scale = static_cast<const uint32_t*>(v_scales->data);
  KK_TRY(require_ready());
  if (a.B * a.T * a.heads == 0) return KK_OK;
  int status = KK_OK;
  if (few_paged4_try(a, rows, q->dtype, &status) || tiles_paged4_try(a, rows, q->dtype, &status)) return status;
  return q->dtype == KK_F16 ? launch_rows<__half>(a, rows) : launch_rows<float>(a, rows);
}

int kk_cross_attention(const kk_tensor* out, const kk_tensor* q, const kk_tensor* k, const kk_tensor* v,
                       const kk_tensor* lengths, const kk_tensor* mask, float scale) {
  const char* who = "cross_attention";
  KK_TRY(check_heads(k, "k", who));
  KK_TRY(check_heads(v, "v", who));
  QueryArgs a{};
  KK_TRY(check_queries(out, q, k->shape[2], k->shape[3], scale, &a, who));
  if (a.D < 1 || a.D > kMaxHead)
    return set_error(KK_E_UNSUPPORTED, "%s: heads of %d values (1 to %d)", who, a.D, kMaxHead);
  if (k->dtype != q->dtype || v->dtype != q->dtype)
    return set_error(KK_E_ARG, "%s: q, k and v must have one dtype", who);
  for (int i = 0; i < 4; ++i)
    if (k->shape[i] != v->shape[i]) return set_error(KK_E_ARG, "%s: k and v must have one shape", who);
  if (k->shape[0] != a.B) return set_error(KK_E_ARG, "%s: k must have q's sequences", who);
  DenseArgs d{};
  d.k = k->data;
  d.v = v->data;
  d.S = k->shape[1];
  for (int i = 0; i < 4; ++i) {
    d.ks[i] = k->strides[i];
    d.vs[i] = v->strides[i];
  }
  if (lengths) {
    KK_TRY(check_per_row(lengths, "lengths", a.B, true, who));
    d.lengths = lengths->data;
    d.lengths_dt = lengths->dtype;
    d.lengths_st = row_stride(lengths);
  }
  if (mask) {
    KK_TRY(check_tensor(mask, "mask"));
    const int r = mask->rank;
    if ((mask->dtype != KK_BOOL && mask->dtype != KK_U8) || r < 2 || r > 3 ||
        (mask->shape[0] != a.B && mask->shape[0] != 1) ||
        (r == 3 && mask->shape[1] != a.T && mask->shape[1] != 1) || mask->shape[r - 1] != d.S)
      return set_error(KK_E_ARG, "%s: mask must be bool [sequences, states] or [sequences, tokens, states]", who);
    d.mask = static_cast<const uint8_t*>(mask->data);
    d.ms[0] = mask->shape[0] > 1 ? mask->strides[0] : 0;
    d.ms[1] = r == 3 && mask->shape[1] > 1 ? mask->strides[1] : 0;
    d.ms[2] = mask->strides[r - 1];
  }
  KK_TRY(require_ready());
  if (a.B * a.T * a.heads == 0) return KK_OK;
  int status = KK_OK;
  if (few_dense_try(a, d, q->dtype, &status) || tiles_dense_try(a, d, q->dtype, &status)) return status;
  return q->dtype == KK_F16 ? launch_rows<__half>(a, DenseRows<__half>{d})
                            : launch_rows<float>(a, DenseRows<float>{d});
}

}  // extern "C"
