// What the decoder's translation units (kk_decode.hip, kk_attention.hip) share:
// loads of index tensors and the checks of their operands.
#pragma once

#include "kk_cache_index.h"
#include "kk_internal.h"

namespace kk {

inline bool is_index(int dt) { return dt == KK_I32 || dt == KK_I64; }

__device__ __forceinline__ int64_t load_index(const void* p, int dt, int64_t i) {
  return dt == KK_I32 ? static_cast<const int32_t*>(p)[i] : static_cast<const int64_t*>(p)[i];
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__half& d, float v) { d = __float2half(v); }

// A [B, T, H, D] operand: f32 or f16, values of a head next to each other.
inline int check_heads(const kk_tensor* t, const char* name, const char* who) {
  KK_TRY(check_tensor(t, name));
  if (t->rank != 4) return set_error(KK_E_ARG, "%s: %s must be [sequences, tokens, heads, values]", who, name);
  if (!is_float(t->dtype)) return set_error(KK_E_ARG, "%s: %s must be f32 or f16", who, name);
  if (numel(t) > 0 && t->shape[3] != 1 && t->strides[3] != 1)
    return set_error(KK_E_ARG, "%s: a head's values of %s must lie next to each other", who, name);
  return KK_OK;
}

inline int check_writable(const kk_tensor* t, const char* name, const char* who) {
  if (numel(t) == 0) return KK_OK;
  for (int i = 0; i < t->rank; ++i)
    if (t->shape[i] != 1 && t->strides[i] == 0)
      return set_error(KK_E_ARG, "%s: %s must not broadcast (axis %d has stride 0)", who, name, i);
  return KK_OK;
}

// One value a row, [B] or [1].
inline int check_per_row(const kk_tensor* t, const char* name, int64_t rows, bool index, const char* who) {
  KK_TRY(check_tensor(t, name));
  if (index ? !is_index(t->dtype) : t->dtype != KK_F32)
    return set_error(KK_E_ARG, "%s: %s must be %s", who, name, index ? "int32 or int64" : "f32");
  if (t->rank != 1 || (t->shape[0] != rows && t->shape[0] != 1))
    return set_error(KK_E_ARG, "%s: %s must have one value, or one a row", who, name);
  return KK_OK;
}
inline int64_t row_stride(const kk_tensor* t) { return t->shape[0] == 1 ? 0 : t->strides[0]; }

// [rows, cols] of `dt`, or [1, cols] / [cols] for all rows; *stride the row's.
inline int check_by_row(const kk_tensor* t, const char* name, int64_t rows, int64_t cols, int64_t* stride,
                        const char* who) {
  KK_TRY(check_tensor(t, name));
  const bool one = t->rank == 1;
  if ((!one && t->rank != 2) || t->shape[t->rank - 1] != cols || (!one && t->shape[0] != rows && t->shape[0] != 1))
    return set_error(KK_E_ARG, "%s: %s must be [%lld] or [%lld, %lld]", who, name, static_cast<long long>(cols),
                     static_cast<long long>(rows), static_cast<long long>(cols));
  if (cols > 1 && rows > 0 && t->strides[t->rank - 1] != 1)
    return set_error(KK_E_ARG, "%s: a row of %s must lie in one piece", who, name);
  *stride = one || t->shape[0] == 1 ? 0 : t->strides[0];
  return KK_OK;
}


// A paged cache of 8-bit codes.
struct CacheShape {
  int64_t pages, heads, block, D, columns, table_stride;
};

// Checks a cache's four tensors against each other.
inline int check_codes(const kk_tensor* k_codes, const kk_tensor* k_scales, const kk_tensor* v_codes,
                       const kk_tensor* v_scales, CacheShape* c, const char* who) {
  const kk_tensor *codes[2] = {k_codes, v_codes}, *scales[2] = {k_scales, v_scales};
  const char *names[2] = {"k_codes", "v_codes"}, *snames[2] = {"k_scales", "v_scales"};
  for (int i = 0; i < 2; ++i) {
    KK_TRY(check_tensor(codes[i], names[i]));
    KK_TRY(check_tensor(scales[i], snames[i]));
    if (codes[i]->dtype != KK_I8 || codes[i]->rank != 4 || !is_contiguous(codes[i]) ||
        reinterpret_cast<uintptr_t>(codes[i]->data) % 16)
      return set_error(KK_E_ARG, "%s: %s must be int8 of four axes in one piece, 16-byte aligned", who, names[i]);
    if (scales[i]->dtype != KK_F32 || scales[i]->rank != 2 || !is_contiguous(scales[i]) ||
        scales[i]->shape[0] != codes[0]->shape[0] || scales[i]->shape[1] != codes[0]->shape[1])
      return set_error(KK_E_ARG, "%s: %s must be f32 [pages, heads] in one piece", who, snames[i]);
  }
  c->pages = k_codes->shape[0];
  c->heads = k_codes->shape[1];
  c->block = k_codes->shape[2];
  c->D = k_codes->shape[3];
  if (v_codes->shape[0] != c->pages || v_codes->shape[1] != c->heads || v_codes->shape[2] != c->D ||
      v_codes->shape[3] != c->block)
    return set_error(KK_E_ARG, "%s: v_codes must be [pages, heads, values, rows] of k_codes' [pages, heads, rows, "
                     "values]", who);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128 && c->block != 256)
    return set_error(KK_E_UNSUPPORTED, "%s: pages of %lld rows (16, 32, 64, 128 or 256)", who,
                     static_cast<long long>(c->block));
  if (c->D < 16 || c->D > 256 || c->D % 16)
    return set_error(KK_E_UNSUPPORTED, "%s: heads of %lld values (16 to 256 in steps of 16)", who,
                     static_cast<long long>(c->D));
  if (c->heads < 1 || c->heads > 65535) return set_error(KK_E_UNSUPPORTED, "%s: %lld heads", who,
                                                         static_cast<long long>(c->heads));
  c->columns = c->table_stride = 0;
  return KK_OK;
}

// A table of a cache's pages.
inline int check_cache_table(const kk_tensor* table, CacheShape* c, const char* who) {
  KK_TRY(check_tensor(table, "table"));
  if (table->dtype != KK_I32 || table->rank != 2)
    return set_error(KK_E_ARG, "%s: table must be int32 [sequences, pages]", who);
  c->columns = table->shape[1];
  if (c->columns > (int64_t{1} << 40))
    return set_error(KK_E_UNSUPPORTED, "%s: a table of %lld columns", who, static_cast<long long>(c->columns));
  if (c->columns > 1 && table->shape[0] > 0 && table->strides[1] != 1)
    return set_error(KK_E_ARG, "%s: a row of table must lie in one piece", who);
  c->table_stride = table->shape[0] > 1 ? table->strides[0] : 0;
  return KK_OK;
}

// The same with a table of its pages.
inline int check_cache(const kk_tensor* k_codes, const kk_tensor* k_scales, const kk_tensor* v_codes,
                       const kk_tensor* v_scales, const kk_tensor* table, CacheShape* c, const char* who) {
  KK_TRY(check_codes(k_codes, k_scales, v_codes, v_scales, c, who));
  return check_cache_table(table, c, who);
}

// A paged cache of 4-bit codes, two a byte, with a step and a lowest value for
// each token and head.
inline int check_codes4(const kk_tensor* k_codes, const kk_tensor* k_scales, const kk_tensor* v_codes,
                        const kk_tensor* v_scales, CacheShape* c, const char* who) {
  const kk_tensor *codes[2] = {k_codes, v_codes}, *scales[2] = {k_scales, v_scales};
  const char *names[2] = {"k_codes", "v_codes"}, *snames[2] = {"k_scales", "v_scales"};
  for (int i = 0; i < 2; ++i) {
    KK_TRY(check_tensor(codes[i], names[i]));
    KK_TRY(check_tensor(scales[i], snames[i]));
    if (codes[i]->dtype != KK_U8 || codes[i]->rank != 4 || !is_contiguous(codes[i]) ||
        reinterpret_cast<uintptr_t>(codes[i]->data) % 16)
      return set_error(KK_E_ARG, "%s: %s must be uint8 of four axes in one piece, 16-byte aligned", who, names[i]);
  }
  c->pages = k_codes->shape[0];
  c->heads = k_codes->shape[1];
  c->block = k_codes->shape[2];
  c->D = 2 * k_codes->shape[3];
  if (v_codes->shape[0] != c->pages || v_codes->shape[1] != c->heads || v_codes->shape[2] != c->D / 2 ||
      v_codes->shape[3] != c->block)
    return set_error(KK_E_ARG, "%s: v_codes must be [pages, heads, values / 2, rows] of k_codes' [pages, heads, rows, "
                     "values / 2]", who);
  for (int i = 0; i < 2; ++i)
    if (scales[i]->dtype != KK_F16 || scales[i]->rank != 4 || !is_contiguous(scales[i]) ||
        scales[i]->shape[0] != c->pages || scales[i]->shape[1] != c->heads || scales[i]->shape[2] != c->block ||
        scales[i]->shape[3] != 2 || reinterpret_cast<uintptr_t>(scales[i]->data) % 16)
      return set_error(KK_E_ARG, "%s: %s must be f16 [pages, heads, rows, 2] in one piece, 16-byte aligned", who,
                       snames[i]);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128 && c->block != 256)
    return set_error(KK_E_UNSUPPORTED, "%s: pages of %lld rows (16, 32, 64, 128 or 256)", who,
                     static_cast<long long>(c->block));
  if (c->D < 32 || c->D > 256 || c->D % 32)
    return set_error(KK_E_UNSUPPORTED, "%s: heads of %lld values (32 to 256 in steps of 32)", who,
                     static_cast<long long>(c->D));
  if (c->heads < 1 || c->heads > 65535) return set_error(KK_E_UNSUPPORTED, "%s: %lld heads", who,
                                                         static_cast<long long>(c->heads));
  if (c->pages > 0x7fffffff) return set_error(KK_E_UNSUPPORTED, "%s: too many pages", who);
  c->columns = c->table_stride = 0;
  return KK_OK;
}

}  // namespace kk
