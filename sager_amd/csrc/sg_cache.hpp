// sg_cache.hpp - the paged caches of keys and values: their checks, and the
// 8-bit values of the quantised one.
//
// A group of 32 values has one scale d, the 16-bit number nearest to its
// largest magnitude / 127; a value's code is the whole number nearest to
// value / d (ties to even), and code * d is what it is read as.
#pragma once

#include "sg_window.hpp"

namespace sg {

constexpr int kKvGroup = 32;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));

// Codes 4 w .. 4 w + 3 as they are read: a byte with its sign flipped behind
// 0x64 is 1024 + 128 + code in 16 bits, so a difference of 1152 is the code
// without an error, and the product is rounded once.
__device__ __forceinline__ void decode4(uint32_t codes, h2 d, uint32_t (&out)[2]) {
  const uint32_t u = codes ^ 0x80808080u;
  const h2 bias = {static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
  const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
  const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
  out[0] = __builtin_bit_cast(uint32_t, (a - bias) * d);
  out[1] = __builtin_bit_cast(uint32_t, (b - bias) * d);
}
// The same in two parts, value rounded and what the rounding took: their sum is
// code * d without an error (18 bits at the most, and a multiple of 2^-24).
__device__ __forceinline__ void decode4(uint32_t codes, h2 d, uint32_t (&out)[2],
                                        uint32_t (&rest)[2]) {
  const uint32_t u = codes ^ 0x80808080u;
  const h2 bias = {static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
  const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
  const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
  const h2 x = a * d, y = b * d;
  out[0] = __builtin_bit_cast(uint32_t, x);
  out[1] = __builtin_bit_cast(uint32_t, y);
  rest[0] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(a, d, -x));
  rest[1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(b, d, -y));
}
__device__ __forceinline__ h2 scale2(uint32_t bits) {  // one scale in both halves
  return __builtin_bit_cast(h2, (bits & 0xFFFFu) * 0x10001u);
}

// ---- host ---------------------------------------------------------------------
static inline int log2_of(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

// What the two caches have in common.
template <typename C>
static int check_cache_shape(const C* c, int n_seq, int n_tokens, int max_window, int most,
                             const char* nm) {
  if (n_seq <= 0 || n_tokens <= 0 || max_window <= 0 || c->n_layers <= 0 || c->n_pages <= 0 ||
      c->pages_per_seq <= 0 || c->n_kv_heads <= 0)
    return set_error(SG_ERR_GEOMETRY,
                     "%s: n_seq=%d n_tokens=%d max_window=%d n_layers=%d n_pages=%d "
                     "pages_per_seq=%d n_kv_heads=%d must be positive",
                     nm, n_seq, n_tokens, max_window, c->n_layers, c->n_pages, c->pages_per_seq,
                     c->n_kv_heads);
  if (max_window > most)
    return set_error(SG_ERR_UNSUPPORTED, "%s: max_window=%d is over %d", nm, max_window, most);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return set_error(SG_ERR_UNSUPPORTED, "%s: head_dim=%d is not 64, 128 or 256", nm, c->head_dim);
  if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) != 0)
    return set_error(SG_ERR_UNSUPPORTED, "%s: page_size=%d is no power of two from 16 on", nm,
                     c->page_size);
  // token positions are 32-bit
  if ((static_cast<long long>(c->pages_per_seq) << log2_of(c->page_size)) > 0x7FFFF000LL)
    return set_error(SG_ERR_UNSUPPORTED, "%s: a sequence of %d pages of %d tokens is too long", nm,
                     c->pages_per_seq, c->page_size);
  return SG_OK;
}
static inline int check_cache(const sg_kv_cache* c, int n_seq, int n_tokens, int max_window,
                              const char* nm, int most = kMaxWindow) {
  if (!c || !c->k || !c->v || !c->pages || !c->length)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null cache", nm);
  if (int st = check_cache_shape(c, n_seq, n_tokens, max_window, most, nm)) return st;
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 ||
      c->layer_stride % 8)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: the cache is not 16-B aligned", nm);
  return SG_OK;
}
static inline int check_cache(const sg_kv_cache_q8* c, int n_seq, int n_tokens, int max_window,
                              const char* nm, int most = kMaxWindow) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->pages || !c->length)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null cache", nm);
  if (int st = check_cache_shape(c, n_seq, n_tokens, max_window, most, nm)) return st;
  if (c->n_layers > 1 && c->layer_stride < static_cast<long long>(c->n_pages) * c->n_kv_heads *
                                               c->page_size * c->head_dim)
    return set_error(SG_ERR_GEOMETRY, "%s: the layer stride is less than a layer", nm);
  // (a row's scales are 4, 8 or 16 B and are read as such)
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) |
       reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) % 16 ||
      c->layer_stride % (16 * kKvGroup))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: the cache is not 16-B aligned, or its layers not a multiple of 512 apart",
                     nm);
  return SG_OK;
}

// Whether n ints lie over one of `layers` layers of `rows` rows of `width` values, `stride` apart
// (width or more), `layer` from one layer to the next; what lies between rows is nobody's.
template <typename T>
static inline bool over_rows(const int* ints, long long n, const T* x, long long width,
                             long long stride, long long rows, long long layer, int layers) {
  for (int l = 0; ints && l < layers; ++l) {
    const T* const base = x + l * layer;
    if (!overlap(ints, n, base, (rows - 1) * stride + width)) continue;
    const long long s = stride * static_cast<long long>(sizeof(T));
    const long long w = width * static_cast<long long>(sizeof(T));
    const long long from = static_cast<long long>(reinterpret_cast<uintptr_t>(ints)) -
                           static_cast<long long>(reinterpret_cast<uintptr_t>(base));
    const long long row = from < w ? 0 : (from - w) / s + 1;  // the first that ends behind them
    if (row < rows && row * s < from + n * static_cast<long long>(sizeof(int))) return true;
  }
  return false;
}

// Whether n ints lie over one of a cache's layers.
static inline bool over_layers(const int* ints, long long n, const sg_kv_cache* c) {
  const long long m = static_cast<long long>(c->n_pages) * c->n_kv_heads * c->page_size * c->head_dim;
  return over_rows(ints, n, c->k, m, m, 1, c->layer_stride, c->n_layers) ||
         over_rows(ints, n, c->v, m, m, 1, c->layer_stride, c->n_layers);
}
static inline bool over_layers(const int* ints, long long n, const sg_kv_cache_q8* c) {
  const long long m = static_cast<long long>(c->n_pages) * c->n_kv_heads * c->page_size * c->head_dim;
  const long long s = m / kKvGroup, layer = c->layer_stride / kKvGroup;
  return over_rows(ints, n, c->k, m, m, 1, c->layer_stride, c->n_layers) ||
         over_rows(ints, n, c->v, m, m, 1, c->layer_stride, c->n_layers) ||
         over_rows(ints, n, c->k_scale, s, s, 1, layer, c->n_layers) ||
         over_rows(ints, n, c->v_scale, s, s, 1, layer, c->n_layers);
}

// Values from a cache's first to its last layer's end.
static inline long long cache_values(const sg_kv_cache_q8* c) {
  return (c->n_layers - 1) * c->layer_stride +
         static_cast<long long>(c->n_pages) * c->n_kv_heads * c->page_size * c->head_dim;
}

}  // namespace sg
