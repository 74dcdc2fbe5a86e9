// sg_kvq8.hip - the quantised cache of keys and values: tokens quantised as
// they are written behind it, and read back as 16-bit rows.
//
// The reference's cache has the same two forms, fp16 and blocks of 32 8-bit
// values (KV append, attention.cu:52-442); here codes and scales lie apart,
// each in pages of their own, so that rows of codes are a power of two long.
//
//   d = fp16(max |x| / 127) over 32 values, at most 515.5 (127 of which are
//   still a finite fp16 number), code = x / d to the nearest, ties to even.
//
// A quotient of two fp16 numbers below 191 lies either on a tie, or 2^-12 away
// from it or more: |x - (n + 1/2) d| is a whole multiple of half of d's last
// bit. So x times a reciprocal (2^-16 off at the most) is first rounded to
// multiples of 2^-13, which brings a quotient on a tie back to it and moves no
// other over one; the code is that of an exact division, without one.
// A group that holds an infinity or a NaN has a NaN for its scale and reads as
// NaN throughout.
#include "sg_cache.hpp"

namespace sg {

typedef unsigned short us2 __attribute__((ext_vector_type(2)));
constexpr int kStoreLayers = 2;  // of a thread, loads under way together
constexpr int kReadLayers = 2;

struct StoreQ8Args {
  const uint16_t *k, *v;
  long long k_stride, v_stride, k_layer, v_layer, layer_stride;
  int8_t *kc, *vc;
  uint16_t *ks, *vs;
  const int *pages, *length, *win_off, *path, *n_path;
  int* length_out;
  int n_tokens, max_window, n_layers, n_kv, dim, n_pages, page_log2, pages_per_seq;
};

// 16 values of a group whose other 16 the next or the last lane has.
__device__ __forceinline__ void quantise16(const u32x4 (&x)[2], u32x4& code, uint32_t& scale) {
  us2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, x[i / 4][i % 4] & 0x7FFF7FFFu));
  int top = max(static_cast<int>(m.x), static_cast<int>(m.y));
  top = max(top, dpp_i<kDppXor1>(top));
  const bool finite = top < 0x7C00;
  const float d = fminf(f16v(f16b(half_bits_to_float(top) / 127.f)), 515.5f);
  scale = finite ? f16b(d) : 0x7E00u;
  const float inv = finite && d > 0.f ? __builtin_amdgcn_rcpf(d) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = 4 * i + j;
      const float v = half_bits_to_float(x[n / 8][n / 2 % 4] >> (16 * (n & 1)) & 0xFFFFu);
      const float t = __builtin_fmaf(finite ? v : 0.f, inv, 1536.f) - 1536.f;
      // (1.5 * 2^23 more: the whole number in the low bits, rounded to even)
      const float r = __builtin_amdgcn_fmed3f(t, -127.f, 127.f) + 12582912.f;
      w |= (__builtin_bit_cast(uint32_t, r) & 0xFFu) << (8 * j);
    }
    code[i] = w;
  }
}

// Grid: (16-value pieces of a window's K and V rows, sequence, kStoreLayers
// layers).  A thread looks its piece's place up once for its layers.  Waves behind
// a window's end leave at once, but there are many where one window is long and
// others are short (1,091 tokens in five windows of up to 1,021, ten layers of 8
// heads of 128: 68 MB in 19 us, 3.6 TB/s, four of five waves and some two fifths of
// the vector instructions without a piece; over the same buffers again and again
// 15.6, as one window 13.7); else memory bounds long windows, and four dependent
// rounds four tokens, 4.4 us.
__global__ void __launch_bounds__(256) kv_store_q8_kernel(const StoreQ8Args a) {
  const int s = blockIdx.y, l0 = blockIdx.z * kStoreLayers;
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  const int n = a.path ? min(max(a.n_path[s], 0), a.max_window) : w.n;
  const int len = a.length[s];
  if (a.length_out && blockIdx.x == 0 && l0 == 0 && threadIdx.x == 0) a.length_out[s] = len + n;
  const int lanes = a.dim / 16;  // (even: a group's two lanes go the same way)
  int x = blockIdx.x * 256 + threadIdx.x;
  const int row = x / lanes, c = x - row * lanes;
  const int i = row / (2 * a.n_kv), in = row - i * 2 * a.n_kv;
  if (i >= n) return;
  const bool is_v = in >= a.n_kv;
  const int h = is_v ? in - a.n_kv : in;
  const int node = a.path ? a.path[static_cast<long long>(s) * a.max_window + i] : i;
  const long long pos = static_cast<long long>(len) + i;
  if (len < 0 || node < 0 || node >= w.n || pos >> a.page_log2 >= a.pages_per_seq) return;
  const int page = a.pages[static_cast<long long>(s) * a.pages_per_seq + (pos >> a.page_log2)];
  if (page < 0 || page >= a.n_pages) return;
  const long long step = is_v ? a.v_layer : a.k_layer;
  const uint16_t* src =
      (is_v ? a.v + (w.off + node) * a.v_stride : a.k + (w.off + node) * a.k_stride) + h * a.dim +
      c * 16 + l0 * step;
  const long long slot = ((static_cast<long long>(page) * a.n_kv + h) << a.page_log2) +
                         (pos & ((1 << a.page_log2) - 1));
  const long long at = l0 * a.layer_stride + slot * a.dim + c * 16;
  int8_t* codes = (is_v ? a.vc : a.kc) + at;
  uint16_t* scales = (is_v ? a.vs : a.ks) + at / kKvGroup;
  const int layers = min(kStoreLayers, a.n_layers - l0);
  u32x4 v[kStoreLayers][2];
#pragma unroll
  for (int l = 0; l < kStoreLayers; ++l)
    if (l < layers) {
      v[l][0] = *reinterpret_cast<const u32x4_u*>(src + l * step);
      v[l][1] = *reinterpret_cast<const u32x4_u*>(src + l * step + 8);
    }
#pragma unroll
  for (int l = 0; l < kStoreLayers; ++l)
    if (l < layers) {
      u32x4 code;
      uint32_t scale;
      quantise16(v[l], code, scale);
      *reinterpret_cast<u32x4*>(codes + l * a.layer_stride) = code;
      if ((c & 1) == 0) scales[l * (a.layer_stride / kKvGroup)] = static_cast<uint16_t>(scale);
    }
}

struct ReadQ8Args {
  const int8_t *kc, *vc;
  const uint16_t *ks, *vs;
  uint16_t *k, *v;
  long long k_stride, v_stride, k_layer, v_layer, layer_stride;
  const int *pages, *first, *rows;
  int n_seq, n_rows, n_layers, n_kv, dim, n_pages, page_log2, pages_per_seq;
};

// Grid: (waves of all rows, K or V, kReadLayers layers).  A wave has one head's
// pieces of as many tokens as it has lanes for, whose codes lie in line.  Bound
// by memory (32,749 tokens of ten layers of 2 heads of 256: 1.03 GB in 205 us,
// 5.0 TB/s, as a large copy), for few tokens by three dependent rounds, 3.3 us.
__global__ void __launch_bounds__(256) kv_read_q8_kernel(const ReadQ8Args a) {
  const int lane = threadIdx.x & 63, lanes = a.dim / 16, rows = 64 / lanes;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int block = wave / a.n_kv, h = wave - block * a.n_kv, l0 = blockIdx.z * kReadLayers;
  const bool is_v = blockIdx.y != 0;
  // (one sequence for the wave's first row, then on to the lane's own)
  const long long r0 = static_cast<long long>(block) * rows;
  if (r0 >= a.n_rows) return;
  int s = seq_of_row(a.rows, a.n_seq, static_cast<int>(r0), lane);
  const int r = static_cast<int>(r0) + lane / lanes, c = lane % lanes;
  if (r >= a.n_rows) return;
  while (s + 1 < a.n_seq && a.rows[s + 1] <= r) ++s;
  const int begin = a.rows[s];
  if (r < begin || begin < 0 || r >= a.rows[s + 1]) return;
  const long long pos = static_cast<long long>(a.first[s]) + (r - begin);
  int page = -1;
  if (pos >= 0 && pos >> a.page_log2 < a.pages_per_seq)
    page = a.pages[static_cast<long long>(s) * a.pages_per_seq + (pos >> a.page_log2)];
  const bool there = page >= 0 && page < a.n_pages;
  const long long slot = ((static_cast<long long>(there ? page : 0) * a.n_kv + h) << a.page_log2) +
                         (there ? pos & ((1 << a.page_log2) - 1) : 0);
  const long long at = l0 * a.layer_stride + slot * a.dim + c * 16;
  const int8_t* codes = (is_v ? a.vc : a.kc) + at;
  const uint16_t* scales = (is_v ? a.vs : a.ks) + at / kKvGroup;
  const long long step = is_v ? a.v_layer : a.k_layer;
  uint16_t* dst = (is_v ? a.v : a.k) + r * (is_v ? a.v_stride : a.k_stride) + h * a.dim + c * 16 +
                  l0 * step;
  const int layers = min(kReadLayers, a.n_layers - l0);
  u32x4 code[kReadLayers];
  uint32_t scale[kReadLayers];
#pragma unroll
  for (int l = 0; l < kReadLayers; ++l)
    if (l < layers) {
      code[l] = *reinterpret_cast<const u32x4*>(codes + l * a.layer_stride);
      scale[l] = scales[l * (a.layer_stride / kKvGroup)];
    }
#pragma unroll
  for (int l = 0; l < kReadLayers; ++l)
    if (l < layers) {
      uint32_t y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t two[2];
        decode4(code[l][i], scale2(scale[l]), two);
        y[2 * i] = there ? two[0] : 0u;
        y[2 * i + 1] = there ? two[1] : 0u;
      }
      u32x4_u* out = reinterpret_cast<u32x4_u*>(dst + l * step);
      out[0] = (u32x4){y[0], y[1], y[2], y[3]};
      out[1] = (u32x4){y[4], y[5], y[6], y[7]};
    }
}

static int store_q8(const uint16_t* k, const uint16_t* v, long long k_stride, long long v_stride,
                    long long k_layer_stride, long long v_layer_stride, const sg_kv_cache_q8* cache,
                    const int* win_off, const int* path, const int* n_path, int* length_out,
                    int n_seq, int n_tokens, int max_window, int most, void* stream,
                    const char* nm) {
  if (!k || !v || !win_off) return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (int st = check_cache(cache, n_seq, n_tokens, max_window, nm, most)) return st;
  const long long row = static_cast<long long>(cache->n_kv_heads) * cache->head_dim;
  if (k_stride < row || v_stride < row)
    return set_error(SG_ERR_GEOMETRY, "%s: a token stride is less than a token", nm);
  if (reinterpret_cast<uintptr_t>(k) % 2 || reinterpret_cast<uintptr_t>(v) % 2)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: k and v must be 2-B aligned", nm);
  const long long pieces = 2LL * max_window * (row / 16);
  if (n_seq > 65535 || cache->n_layers > 65535 || pieces > 0x7FFFFFFF - 256)
    return set_error(SG_ERR_UNSUPPORTED, "%s: n_seq=%d n_layers=%d max_window=%d n_kv_heads=%d", nm,
                     n_seq, cache->n_layers, max_window, cache->n_kv_heads);
  // (a sequence's first workgroup writes its new length, the others read on)
  const long long paths = static_cast<long long>(n_seq) * max_window;
  const long long pages = static_cast<long long>(n_seq) * cache->pages_per_seq;
  if (length_out &&
      (overlap(length_out, n_seq, cache->length, n_seq) || overlap(length_out, n_seq, n_path, n_seq) ||
       overlap(length_out, n_seq, path, paths) || overlap(length_out, n_seq, win_off, n_seq + 1LL) ||
       overlap(length_out, n_seq, cache->pages, pages) ||
       over_rows(length_out, n_seq, k, row, k_stride, n_tokens, k_layer_stride, cache->n_layers) ||
       over_rows(length_out, n_seq, v, row, v_stride, n_tokens, v_layer_stride, cache->n_layers) ||
       over_layers(length_out, n_seq, cache)))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: length_out overlaps the cache, n_path, path, win_off, k or v", nm);
  StoreQ8Args a;
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.k_layer = k_layer_stride;
  a.v_layer = v_layer_stride;
  a.layer_stride = cache->layer_stride;
  a.kc = cache->k;
  a.vc = cache->v;
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.pages = cache->pages;
  a.length = cache->length;
  a.win_off = win_off;
  a.path = path;
  a.n_path = n_path;
  a.length_out = length_out;
  a.n_tokens = n_tokens;
  a.max_window = max_window;
  a.n_layers = cache->n_layers;
  a.n_kv = cache->n_kv_heads;
  a.dim = cache->head_dim;
  a.n_pages = cache->n_pages;
  a.page_log2 = log2_of(cache->page_size);
  a.pages_per_seq = cache->pages_per_seq;
  hipLaunchKernelGGL(kv_store_q8_kernel,
                     dim3(static_cast<unsigned>((pieces + 255) / 256), n_seq,
                          (cache->n_layers + kStoreLayers - 1) / kStoreLayers),
                     dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return check_launch(nm);
}

}  // namespace sg

extern "C" {

int sg_kv_commit_q8(const uint16_t* k, const uint16_t* v, long long k_stride, long long v_stride,
                    long long k_layer_stride, long long v_layer_stride, const sg_kv_cache_q8* cache,
                    const int* win_off, const int* path, const int* n_path, int* length_out,
                    int n_seq, int n_tokens, int max_window, void* stream) {
  const char* nm = "sg_kv_commit_q8";
  if (!path || !n_path) return sg::set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  return sg::store_q8(k, v, k_stride, v_stride, k_layer_stride, v_layer_stride, cache, win_off,
                      path, n_path, length_out, n_seq, n_tokens, max_window, sg::kMaxWindow,
                      stream, nm);
}

int sg_kv_append_q8(const uint16_t* k, const uint16_t* v, long long k_stride, long long v_stride,
                    long long k_layer_stride, long long v_layer_stride, const sg_kv_cache_q8* cache,
                    const int* win_off, int* length_out, int n_seq, int n_tokens, int max_window,
                    void* stream) {
  return sg::store_q8(k, v, k_stride, v_stride, k_layer_stride, v_layer_stride, cache, win_off,
                      nullptr, nullptr, length_out, n_seq, n_tokens, max_window, 0x7FFFF000,
                      stream, "sg_kv_append_q8");
}

int sg_kv_read_q8(const sg_kv_cache_q8* cache, const int* first, const int* row_off, uint16_t* k,
                  uint16_t* v, long long k_stride, long long v_stride, long long k_layer_stride,
                  long long v_layer_stride, int n_seq, int n_rows, void* stream) {
  const char* nm = "sg_kv_read_q8";
  using namespace sg;
  if (!k || !v || !first || !row_off)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (int st = check_cache(cache, n_seq, n_rows, 1, nm)) return st;
  const long long row = static_cast<long long>(cache->n_kv_heads) * cache->head_dim;
  if (k_stride < row || v_stride < row)
    return set_error(SG_ERR_GEOMETRY, "%s: a token stride is less than a token", nm);
  const long long span_k = (n_rows - 1LL) * k_stride + row, span_v = (n_rows - 1LL) * v_stride + row;
  if (cache->n_layers > 1 && (k_layer_stride < span_k || v_layer_stride < span_v))
    return set_error(SG_ERR_GEOMETRY, "%s: a layer stride is less than a layer's rows", nm);
  if (reinterpret_cast<uintptr_t>(k) % 2 || reinterpret_cast<uintptr_t>(v) % 2)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: k and v must be 2-B aligned", nm);
  const int rows = 64 / (cache->head_dim / 16);  // of a wave
  const long long waves = (n_rows - 1LL + rows) / rows * cache->n_kv_heads;
  const int groups = (cache->n_layers + kReadLayers - 1) / kReadLayers;
  // (a launch has less than 2^32 threads in a row)
  if (cache->n_layers > 65535 || waves > 0xFFFFFFFFLL / 64 - 4)
    return set_error(SG_ERR_UNSUPPORTED, "%s: n_rows=%d n_layers=%d n_kv_heads=%d", nm, n_rows,
                     cache->n_layers, cache->n_kv_heads);
  const long long nk = (cache->n_layers - 1) * k_layer_stride + span_k;
  const long long nv = (cache->n_layers - 1) * v_layer_stride + span_v;
  const long long codes = cache_values(cache), scales = codes / kKvGroup;
  const uint16_t* const outs[2] = {k, v};
  const long long sizes[2] = {nk, nv};
  for (int i = 0; i < 2; ++i)
    if (overlap(outs[i], sizes[i], cache->k, codes) || overlap(outs[i], sizes[i], cache->v, codes) ||
        overlap(outs[i], sizes[i], cache->k_scale, scales) ||
        overlap(outs[i], sizes[i], cache->v_scale, scales) ||
        overlap(outs[i], sizes[i], cache->pages, static_cast<long long>(n_seq) * cache->pages_per_seq) ||
        overlap(outs[i], sizes[i], first, n_seq) || overlap(outs[i], sizes[i], row_off, n_seq + 1LL))
      return set_error(SG_ERR_INVALID_ARGUMENT,
                       "%s: an output overlaps the cache, first or row_off", nm);
  if (overlap(k, nk, v, nv)) return set_error(SG_ERR_INVALID_ARGUMENT, "%s: k overlaps v", nm);
  ReadQ8Args a;
  a.kc = cache->k;
  a.vc = cache->v;
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.k_layer = k_layer_stride;
  a.v_layer = v_layer_stride;
  a.layer_stride = cache->layer_stride;
  a.pages = cache->pages;
  a.first = first;
  a.rows = row_off;
  a.n_seq = n_seq;
  a.n_rows = n_rows;
  a.n_layers = cache->n_layers;
  a.n_kv = cache->n_kv_heads;
  a.dim = cache->head_dim;
  a.n_pages = cache->n_pages;
  a.page_log2 = log2_of(cache->page_size);
  a.pages_per_seq = cache->pages_per_seq;
  hipLaunchKernelGGL(kv_read_q8_kernel,
                     dim3(static_cast<unsigned>((waves + 3) / 4), 2, groups), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch(nm);
}

}  // extern "C"
