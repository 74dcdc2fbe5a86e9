// sg_norm.hip - residual addition, RMS norm and Q8_K of the result in one
// launch: what lies between a layer's output projection and the next
// projections, the router or the MoE layer (which take the fp16 rows and
// their Q8_K).
//
//   r = x + y (rounded to the buffers' type: the residual stream as stored),
//   s = 1 / sqrt(mean(r^2) + eps),   xn = (r * s) * w (rounded likewise),
//   Q8_K(xn), the codes of sg_quantize_q8_k{,_f16}.
//
// The sum of squares is fp32: per lane in index order, then over the lanes.
// Squares are summed in 32 bits because 16 would lose the small channels
// beside the few large ones of a residual stream.
//
// Every value is read and written once and lives in registers in between: a
// workgroup a row, a wave a block of 256 values as far as 16 waves go, which
// is also the Q8_K quantizer's layout.  Few rows are bound by latency (one
// round of loads, one barrier, one round of stores): 4 rows of 2048 fp16
// values 2.6 us.  Many are bound by memory: 4096 rows, 76 MB with r, xn and
// the blocks, 20 us, 3.8 TB/s where a large copy gets 4.8.  (Four waves with
// two of the blocks each: 3.3 us for the 4 rows.)
#include "sg_common.hpp"

namespace sg {

// four consecutive values of a row, at the element's own alignment (buffers
// may be slices of larger ones)
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_u __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
struct Act;
template <>
struct Act<float> {
  typedef f32x4_u vec;
  static __device__ __forceinline__ float val(float v) { return v; }
  static __device__ __forceinline__ float bits(float v) { return v; }
};
template <>
struct Act<uint16_t> {
  typedef u16x4_u vec;
  static __device__ __forceinline__ float val(uint16_t v) { return half_bits_to_float(v); }
  static __device__ __forceinline__ uint16_t bits(float v) { return f16b(v); }
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  const typename Act<T>::vec q = *reinterpret_cast<const typename Act<T>::vec*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = Act<T>::val(q[i]);
}
// stores v rounded to T and leaves in v what was stored
template <typename T>
__device__ __forceinline__ void store4(T* p, float (&v)[4]) {
  typename Act<T>::vec q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    q[i] = Act<T>::bits(v[i]);
    v[i] = Act<T>::val(q[i]);
  }
  *reinterpret_cast<typename Act<T>::vec*>(p) = q;
}
template <typename T>
__device__ __forceinline__ void round4(float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = Act<T>::val(Act<T>::bits(v[i]));
}

// Sum over the wave in a fixed order, same value in every lane.
__device__ __forceinline__ float wave_sum_dpp(float v) {
  v += dpp_f<kDppXor1>(v);
  v += dpp_f<kDppXor2>(v);
  v += dpp_f<kDppHalfMirror>(v);
  v += dpp_f<kDppMirror>(v);
  return (readlane_f(v, 0) + readlane_f(v, 16)) + (readlane_f(v, 32) + readlane_f(v, 48));
}

// kNW waves per row, each up to kB blocks of 256 values held in registers
// (lane l has values 4l..4l+3 of a block, the layout of the Q8_K quantizer).
template <typename T, int kNW, int kB>
__global__ void __launch_bounds__(64 * kNW)
    add_rmsnorm_kernel(const T* x, const T* y, T* x_out, const float* w, T* xn,
                       unsigned char* xq, int n, int n_rows, float eps) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const long long row = blockIdx.x;
  const int nb = n / kQK;
  const long long at = row * n + 4 * lane;
  float v[kB][4], wv[kB][4];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kB; ++i) {
    const int b = wave + kNW * i;
    if (b < nb) {
      load4(x + at + b * kQK, v[i]);
      load4(w + b * kQK + 4 * lane, wv[i]);
    }
  }
  if (y) {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int b = wave + kNW * i;
      if (b < nb) {
        float a[4];
        load4(y + at + b * kQK, a);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] += a[j];
        store4(x_out + at + b * kQK, v[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kB; ++i)
    if (wave + kNW * i < nb)
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(v[i][j], v[i][j], ss);
  ss = wave_sum_dpp(ss);
  __shared__ float part_ss[kNW];
  if (lane == 0) part_ss[wave] = ss;
  __syncthreads();
  ss = part_ss[0];
#pragma unroll
  for (int i = 1; i < kNW; ++i) ss += part_ss[i];
  const float s = 1.f / sqrtf(ss / static_cast<float>(n) + eps);
#pragma unroll
  for (int i = 0; i < kB; ++i) {
    const int b = wave + kNW * i;
    if (b < nb) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = (v[i][j] * s) * wv[i][j];
      if (xn)
        store4(xn + at + b * kQK, v[i]);
      else
        round4<T>(v[i]);
      if (xq) quantize_block_wave(v[i], xq + (row * nb + b) * kQ8Bytes, lane);
    }
  }
}

template <typename T, int kNW, int kB>
static void norm_go(const T* x, const T* y, T* x_out, const float* w, float eps, T* xn,
                    sg_block_q8k* xq, int n, int n_rows, hipStream_t s) {
  hipLaunchKernelGGL((add_rmsnorm_kernel<T, kNW, kB>), dim3(n_rows), dim3(64 * kNW), 0, s, x, y,
                     x_out, w, xn, reinterpret_cast<unsigned char*>(xq), n, n_rows, eps);
}

template <typename T>
static int norm_launch(const T* x, const T* y, T* x_out, const float* w, float eps, T* xn,
                       sg_block_q8k* xq, int n, int n_rows, void* stream, const char* nm) {
  if (!x || !w || (!xn && !xq) || (y && !x_out) || (!y && x_out))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: x, w and xn or xq are needed, x_out exactly when there is y", nm);
  if (n <= 0 || n % kQK != 0 || n_rows <= 0)
    return set_error(SG_ERR_GEOMETRY, "%s: n=%d must be a positive multiple of 256, n_rows=%d",
                     nm, n, n_rows);
  if (n > 64 * kQK || n_rows >= 1 << 22)  // (a launch has less than 2^32 threads)
    return set_error(SG_ERR_UNSUPPORTED, "%s: n=%d is over %d, or n_rows=%d over 2^22 - 1", nm, n,
                     64 * kQK, n_rows);
  if (reinterpret_cast<uintptr_t>(xq) % 4 || reinterpret_cast<uintptr_t>(x) % sizeof(T) ||
      reinterpret_cast<uintptr_t>(y) % sizeof(T) || reinterpret_cast<uintptr_t>(x_out) % sizeof(T) ||
      reinterpret_cast<uintptr_t>(xn) % sizeof(T) || reinterpret_cast<uintptr_t>(w) % 4)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: a buffer is not aligned to its elements", nm);
  // (a row's values are read before they are written, other rows' at any time)
  const long long all = static_cast<long long>(n_rows) * n;
  const long long q = all / kQK * kQ8Bytes;
  const unsigned char* const codes = reinterpret_cast<const unsigned char*>(xq);
  auto over = [&](const T* out, const T* in) { return out != in && overlap(out, all, in, all); };
  if (over(x_out, x) || over(x_out, y) || over(xn, x) || over(xn, y) ||
      overlap(xn, all, x_out, all) || overlap(x_out, all, w, n) || overlap(xn, all, w, n) ||
      overlap(codes, q, x, all) || overlap(codes, q, y, all) || overlap(codes, q, w, n) ||
      overlap(codes, q, x_out, all) || overlap(codes, q, xn, all))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: an output overlaps another buffer (x_out and xn may each be x or y, "
                     "not both the same)", nm);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int nb = n / kQK;
  // one block a wave as far as the waves go
  if (nb <= 4)
    norm_go<T, 4, 1>(x, y, x_out, w, eps, xn, xq, n, n_rows, s);
  else if (nb <= 8)
    norm_go<T, 8, 1>(x, y, x_out, w, eps, xn, xq, n, n_rows, s);
  else if (nb <= 16)
    norm_go<T, 16, 1>(x, y, x_out, w, eps, xn, xq, n, n_rows, s);
  else if (nb <= 32)
    norm_go<T, 16, 2>(x, y, x_out, w, eps, xn, xq, n, n_rows, s);
  else
    norm_go<T, 16, 4>(x, y, x_out, w, eps, xn, xq, n, n_rows, s);
  return check_launch(nm);
}

}  // namespace sg

extern "C" {

int sg_add_rmsnorm_q8_k(const float* x, const float* y, float* x_out, const float* w, float eps,
                        float* xn, sg_block_q8k* xq, int n, int n_rows, void* stream) {
  return sg::norm_launch<float>(x, y, x_out, w, eps, xn, xq, n, n_rows, stream,
                                "sg_add_rmsnorm_q8_k");
}

int sg_add_rmsnorm_q8_k_f16(const uint16_t* x, const uint16_t* y, uint16_t* x_out, const float* w,
                            float eps, uint16_t* xn, sg_block_q8k* xq, int n, int n_rows,
                            void* stream) {
  return sg::norm_launch<uint16_t>(x, y, x_out, w, eps, xn, xq, n, n_rows, stream,
                                   "sg_add_rmsnorm_q8_k_f16");
}

}  // extern "C"
