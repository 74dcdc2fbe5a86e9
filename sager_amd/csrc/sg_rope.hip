// sg_rope.hip - the heads' RMS norms and the rotary positions of q and k, in
// one launch: what lies between a layer's projections and its attention.
//
//   y = (x / sqrt(mean(x^2) + eps)) * w         (where the head has a norm)
//   (a, b) -> (a c - b s, b c + a s),  c, s = mscale * cos, sin(2 pi turns_i pos)
//
// over the pairs i of the head's first rot_dim values: (i, i + rot_dim / 2) or
// (2 i, 2 i + 1).  The reference's norm and rotary launches are
// norm_rotary.cu's (rmsnorm and RoPE there are separate).
//
// The angle: a position of 2^19 times a frequency near 1 is rounded by 0.03
// radians in 32 bits.  The table therefore holds turns a position in fp64; the
// product's whole turns are taken off in fp64, and what is left, within half a
// turn, is exact enough in fp32 (2^-25 of a turn) for fp32's sine and cosine:
// outputs of fp32 are 6e-8 of their size off, 4.5e-8 with both in fp64, those of
// fp16 no more than with fp64.
// Sums of squares and all between the load and the store are fp32; the result
// is rounded once.
//
// A workgroup a token, or a part of a token's heads: its first threads make the token's sines and cosines,
// once for all its heads, while the first heads' values are already on their way
// into registers (eight consecutive ones a lane).  The half layout's partners come
// through LDS, within the wave.
#include <algorithm>
#include <cmath>

#include "sg_window.hpp"

namespace sg {

constexpr int kRopeDim = 512;      // largest head
// (4,096 tokens of 40 heads of 128: 22.3 us with 128 threads, 23.1 with 256,
// 28.8 with 512; with three rows of values a thread 25.5)
constexpr int kRopeThreads = 128;
constexpr int kRopeGroups = 1024;  // workgroups that a call of few tokens has at the most

struct RopeArgs {
  const void *q, *k;
  void *q_out, *k_out;
  long long q_stride, k_stride, qo_stride, ko_stride;
  const float *q_norm, *k_norm;
  const double* turns;
  const int *positions, *win_off, *parent, *length;
  int n_tokens, n_seq, n_heads, n_rows, dim, half, lanes_log2;
  bool pairs;  // neighbours
  float eps, mscale;
};

typedef uint32_t rope_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float rope_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float lds_f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void rope_load(const uint16_t* p, float (&v)[8]) {
  const rope_u4 w = *reinterpret_cast<const rope_u4*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = half_bits_to_float(w[i / 2] >> (16 * (i & 1)) & 0xFFFFu);
}
__device__ __forceinline__ void rope_load(const float* p, float (&v)[8]) {
  const rope_f4 a = *reinterpret_cast<const rope_f4*>(p);
  const rope_f4 b = *reinterpret_cast<const rope_f4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}
__device__ __forceinline__ void rope_store(uint16_t* p, const float (&v)[8]) {
  rope_u4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = f16b(v[2 * i]) | static_cast<uint32_t>(f16b(v[2 * i + 1])) << 16;
  *reinterpret_cast<rope_u4*>(p) = w;
}
__device__ __forceinline__ void rope_store(float* p, const float (&v)[8]) {
  *reinterpret_cast<rope_f4*>(p) = (rope_f4){v[0], v[1], v[2], v[3]};
  *reinterpret_cast<rope_f4*>(p + 4) = (rope_f4){v[4], v[5], v[6], v[7]};
}

// The position of row t; false if the row is in no window, or absent from its tree.
__device__ __forceinline__ bool position_of(const RopeArgs& a, int t, int lane, int* pos) {
  if (a.positions) {
    *pos = a.positions[t];
    return true;
  }
  const int s = seq_of_row(a.win_off, a.n_seq, t, lane);
  const int off = a.win_off[s], node = t - off;
  if (node < 0 || off < 0 || t >= a.win_off[s + 1]) return false;
  const int len = a.length[s];
  if (!a.parent) {
    *pos = len + node;
    return true;
  }
  if (node >= kMaxWindow) return false;
  const Window w = window_of(a.win_off, s, a.n_tokens, kMaxWindow);
  const uint64_t up = __shfl(ancestors(a.parent, w, lane), node);
  *pos = len + __popcll(up) - 1;
  return up != 0;
}

// Grid: (tokens, parts of a token's rows).  Rows of a token: its q heads, then
// its k heads.  Bound by vector instructions for many tokens (4,096 of 40 heads of
// 128: 84 MB in 22 us, 3.8 TB/s; some 250 a round of eight values a lane, 40 of the
// 54 thousand cycles), by the chain of loads before the first angle for few.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[2][kRopeDim / 2];
  __shared__ __attribute__((aligned(16))) float part[kRopeThreads / 64][64 * 8];
  __shared__ int there;
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lanes = 1 << a.lanes_log2;
  const int e = (tid & (lanes - 1)) * 8;       // the thread's values of a row
  const int per = blockDim.x >> a.lanes_log2;  // rows at a time
  const int rot = 2 * a.half;
  float* const mine = part[wave] + (lane & ~(lanes - 1)) * 8;  // the row's values

  auto at = [&](int r, const T** in, T** out) {  // row r's values from e on
    const bool is_q = r < a.n_heads;
    const int h = is_q ? r : r - a.n_heads;
    *in = static_cast<const T*>(is_q ? a.q : a.k) + t * (is_q ? a.q_stride : a.k_stride) +
          h * a.dim + e;
    *out = static_cast<T*>(is_q ? a.q_out : a.k_out) + t * (is_q ? a.qo_stride : a.ko_stride) +
           h * a.dim + e;
  };
  float v[8];
  auto load = [&](int r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (r < a.n_rows && e < a.dim) {
      const T* in;
      T* out;
      at(r, &in, &out);
      rope_load(in, v);
    }
  };
  const int first = blockIdx.y * per, turn_rows = gridDim.y * per;
  load(first + (tid >> a.lanes_log2));
  if (wave == 0) {
    int pos = 0;
    const bool ok = position_of(a, t, lane, &pos);
    if (lane == 0) there = ok;
    for (int i = lane; i < a.half; i += 64) {
      const double turn = static_cast<double>(pos) * a.turns[i];
      const float x = static_cast<float>(2. * (turn - rint(turn)));  // half turns
      float s, c;
      sincospif(x, &s, &c);
      cs[0][i] = c * a.mscale;
      cs[1][i] = s * a.mscale;
    }
  }
  __syncthreads();
  if (!there) return;

  for (int r0 = first; r0 < a.n_rows; r0 += turn_rows) {
    const int r = r0 + (tid >> a.lanes_log2);
    if (r0 > first) load(r);
    const bool some = r < a.n_rows && e < a.dim;
    const float* const w = r < a.n_heads ? a.q_norm : a.k_norm;
    if (a.q_norm || a.k_norm) {  // (the sum over a row's lanes: all of them take part)
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
      for (int m = 1; m < lanes; m <<= 1) ss += __shfl_xor(ss, m);
      if (some && w) {
        const float s = 1.f / sqrtf(ss / static_cast<float>(a.dim) + a.eps);
        float wv[8];
        rope_load(w + e, wv);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (v[i] * s) * wv[i];
      }
    }
    float y[8];
    if (a.pairs) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = min(e / 2 + i, kRopeDim / 2 - 1);
        const float c = cs[0][p], s = cs[1][p], x0 = v[2 * i], x1 = v[2 * i + 1];
        const bool in = e + 2 * i < rot;
        y[2 * i] = in ? x0 * c - x1 * s : x0;
        y[2 * i + 1] = in ? x1 * c + x0 * s : x1;
      }
    } else {
      // the partners by way of LDS; a wave's own rows, so no barrier
      *reinterpret_cast<lds_f4*>(mine + e) = (lds_f4){v[0], v[1], v[2], v[3]};
      *reinterpret_cast<lds_f4*>(mine + e + 4) = (lds_f4){v[4], v[5], v[6], v[7]};
      wait_lds();
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        // four values in one half of the pairs, their partners in line: 16-B reads
        const int x = e + j, to = x < a.half ? x + a.half : x - a.half;
        if (a.half % 4 == 0) {
          if (x < rot) {
            const int p = x < a.half ? x : x - a.half;
            const lds_f4 o = *reinterpret_cast<const lds_f4*>(mine + to);
            const lds_f4 c = *reinterpret_cast<const lds_f4*>(cs[0] + p);
            const lds_f4 s = *reinterpret_cast<const lds_f4*>(cs[1] + p);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              y[j + i] = x < a.half ? v[j + i] * c[i] - o[i] * s[i]
                                    : v[j + i] * c[i] + o[i] * s[i];
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[j + i] = v[j + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int xi = x + i;
            const bool low = xi < a.half;
            y[j + i] = v[j + i];
            if (xi < rot) {
              const int p = low ? xi : xi - a.half;
              const float o = mine[low ? xi + a.half : p], c = cs[0][p], s = cs[1][p];
              y[j + i] = low ? y[j + i] * c - o * s : y[j + i] * c + o * s;
            }
          }
        }
      }
      wait_lds();  // (read before the next row is written)
    }
    if (some) {
      const T* in;
      T* out;
      at(r, &in, &out);
      rope_store(out, y);
    }
  }
}

// Whether rows of wa values from a on, sa apart, and of wb from b, sb apart, n of each, share
// memory.  Of one stride: row i of one and row j of the other lie (b - a) + (j - i) s apart, and
// only the two differences j - i next to (a - b) / s come near; else their whole extents count.
template <typename T>
static bool rows_overlap(const T* a, long long wa, long long sa, const T* b, long long wb,
                         long long sb, long long n) {
  if (!a || !b || n <= 0 || wa <= 0 || wb <= 0) return false;
  if (!overlap(a, (n - 1) * sa + wa, b, (n - 1) * sb + wb)) return false;
  if (sa != sb) return true;
  const long long s = sa * static_cast<long long>(sizeof(T));
  const long long d = static_cast<long long>(reinterpret_cast<uintptr_t>(b)) -
                      static_cast<long long>(reinterpret_cast<uintptr_t>(a));
  const long long m0 = -d / s;
  for (long long m = m0 - 1; m <= m0 + 1; ++m) {
    const long long x = d + m * s;
    if (m > -n && m < n && x < wa * static_cast<long long>(sizeof(T)) &&
        -x < wb * static_cast<long long>(sizeof(T)))
      return true;
  }
  return false;
}

template <typename T>
static int rope_launch(const T* q, const T* k, T* q_out, T* k_out, long long q_stride,
                       long long k_stride, long long qo_stride, long long ko_stride,
                       const float* q_norm, const float* k_norm, float eps, const double* turns,
                       float mscale, const int* positions, const int* win_off, const int* parent,
                       const int* length, int n_tokens, int n_seq, int n_heads, int n_kv_heads,
                       int head_dim, int rot_dim, int neighbours, void* stream, const char* nm) {
  if (!q || !q_out || !turns || (n_kv_heads > 0 && (!k || !k_out)) ||
      (!positions && (!win_off || !length)))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: q, its output, the table and positions or windows are needed, k and its "
                     "output where n_kv_heads is not 0", nm);
  if (n_tokens <= 0 || n_heads <= 0 || n_kv_heads < 0 || (!positions && n_seq <= 0) ||
      head_dim <= 0 || head_dim % 8 != 0 || rot_dim <= 0 || rot_dim % 2 != 0 || rot_dim > head_dim)
    return set_error(SG_ERR_GEOMETRY,
                     "%s: n_tokens=%d n_seq=%d n_heads=%d n_kv_heads=%d, head_dim=%d must be a "
                     "multiple of 8, rot_dim=%d even and no more",
                     nm, n_tokens, n_seq, n_heads, n_kv_heads, head_dim, rot_dim);
  if (head_dim > kRopeDim || n_tokens >= 1 << 24 || n_heads > 1 << 20 || n_kv_heads > 1 << 20)
    return set_error(SG_ERR_UNSUPPORTED, "%s: head_dim=%d is over %d, or n_tokens=%d over 2^24 - 1",
                     nm, head_dim, kRopeDim, n_tokens);
  const long long qw = static_cast<long long>(n_heads) * head_dim;
  const long long kw = static_cast<long long>(n_kv_heads) * head_dim;
  if (q_stride < qw || qo_stride < qw || (kw > 0 && (k_stride < kw || ko_stride < kw)))
    return set_error(SG_ERR_GEOMETRY, "%s: a token stride is less than a token", nm);
  auto odd = [](const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; };
  if (odd(q, sizeof(T)) || odd(k, sizeof(T)) || odd(q_out, sizeof(T)) || odd(k_out, sizeof(T)) ||
      odd(q_norm, 4) || odd(k_norm, 4) || odd(turns, 8))
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: a buffer is not aligned to its elements", nm);
  if (kw == 0) k = nullptr, k_out = nullptr;
  // (a row is read before it is written, other rows at any time)
  const bool q_same = q == q_out && (q_stride == qo_stride || n_tokens == 1);
  const bool k_same = k == k_out && (k_stride == ko_stride || n_tokens == 1);
  if ((!q_same && rows_overlap<T>(q, qw, q_stride, q_out, qw, qo_stride, n_tokens)) ||
      (!k_same && rows_overlap<T>(k, kw, k_stride, k_out, kw, ko_stride, n_tokens)) ||
      rows_overlap<T>(q, qw, q_stride, k_out, kw, ko_stride, n_tokens) ||
      rows_overlap<T>(k, kw, k_stride, q_out, qw, qo_stride, n_tokens) ||
      rows_overlap<T>(q_out, qw, qo_stride, k_out, kw, ko_stride, n_tokens))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: an output overlaps q, k or the other output (each may be its own input)",
                     nm);
  const T* const outs[2] = {q_out, k_out};
  const long long sizes[2] = {(n_tokens - 1) * qo_stride + qw, (n_tokens - 1) * ko_stride + kw};
  for (int i = 0; i < 2; ++i)
    if (overlap(outs[i], sizes[i], q_norm, head_dim) || overlap(outs[i], sizes[i], k_norm, head_dim) ||
        overlap(outs[i], sizes[i], turns, rot_dim / 2) ||
        overlap(outs[i], sizes[i], positions, n_tokens) ||
        (!positions && (overlap(outs[i], sizes[i], win_off, n_seq + 1LL) ||
                        overlap(outs[i], sizes[i], parent, n_tokens) ||
                        overlap(outs[i], sizes[i], length, n_seq))))
      return set_error(SG_ERR_INVALID_ARGUMENT,
                       "%s: an output overlaps the norms, the table, the positions or the windows",
                       nm);
  RopeArgs a;
  a.q = q;
  a.k = k;
  a.q_out = q_out;
  a.k_out = k_out;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.qo_stride = qo_stride;
  a.ko_stride = ko_stride;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.turns = turns;
  a.positions = positions;
  a.win_off = win_off;
  a.parent = parent;
  a.length = length;
  a.n_tokens = n_tokens;
  a.n_seq = n_seq;
  a.n_heads = n_heads;
  a.n_rows = n_heads + n_kv_heads;
  a.dim = head_dim;
  a.half = rot_dim / 2;
  a.lanes_log2 = 0;
  while (8 << a.lanes_log2 < head_dim) ++a.lanes_log2;
  a.pairs = neighbours != 0;
  a.eps = eps;
  a.mscale = mscale;
  // Few tokens' heads are spread over workgroups that each make the angles
  // (4 tokens of 18 heads of 256: 4.7 us on the device, 8.5 by one a token).
  // A wave does for a token of few values (50,140 tokens of two heads of 64: 32 us,
  // two waves 47).
  const int threads = a.n_rows << a.lanes_log2 <= 64 ? 64 : kRopeThreads;
  const int per = threads >> a.lanes_log2;
  const int split = std::min((a.n_rows + per - 1) / per, std::max(1, kRopeGroups / n_tokens));
  hipLaunchKernelGGL(rope_kernel<T>, dim3(n_tokens, split), dim3(threads), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch(nm);
}

}  // namespace sg

extern "C" {

int sg_rope(const float* q, const float* k, float* q_out, float* k_out, long long q_stride,
            long long k_stride, long long qo_stride, long long ko_stride, const float* q_norm,
            const float* k_norm, float eps, const double* turns, float mscale,
            const int* positions, const int* win_off, const int* parent, const int* length,
            int n_tokens, int n_seq, int n_heads, int n_kv_heads, int head_dim, int rot_dim,
            int neighbours, void* stream) {
  return sg::rope_launch<float>(q, k, q_out, k_out, q_stride, k_stride, qo_stride, ko_stride,
                                q_norm, k_norm, eps, turns, mscale, positions, win_off, parent,
                                length, n_tokens, n_seq, n_heads, n_kv_heads, head_dim, rot_dim,
                                neighbours, stream, "sg_rope");
}

int sg_rope_f16(const uint16_t* q, const uint16_t* k, uint16_t* q_out, uint16_t* k_out,
                long long q_stride, long long k_stride, long long qo_stride, long long ko_stride,
                const float* q_norm, const float* k_norm, float eps, const double* turns,
                float mscale, const int* positions, const int* win_off, const int* parent,
                const int* length, int n_tokens, int n_seq, int n_heads, int n_kv_heads,
                int head_dim, int rot_dim, int neighbours, void* stream) {
  return sg::rope_launch<uint16_t>(q, k, q_out, k_out, q_stride, k_stride, qo_stride, ko_stride,
                                   q_norm, k_norm, eps, turns, mscale, positions, win_off, parent,
                                   length, n_tokens, n_seq, n_heads, n_kv_heads, head_dim, rot_dim,
                                   neighbours, stream, "sg_rope_f16");
}

int sg_rope_turns(double* turns, int rot_dim, double base, int scaling, double factor,
                  double trained, double slow, double fast) {
  const char* nm = "sg_rope_turns";
  using namespace sg;
  if (!turns) return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (rot_dim <= 0 || rot_dim % 2 != 0)
    return set_error(SG_ERR_GEOMETRY, "%s: rot_dim=%d must be even and positive", nm, rot_dim);
  if (scaling < SG_ROPE_PLAIN || scaling > SG_ROPE_BY_TURNS)
    return set_error(SG_ERR_UNSUPPORTED, "%s: scaling=%d", nm, scaling);
  const bool ramped = scaling == SG_ROPE_BY_INDEX || scaling == SG_ROPE_BY_TURNS;
  if (!(base > 1.) || !std::isfinite(base) ||
      (scaling != SG_ROPE_PLAIN && (!(factor > 0.) || !std::isfinite(factor))) ||
      (ramped && (!(trained > 0.) || !std::isfinite(trained) || !(slow > 0.) || !(fast > slow) ||
                  !std::isfinite(fast))))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: base must be over 1, factor and trained positive, 0 < slow < fast", nm);
  const double turn = 2 * M_PI;
  // the pair that turns so many times in a trained context
  auto pair = [&](double turns_there) {
    return rot_dim * std::log(trained / (turns_there * turn)) / (2 * std::log(base));
  };
  double lo = 0, hi = 0;
  if (scaling == SG_ROPE_BY_INDEX) {
    lo = std::max(std::floor(pair(fast)), 0.);
    hi = std::min(std::ceil(pair(slow)), rot_dim - 1.);
  }
  for (int i = 0; i < rot_dim / 2; ++i) {
    const double f = std::pow(base, -2. * i / rot_dim) / turn;
    double share = 0;  // of the stretched frequency
    if (scaling == SG_ROPE_LINEAR) share = 1;
    if (scaling == SG_ROPE_BY_INDEX)
      share = std::min(std::max((i - lo) / std::max(hi - lo, 0.001), 0.), 1.);
    if (scaling == SG_ROPE_BY_TURNS)
      share = 1 - std::min(std::max((trained * f - slow) / (fast - slow), 0.), 1.);
    turns[i] = share == 0 ? f : f / factor * share + f * (1 - share);
  }
  return SG_OK;
}

}  // extern "C"
