// sg_verify.hip - which drafted tokens of a window the target's
// probabilities accept, and the token after them, from given random numbers.
//
// The vocabulary is cut into chunks.  verify_rows_kernel reads every row of
// logits once and leaves per chunk the largest logit m_c and
// sum 2^((x - m_c) log2(e) / temperature) less the largest logit's own 1
// (greedy: where m_c lies), and per node what its tree says of it; verify_walk_kernel, one workgroup a
// sequence, joins the chunks of each row, goes down the tree and draws the
// last token: first its chunk, by the chunks' sums, then the token inside it,
// so that of the last row only one chunk is read again.  With the drafter's
// distributions, what a rejection leaves, max(R - q, 0), has to be summed over
// the vocabulary before the next sibling can be tried: verify_rest_kernel does
// it for all children of one rank of all nodes, as if their earlier siblings
// had been rejected.
//
// Weights and sums are fp64: the last token is found by comparing running
// sums, and with a vocabulary's worth of borders an fp32 sum would move one
// over the random number now and then.  The largest logit's weight stays apart
// from its chunk's and its row's sum, for it may be nearly all of them: what
// its rejection leaves is then no difference.
#include "sg_window.hpp"

namespace sg {

constexpr int kChunk = 4096;      // logits of a workgroup of verify_rows_kernel
constexpr int kWalk = 1024;       // threads of verify_walk_kernel, kChunk / 4
constexpr int kMaxChildren = 16;
constexpr double kRest = 0x1p-30; // a smaller share of the mass counts as none
// What other rejected tokens leave of a sum is found by subtraction down to this share of it: the
// sums' errors (2^-47) are then 2^-27 of what is left.
constexpr double kLittle = 0x1p-20;

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));

// log2(e) / t.  A subnormal temperature counts as the least normal one: the
// factor has to be an fp32 number too.
__device__ __forceinline__ double per_temperature(float t) {
  return 1.4426950408889634074 / static_cast<double>(fmaxf(t, 0x1p-126f));
}
__device__ __forceinline__ float no_nan(float x) { return x == x ? x : -INFINITY; }

// The weight 2^((x - m) c) of logit x under the row's (or chunk's) largest m,
// which is finite; c = log2(e) / temperature.  (x - m) c = n + f, |f| a little
// over 1/2, and 2^f = 1 + f g(f) with g of degree 10 through its Chebyshev
// nodes on +-0.502: with the roundings 2^-52.9 of the weight at most, and
// 2^-53 |(x - m) c| from the exponent.  All of fp64's bits, because what a
// rejection leaves is a difference of such sums: with g of degree 7 (2e-12) a
// third sibling's probability was off by 1.6e-5 where the first two had all
// but 1e-8 of the mass.  n comes from the same difference in fp32, where its
// rounding takes no fp64 operation (an fp64 operation takes about 10 cycles a
// wave: 64 rows of 248,320 logits 19.2 us, 17.5 with g of degree 7).  Exactly 1
// for x == m; 0 below 2^-1000 and for NaN and -infinity.
struct Scale {
  double c, m;
  float c32, m32;
};
__device__ __forceinline__ Scale scale_of(double c, float m) {
  return Scale{c, static_cast<double>(m), static_cast<float>(c), m};
}
// A constant in scalar registers: an operand of v_fma_f64 as it is, where a literal is first moved
// into two vector registers.
__device__ __forceinline__ double in_sgpr(double c) {
  asm("" : "+s"(c));
  return c;
}
__device__ __forceinline__ double weight_of(float x, const Scale& s) {
  const float y = (x - s.m32) * s.c32;
  const float n = __builtin_rintf(fmaxf(y, -1010.f));
  const double f = __builtin_fma(static_cast<double>(x) - s.m, s.c, -static_cast<double>(n));
  double g = in_sgpr(4.455036203781184e-10);
  g = __builtin_fma(g, f, in_sgpr(7.072727791672384e-09));
  g = __builtin_fma(g, f, in_sgpr(1.017806206630947e-07));
  g = __builtin_fma(g, f, in_sgpr(1.3215441875881882e-06));
  g = __builtin_fma(g, f, in_sgpr(1.525273383046128e-05));
  g = __builtin_fma(g, f, in_sgpr(0.00015403530442908896));
  g = __builtin_fma(g, f, in_sgpr(0.0013333558146416563));
  g = __builtin_fma(g, f, in_sgpr(0.009618129107606187));
  g = __builtin_fma(g, f, in_sgpr(0.0555041086648216));
  g = __builtin_fma(g, f, in_sgpr(0.240226506959101));
  g = __builtin_fma(g, f, in_sgpr(0.6931471805599453));
  g = __builtin_fma(g, f, 1.0);
  const uint64_t b = __builtin_bit_cast(uint64_t, g);
  const uint32_t hi = static_cast<uint32_t>(b >> 32) + (static_cast<uint32_t>(static_cast<int>(n)) << 20);
  const double r =
      __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | static_cast<uint32_t>(b));
  return y >= -1000.f ? r : 0.0;
}

// The same for any m but -infinity: equal logits get exactly 1, also where
// both are infinite.
__device__ __forceinline__ double weight(float x, float m, double c) {
  return x == m ? 1.0 : m == INFINITY ? 0.0 : weight_of(x, scale_of(c, m));
}

// What the tree says of a node.
struct Node {
  int up, rank;        // its parent (-1: the root, or absent), its place among the siblings
  uint64_t sib, same;  // its earlier siblings; those of them with its token
  float x, q;          // its token's logit at the parent, and draft probability
  int tok, pad;        // -1: no token of the vocabulary
};

struct VerifyArgs {
  const float* logits;
  const int *tokens, *win_off, *parent;
  const float *draft, *temperature, *u_accept, *u_sample;
  int *path, *n_path, *next;
  float* prob;
  Node* nodes;    // [token]
  double* csum;   // [token][chunk]: sum of weights less 1; greedy: index of the largest logit
  double* rest;   // [token][chunk]: sum of max(R - q, 0) once the node is rejected
  float* cmax;    // [token][chunk]
  int n_tokens, max_window, vocab, n_chunks, max_children;
};

// Sums over the wave (the same in every lane) and running sums, by DPP; a
// double goes in two halves.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWS, 0xF, false);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double readlane_d(double v, int l) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), l);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), l);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_run_sum(double v) {  // lane l: of lanes 0..l
  v += dpp_d<0x111>(v);  // row_shr 1, 2, 4, 8
  v += dpp_d<0x112>(v);
  v += dpp_d<0x114>(v);
  v += dpp_d<0x118>(v);
  v += dpp_d<0x142, 0xA>(v);  // row_bcast 15 into rows 1 and 3, 31 into 2 and 3
  v += dpp_d<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) { return readlane_d(wave_run_sum(v), 63); }

// Node `lane` of a window, for the calling wave.
__device__ __forceinline__ Node tree_node(const VerifyArgs& a, Window w, int lane) {
  Node n;
  const bool here = lane < w.n;
  const int tok = here ? a.tokens[w.off + lane] : -1;
  n.tok = tok >= 0 && tok < a.vocab ? tok : -1;
  int up = parent_of(a.parent, w, lane);
  n.sib = n.same = 0;
  for (int j = 1; j < w.n; ++j) {
    const int pj = __builtin_amdgcn_readlane(up, j), tj = __builtin_amdgcn_readlane(n.tok, j);
    const bool s = j < lane && pj == up && pj != j && up != lane;
    n.sib |= s ? 1ull << j : 0;
    n.same |= s && tj == n.tok ? 1ull << j : 0;
  }
  n.rank = __popcll(n.sib);
  if (a.draft && n.rank >= a.max_children) up = lane;
  n.up = masks_up(up, w.n, lane) != 0 && lane > 0 ? up : -1;
  const bool real = n.up >= 0 && n.tok >= 0;
  n.x = real ? no_nan(a.logits[static_cast<long long>(w.off + n.up) * a.vocab + n.tok]) : 0.f;
  n.q = real && a.draft ? a.draft[static_cast<long long>(w.off + lane) * a.vocab + n.tok] : 0.f;
  n.pad = 0;
  return n;
}

// Whether what lies at node i of a window can be its own: a window that shares
// rows with another one (win_off not ascending) may find the other's nodes
// there, or half of them.  Such a node counts as absent, so that every row that
// a node names is one of its window's.
__device__ __forceinline__ bool node_ok(const Node& n, int i) {
  return n.up >= 0 && n.up < i && n.sib >> i == 0 && n.rank == __popcll(n.sib);
}

// Grid: (chunk, node, sequence); the workgroup past the chunks of node 0
// does the tree.  64 rows of 248,320 take 19.7 us, 3.2 TB/s: 14 fp64 operations
// a logit, with memory close behind them; 4 rows 4.8 us, one round of loads.
// (When the 64 rows took 17 us, with weights of fewer bits: workgroups of
// several chunks, the next one's logits under way, 22; 512 threads of 8 logits
// 20.)
__global__ void __launch_bounds__(256) verify_rows_kernel(const VerifyArgs a) {
  const int s = blockIdx.z, node = blockIdx.y, c = blockIdx.x;
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  if (node >= w.n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (c == a.n_chunks) {
    if (node == 0 && wave == 0) {
      const Node n = tree_node(a, w, lane);
      if (lane < w.n) a.nodes[w.off + lane] = n;
    }
    return;
  }
  const long long row = w.off + node;
  const float* x = a.logits + row * a.vocab;
  constexpr int kLoads = kChunk / 1024;
  f32x4_u v[kLoads];
  const int v0 = c * kChunk + 4 * threadIdx.x;
  if ((c + 1) * kChunk <= a.vocab) {
#pragma unroll
    for (int h = 0; h < kLoads; ++h) v[h] = *reinterpret_cast<const f32x4_u*>(x + v0 + h * 1024);
  } else {
#pragma unroll
    for (int h = 0; h < kLoads; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = v0 + h * 1024 + i;
        v[h][i] = at < a.vocab ? x[at] : -INFINITY;
      }
  }
  const float t = a.temperature[s];
  const bool sampled = t > 0.f;
  const double k = sampled ? per_temperature(t) : 1.0;
  __shared__ float sm[4];
  __shared__ double ss[4];
  __shared__ int sn[4];  // whether the wave has one of the largest
  float m = -INFINITY;  // (fmaxf passes a NaN over)
#pragma unroll
  for (int h = 0; h < kLoads; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, v[h][i]);
  const float mine = m;
  m = wave_max_dpp(m);
  if (lane == 0) sm[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  double sum = 0.0;
  const uint64_t has = __ballot(mine == m);
  if (sampled) {
    if (has) {  // one of the largest stays apart from the wave's sum
      bool out = lane == __builtin_ctzll(has);
#pragma unroll
      for (int h = 0; h < kLoads; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool it = out && v[h][i] == m;
          v[h][i] = it ? -INFINITY : v[h][i];
          out = out && !it;
        }
    }
    if (m == INFINITY) {
#pragma unroll
      for (int h = 0; h < kLoads; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += v[h][i] == m ? 1.0 : 0.0;
    } else if (m > -INFINITY) {
      const Scale sc = scale_of(k, m);
#pragma unroll
      for (int h = 0; h < kLoads; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += weight_of(v[h][i], sc);
    }
    sum = wave_sum(sum);
  } else {  // the lowest index of the largest logit, as a number
    int at = a.vocab;
#pragma unroll
    for (int h = 0; h < kLoads; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) at = v[h][i] == m ? min(at, v0 + h * 1024 + i) : at;
    sum = static_cast<double>(-wave_max_i32(-at));
  }
  if (lane == 0) {
    ss[wave] = sum;
    sn[wave] = has != 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.cmax[row * a.n_chunks + c] = m;
    a.csum[row * a.n_chunks + c] =
        sampled ? ((ss[0] + ss[1]) + (ss[2] + ss[3])) + (sn[0] + sn[1] + sn[2] + sn[3] - 1)
                : fmin(fmin(ss[0], ss[1]), fmin(ss[2], ss[3]));
  }
}

// A row's largest logit, its sum of weights, and that less the largest logit's
// 1 (greedy: s is the lowest index of the largest logit; -1 if all are
// -infinity), by one wave.
struct RowStat {
  float m;
  double s, others;
};
// The first 128 chunks (half a million tokens), so that several rows' loads can be under way.
struct RowHead {
  float m[2];
  double s[2];
};
__device__ __forceinline__ RowHead row_head(const VerifyArgs& a, long long row, int lane) {
  RowHead h;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = lane + 64 * i;
    h.m[i] = c < a.n_chunks ? a.cmax[row * a.n_chunks + c] : -INFINITY;
    h.s[i] = c < a.n_chunks ? a.csum[row * a.n_chunks + c] : 0.0;
  }
  return h;
}
__device__ __forceinline__ RowStat row_stat(const VerifyArgs& a, long long row, const RowHead& h,
                                            bool sampled, double k, int lane) {
  const float* cm = a.cmax + row * a.n_chunks;
  const double* cs = a.csum + row * a.n_chunks;
  RowStat r;
  float m = fmaxf(h.m[0], h.m[1]);
  for (int c = lane + 128; c < a.n_chunks; c += 64) m = fmaxf(m, cm[c]);
  r.m = m = wave_max_dpp(m);
  r.others = 0.0;
  if (sampled) {
    // all chunks' sums, but of one that has the largest logit without its 1
    double s = 0.0;
    bool apart = false;
    auto add = [&](float mc, double sc) {
      const uint64_t has = __ballot(mc == m);
      const bool one = !apart && has && lane == __builtin_ctzll(has);
      apart |= has != 0;
      if (mc > -INFINITY) s += one ? sc : (sc + 1.0) * weight(mc, m, k);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) add(h.m[i], h.s[i]);
    for (int c0 = 128; c0 < a.n_chunks; c0 += 64) {
      const int c = min(c0 + lane, a.n_chunks - 1);
      add(c == c0 + lane ? cm[c] : -INFINITY, cs[c]);
    }
    r.others = wave_sum(s);
    r.s = m > -INFINITY ? r.others + 1.0 : 0.0;
  } else {
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 1; i >= 0; --i) at = h.m[i] == m && h.s[i] < at ? static_cast<int>(h.s[i]) : at;
    for (int c = lane + 128; c < a.n_chunks; c += 64)
      if (cm[c] == m && cs[c] < at) at = static_cast<int>(cs[c]);
    at = -wave_max_i32(-at);
    r.s = m > -INFINITY ? static_cast<double>(at) : -1.0;
  }
  return r;
}
// The sum of a node's rest, by one wave.
__device__ __forceinline__ double rest_sum(const VerifyArgs& a, long long row, int lane) {
  double s = 0.0;
  for (int c = lane; c < a.n_chunks; c += 64) s += a.rest[row * a.n_chunks + c];
  return wave_sum(s);
}
// The row's sum of weights without n tokens, this wave's part of it: the chunks' sums as they are, and
// a chunk with such a token weight by weight.
__device__ __forceinline__ double part_without(const VerifyArgs& a, long long row, float m,
                                               const int* toks, int n, double k) {
  const float* x = a.logits + row * a.vocab;
  double s = 0.0;
  for (int c = threadIdx.x; c < a.n_chunks; c += kWalk) {
    const float cm = a.cmax[row * a.n_chunks + c];
    bool has = false;
    for (int i = 0; i < n; ++i) has |= toks[i] / kChunk == c;
    if (!has && cm > -INFINITY) s += (a.csum[row * a.n_chunks + c] + 1.0) * weight(cm, m, k);
  }
  for (int i = 0; i < n; ++i) {
    const int c = toks[i] / kChunk;
    bool again = false;
    for (int j = 0; j < i; ++j) again |= toks[j] / kChunk == c;
    if (again) continue;
    const int v0 = c * kChunk + 4 * threadIdx.x;
    float xv[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) xv[h] = v0 + h < a.vocab ? no_nan(x[v0 + h]) : -INFINITY;
    for (int j = 0; j < n; ++j)
#pragma unroll
      for (int h = 0; h < 4; ++h) xv[h] = toks[j] == v0 + h ? -INFINITY : xv[h];
#pragma unroll
    for (int h = 0; h < 4; ++h) s += weight(xv[h], m, k);
  }
  return wave_sum(s);
}
// The target's probability of token v (logit x) in a row; inv: 1 / r.s.
__device__ __forceinline__ double target_p(RowStat r, double inv, float x, int v, bool sampled,
                                           double k) {
  if (!sampled) return static_cast<double>(v) == r.s ? 1.0 : 0.0;
  return r.m > -INFINITY ? weight(x, r.m, k) * inv : 0.0;
}

// The siblings of rank 0 .. n-1 below a node: rows, and one over the sums of
// their rests (0: less than kRest, which counts as none).
struct Chain {
  int row[kMaxChildren];
  double inv[kMaxChildren];
};
// R(v) after the rejection of the first n siblings, normalized by the last
// rest that counts.  r: the target's probability.
__device__ __forceinline__ double chain_rest(const VerifyArgs& a, const Chain& ch, int n, double r,
                                             int v) {
  for (int i = 0; i < n; ++i) {
    if (ch.inv[i] == 0.0) continue;
    const double q = a.draft[static_cast<long long>(ch.row[i]) * a.vocab + v];
    r = fmax(r - q, 0.0) * ch.inv[i];
  }
  return r;
}

// Grid: (chunk, node, sequence), for the children of rank `rank`; a workgroup
// takes every gridDim.x-th chunk.
// What its time goes into is one round after the other (the node, its row's
// chunks, the siblings' sums, the tokens), so the tokens are spread over 1024
// threads: 42 rows of 50,257 logits 6.2 us for the first children and 8 us for
// the second ones, 64 rows of 248,320 (three ranks, the other launches with
// them) 100 us, a chunk a workgroup; 256 threads of 16 tokens: 10, 14 and 123.
constexpr int kRestThreads = 1024;
__global__ void __launch_bounds__(kRestThreads, 8) verify_rest_kernel(const VerifyArgs a, int rank) {
  const int s = blockIdx.z, node = blockIdx.y;
  int c = blockIdx.x;
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  if (node >= w.n) return;
  const Node me = a.nodes[w.off + node];
  if (!node_ok(me, node) || me.rank != rank) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* x = a.logits + static_cast<long long>(w.off + me.up) * a.vocab;
  const float* q = a.draft + static_cast<long long>(w.off + node) * a.vocab;
  constexpr int kEach = kChunk / kRestThreads, kWaves = kRestThreads / 64;
  float xv[kEach], qv[kEach], next[kEach];
  auto load = [&](float (&o)[kEach], const float* from, float none) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int v = c * kChunk + i * kRestThreads + threadIdx.x;
      o[i] = v < a.vocab ? from[v] : none;
    }
  };
  auto sibling = [&](uint64_t b) {
    return a.draft + static_cast<long long>(w.off + __builtin_ctzll(b)) * a.vocab;
  };
  load(xv, x, -INFINITY);
  load(qv, q, 0.f);
  const float t = a.temperature[s];
  const bool sampled = t > 0.f;
  const double k = sampled ? per_temperature(t) : 1.0;
  __shared__ Chain ch;
  __shared__ RowStat rs;
  __shared__ double ss[kWaves];
  if (wave == 0) {
    const RowStat r =
        row_stat(a, w.off + me.up, row_head(a, w.off + me.up, lane), sampled, k, lane);
    if (lane == 0) rs = r;
  }
  if (rank > 0) {
    load(next, sibling(me.sib), 0.f);
    uint64_t b = me.sib;
    for (int i = 0; i < rank; ++i, b &= b - 1)
      if (i == kWaves - 1 - wave) {  // (the last wave first: wave 0 has the row)
        const int row = w.off + __builtin_ctzll(b);
        const double r = rest_sum(a, row, lane);
        if (lane == 0) {
          ch.row[i] = row;
          ch.inv[i] = r < kRest ? 0.0 : 1.0 / r;
        }
      }
  }
  __syncthreads();
  const RowStat st = rs;
  const double inv = 1.0 / st.s;
  while (true) {
    double p[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      p[i] = target_p(st, inv, xv[i], c * kChunk + i * kRestThreads + threadIdx.x, sampled, k);
    uint64_t b = me.sib;
    for (int j = 0; j < rank; ++j) {  // a sibling's row at a time, the next one's loads under way
      const double jnv = ch.inv[j];
      float o[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) o[i] = next[i];
      b &= b - 1;
      if (b) load(next, sibling(b), 0.f);
      if (jnv == 0.0) continue;
#pragma unroll
      for (int i = 0; i < kEach; ++i) p[i] = fmax(p[i] - static_cast<double>(o[i]), 0.0) * jnv;
    }
    double sum = 0.0;  // (past the vocabulary x is -infinity and q 0)
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += fmax(p[i] - static_cast<double>(qv[i]), 0.0);
    const int done = c;
    c += gridDim.x;
    const bool more = c < a.n_chunks;
    if (more) {
      load(xv, x, -INFINITY);
      load(qv, q, 0.f);
      if (rank > 0) load(next, sibling(me.sib), 0.f);
    }
    sum = wave_sum(sum);
    if (lane == 0) ss[wave] = sum;
    __syncthreads();
    if (wave == 0) {
      const double all = wave_sum(lane < kWaves ? ss[lane] : 0.0);
      if (lane == 0) a.rest[static_cast<long long>(w.off + node) * a.n_chunks + done] = all;
    }
    if (!more) return;
    __syncthreads();
  }
}

// One workgroup a sequence, 16 waves: rows shared out among them, then the tree
// in one, the end's chunk in each by itself, and that chunk's tokens over all
// threads.  8.5 us for a window of 4, 12 for one of 64: the dependent rounds
// (window; chunks and nodes; the end's chunks; its tokens).  (The chunk found
// by the workgroup, and the token with four barriers instead of one: 1.3 more.)
__global__ void __launch_bounds__(kWalk) verify_walk_kernel(const VerifyArgs a) {
  const int s = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  int* path = a.path + static_cast<long long>(s) * a.max_window;
  if (w.n == 0) {
    if (static_cast<int>(threadIdx.x) < a.max_window) path[threadIdx.x] = -1;
    if (threadIdx.x == 0) {
      a.n_path[s] = 0;
      a.next[s] = -1;
    }
    return;
  }
  __shared__ RowStat stat[kMaxWindow];
  __shared__ double left[kMaxWindow];   // a rejected node's rest; a point mass: 1 if its share is taken
  __shared__ double whole[kMaxWindow];  // of R at a node, point masses: a sum, less the shares
  __shared__ double taken[kMaxWindow];  // that were taken away since it was one
  __shared__ int kid_tok[kMaxWindow];   // the end's children whose share is taken
  __shared__ int s_end, s_kids;
  __shared__ double ws[kWalk / 64];
  // What all waves sum for the one that goes down the tree: a node's row (-1: no more) without tokens
  __shared__ int job, job_n, job_tok[kMaxWindow];
  __shared__ Chain chain;
  const float t = a.temperature[s];
  const float us = a.u_sample[s];
  const bool sampled = t > 0.f;
  const double k = sampled ? per_temperature(t) : 1.0;
  Node n;
  n.up = -1;
  n.rank = 0;
  n.sib = n.same = 0;
  n.x = n.q = 0.f;
  n.tok = -1;
  float u = 1.f;
  if (wave == 0 && lane < w.n) {
    n = a.nodes[w.off + lane];
    u = a.u_accept[w.off + lane];
  }
  constexpr int kRounds = kMaxWindow / (kWalk / 64);
  RowHead head[kRounds];
#pragma unroll
  for (int j = 0; j < kRounds; ++j)
    head[j] = row_head(a, w.off + min(wave + j * (kWalk / 64), w.n - 1), lane);
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    const int i = wave + j * (kWalk / 64);
    if (i < w.n) {
      const RowStat r = row_stat(a, w.off + i, head[j], sampled, k, lane);
      if (lane == 0) {
        stat[i] = r;
        whole[i] = r.m > -INFINITY ? 1.0 : 0.0;
        taken[i] = 0.0;
      }
    }
  }
  if (a.draft)  // (of nodes that are nobody's child, whatever lies there: it is not used)
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const int i = wave + j * (kWalk / 64);
      if (i < w.n) {
        const double rest = rest_sum(a, w.off + i, lane);
        if (lane == 0) left[i] = rest;
      }
    }
  __syncthreads();
  if (wave == 0) {
    const bool in = node_ok(n, lane) && (!a.draft || n.rank < a.max_children);
    const int up = in ? n.up : 0;
    // R of the node's token at its parent, R's mass there, the bar u has to stay under
    const double inv = 1.0 / stat[up].s;
    double r = in && n.tok >= 0 ? target_p(stat[up], inv, n.x, n.tok, sampled, k) : 0.0;
    double m = whole[up], q = 1.0;
    if (a.draft) {
      q = n.q;
      for (uint64_t b = in ? n.sib : 0; b; b &= b - 1) {
        const int j = __builtin_ctzll(b);
        if (left[j] < kRest) continue;
        const double qj = n.tok >= 0
                              ? a.draft[static_cast<long long>(w.off + j) * a.vocab + n.tok] : 0.0;
        r = fmax((m > 0.0 ? r / m : 0.0) - qj, 0.0);
        m = left[j];
      }
    } else {
      // A point mass: a rejected sibling takes its token's share away.  All
      // children of one rank at once.  The largest logit's leaves the others'
      // sum, another one a difference, down to kLittle; then what is left is
      // summed anew, if there are later siblings or it may be none.
      uint64_t gone = 0;  // the nodes whose share is taken
      const uint64_t largest = __ballot(in && sampled && n.tok >= 0 && n.x == stat[up].m);
      const double others = stat[up].others * inv;
      for (int j = 0; __any(in && n.rank >= j); ++j) {
        const bool now = in && n.rank == j;
        double all = 0.0, less = 0.0;
        bool little = false;
        if (now) {
          if (n.same & gone) r = 0.0;
          all = whole[up];
          less = taken[up];
          m = all - less;
          if ((largest >> lane & 1) && !(n.sib & gone & largest))
            all = others;
          else
            less += r;
          little = sampled && all - less < kLittle * all;
        }
        if (__any(little)) {
          uint64_t later = in ? n.sib : 0;
          for (int o = 1; o < 64; o <<= 1) later |= __shfl_xor(later, o);
          little = little && ((later >> lane & 1) || m < 0x1p-10 * whole[up]);
          for (uint64_t b = __ballot(little); b; b &= b - 1) {
            const int l = __builtin_ctzll(b);
            const uint64_t out = (__shfl(n.sib, l) & gone) | 1ull << l;
            const int at = __builtin_amdgcn_readlane(up, l);
            if (out >> lane & 1) job_tok[__popcll(out & ((1ull << lane) - 1))] = n.tok;
            if (lane == 0) {
              job = at;
              job_n = __popcll(out);
            }
            bar();
            const double part =
                part_without(a, w.off + at, stat[at].m, job_tok, __popcll(out), k);
            if (lane == 0) ws[0] = part;
            bar();
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < kWalk / 64; ++i) sum += ws[i];
            if (lane == l) {
              all = sum / stat[at].s;
              less = 0.0;
            }
          }
        }
        const bool take = now && all - less >= kRest * m;
        if (take) {
          whole[up] = all;
          taken[up] = less;
        }
        gone |= __ballot(take);
        wait_lds();
        asm volatile("" ::: "memory");  // (whole and taken are other lanes' next)
      }
      if (lane < w.n) left[lane] = gone >> lane & 1 ? 1.0 : 0.0;
      if (lane == 0) job = -1;
      bar();
    }
    const double bar = q * m;
    const bool ok = in && static_cast<double>(u) * bar < r;
    if (a.prob && lane < w.n)
      a.prob[w.off + lane] =
          lane == 0 ? 1.f : !in ? 0.f : r >= bar ? (r > 0.0 ? 1.f : 0.f)
                                                 : static_cast<float>(r / bar);
    // down the tree: the first accepted child of each node
    const uint64_t yes = __ballot(ok);
    int at = 0, np = 0, mine = -1;
    while (true) {
      if (lane == np) mine = at;
      ++np;
      const uint64_t kid = __ballot(in && up == at) & yes;
      if (!kid) break;
      at = __builtin_ctzll(kid);
    }
    if (lane < a.max_window) path[lane] = mine;
    const int most = a.draft ? a.max_children : kMaxWindow;
    const uint64_t kid = __ballot(in && up == at);
    const int place = __popcll(kid & ((1ull << lane) - 1));  // (the rank)
    if (in && up == at && place < most) {
      kid_tok[place] = left[lane] > 0.0 ? n.tok : -1;
      if (a.draft) {
        chain.row[place] = w.off + lane;
        chain.inv[place] = left[lane] < kRest ? 0.0 : 1.0 / left[lane];
      }
    }
    if (lane == 0) {
      s_end = at;
      s_kids = min(__popcll(kid), most);
      a.n_path[s] = np;
    }
  } else if (!a.draft) {
    while (true) {
      bar();
      const int at = job;
      if (at < 0) break;
      const double part = part_without(a, w.off + at, stat[at].m, job_tok, job_n, k);
      if (lane == 0) ws[wave] = part;
      bar();
    }
  }
  __syncthreads();

  // The last token: R at the end of the path, in units of the row's weights.
  const int end = s_end, nk = s_kids;
  const RowStat st = stat[end];
  if (!sampled || st.m == -INFINITY) {  // all the mass is on one token, rejections or not; or none
    if (threadIdx.x == 0) a.next[s] = st.m > -INFINITY ? static_cast<int>(st.s) : -1;
    return;
  }
  const long long row = w.off + end;
  const float* x = a.logits + row * a.vocab;
  int from = -1;  // the rejected child whose rest is what is left
  double unit = 0.0;
  if (a.draft)
    for (int i = 0; i < nk; ++i)
      if (chain.inv[i] != 0.0) {
        from = chain.row[i];
        unit = left[from - w.off];
      }
  // R of chunk c's tokens, four consecutive ones a thread; returns their sum
  auto tokens_of = [&](int c, double (&r)[4]) {
    const int v0 = c * kChunk + 4 * threadIdx.x;
    double sum = 0.0;
    float xv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = v0 + i < a.vocab ? no_nan(x[v0 + i]) : -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int v = v0 + i;
      if (from >= 0) {  // (the rest as it was summed: not normalized)
        r[i] = v < a.vocab
                   ? chain_rest(a, chain, nk, target_p(st, 1.0 / st.s, xv[i], v, true, k), v) * unit
                   : 0.0;
      } else {
        r[i] = weight(xv[i], st.m, k);
        if (!a.draft)
          for (int j = 0; j < nk; ++j)
            if (kid_tok[j] == v) r[i] = 0.0;
      }
      sum += r[i];
    }
    return sum;
  };
  // Its chunk: every wave by itself, with the same numbers.  64 chunks at a time, from the last ones
  // down to the first for the total, then up for the chunk.  (The row's sum less what is rejected
  // would be that total too, but for the difference's rounding.)
  int c_at = -1, c_last = 0;
  double before = 0.0, passed = 0.0, total = 0.0, goal = 0.0;
  const int blocks = (a.n_chunks + 63) / 64;
  for (int b = 1 - blocks; b < blocks && c_at < 0; ++b) {
    const int c0 = 64 * abs(b), c = c0 + lane;
    // v: the chunk's sum; gone: its rejected tokens' weights, but for the largest logit's, which is
    // left out of v
    double v = 0.0, gone = 0.0;
    bool struck = false;
    if (c < a.n_chunks) {
      if (from >= 0) {
        v = a.rest[static_cast<long long>(from) * a.n_chunks + c];
      } else {
        const float cm = a.cmax[row * a.n_chunks + c];
        const double cs = a.csum[row * a.n_chunks + c];
        bool largest = false;
        if (!a.draft)
          for (int i = 0; i < nk; ++i) {
            const int tok = kid_tok[i];
            if (tok < 0 || tok / kChunk != c) continue;
            bool again = false;
            for (int j = 0; j < i; ++j) again |= kid_tok[j] == tok;
            if (again) continue;
            struck = true;
            const float xt = no_nan(x[tok]);
            if (xt == cm && !largest)
              largest = true;
            else
              gone += weight(xt, st.m, k);
          }
        if (cm > -INFINITY) v = (cs + (largest ? 0.0 : 1.0)) * weight(cm, st.m, k);
      }
    }
    v -= gone;
    // Where little is left of a chunk, the difference is its sums' rounding, or below what a weight
    // can be: such a chunk is summed again without the rejected tokens, by all waves (they take the
    // same turns: their numbers are the same).  Its sum is then 0 exactly where no token of it has a
    // share.
    for (uint64_t little = __ballot(struck && (v < kLittle * gone || (v > 0.0 && v < 0x1p-900)));
         little; little &= little - 1) {
      const int at = __builtin_ctzll(little);
      double r[4];
      const double part = wave_sum(tokens_of(c0 + at, r));
      if (lane == 0) ws[wave] = part;
      __syncthreads();
      double all = 0.0;
#pragma unroll
      for (int i = 0; i < kWalk / 64; ++i) all += ws[i];
      if (lane == at) v = all;
      __syncthreads();
    }
    const double run = wave_run_sum(v);
    if (b <= 0) total += readlane_d(run, 63);
    if (b < 0) continue;
    goal = static_cast<double>(us) * total;
    const uint64_t hit = __ballot(v > 0.0 && passed + run > goal), some = __ballot(v > 0.0);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      c_at = c0 + at;
      before = readlane_d(passed + run - v, at);
    }
    if (some) c_last = c0 + 63 - __builtin_clzll(some);
    passed += readlane_d(run, 63);
  }
  const bool past = c_at < 0;  // u_sample is 1 or more, or the sums round so
  if (past) c_at = c_last;
  // the token in it
  const int v0 = c_at * kChunk + 4 * threadIdx.x;
  double r[4];
  const double sum = tokens_of(c_at, r);
  const double run = wave_run_sum(sum);
  if (lane == 63) ws[wave] = run;
  __syncthreads();
  // the wave whose sums pass the goal; the last one with any where none does (the sums round so)
  int who = -1;
  double base = before, all = before;
  bool found = false;
#pragma unroll
  for (int i = 0; i < kWalk / 64; ++i) {
    const double w_sum = ws[i];
    if (!found && w_sum > 0.0) {
      who = i;
      base = all;
      found = !past && all + w_sum > goal;
    }
    all += w_sum;
  }
  // (a chunk with a sum has a token with a share; windows that overlap, against the rules, may differ)
  if (who < 0 && threadIdx.x == 0) a.next[s] = -1;
  if (wave != who) return;
  // its lane, and the token there, likewise
  const uint64_t some = __ballot(sum > 0.0);
  const uint64_t hit = found ? __ballot(sum > 0.0 && base + run > goal) : 0;
  if (lane != (hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some))) return;
  int tok = -1;
  bool done = false;
  double b = base + run - sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    b += r[i];
    if (r[i] > 0.0 && !done) tok = v0 + i;
    done |= r[i] > 0.0 && hit && b > goal;
  }
  a.next[s] = tok;
}

static size_t up16(size_t n) { return (n + 15) / 16 * 16; }
struct VerifyWs {
  size_t nodes, csum, cmax, rest, bytes;
};
static VerifyWs verify_ws(int n_tokens, int vocab, int max_children) {
  const size_t t = n_tokens, c = (vocab + kChunk - 1) / kChunk;
  VerifyWs w;
  w.nodes = 0;
  w.csum = w.nodes + up16(t * sizeof(Node));
  w.cmax = w.csum + up16(t * c * sizeof(double));
  w.rest = w.cmax + up16(t * c * sizeof(float));
  w.bytes = w.rest + (max_children > 0 ? up16(t * c * sizeof(double)) : 0);
  return w;
}

}  // namespace sg

extern "C" {

size_t sg_tree_verify_workspace_bytes(int n_tokens, int vocab, int max_children) {
  if (n_tokens <= 0 || vocab <= 0) return 0;
  return sg::verify_ws(n_tokens, vocab, max_children).bytes;
}

int sg_tree_verify(const float* logits, const int* tokens, const int* win_off, const int* parent,
                   const float* draft_probs, const float* temperature, const float* u_accept,
                   const float* u_sample, int* path, int* n_path, int* next, float* prob, void* ws,
                   size_t ws_bytes, int n_seq, int n_tokens, int max_window, int vocab,
                   int max_children, void* stream) {
  const char* nm = "sg_tree_verify";
  using namespace sg;
  if (!logits || !tokens || !win_off || !temperature || !u_accept || !u_sample || !path || !n_path ||
      !next || !ws)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (n_seq <= 0 || n_tokens <= 0 || max_window <= 0 || vocab <= 0 ||
      (draft_probs && max_children <= 0))
    return set_error(SG_ERR_GEOMETRY,
                     "%s: n_seq=%d n_tokens=%d max_window=%d vocab=%d max_children=%d", nm, n_seq,
                     n_tokens, max_window, vocab, max_children);
  if (max_window > kMaxWindow || vocab > 1 << 24 || n_seq > 65535 ||
      (draft_probs && max_children > kMaxChildren))
    return set_error(SG_ERR_UNSUPPORTED,
                     "%s: at most a window of %d, a vocabulary of 2^24, 65535 sequences, %d "
                     "children",
                     nm, kMaxWindow, kMaxChildren);
  const VerifyWs l = verify_ws(n_tokens, vocab, draft_probs ? max_children : 0);
  if (ws_bytes < l.bytes || reinterpret_cast<uintptr_t>(ws) % 16)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: the workspace needs %zu bytes, 16-B aligned", nm,
                     l.bytes);
  // (a sequence's results are written while others' are found)
  const long long full = static_cast<long long>(n_tokens) * vocab;
  auto clear = [&](const auto* out, long long n) {
    return !(overlap(out, n, logits, full) || overlap(out, n, tokens, n_tokens) ||
             overlap(out, n, win_off, n_seq + 1LL) || overlap(out, n, parent, n_tokens) ||
             overlap(out, n, draft_probs, full) || overlap(out, n, temperature, n_seq) ||
             overlap(out, n, u_accept, n_tokens) || overlap(out, n, u_sample, n_seq) ||
             overlap(out, n, static_cast<unsigned char*>(ws), static_cast<long long>(l.bytes)));
  };
  const long long paths = static_cast<long long>(n_seq) * max_window;
  if (!clear(path, paths) || !clear(n_path, n_seq) || !clear(next, n_seq) || !clear(prob, n_tokens) ||
      overlap(path, paths, n_path, n_seq) || overlap(path, paths, next, n_seq) ||
      overlap(path, paths, prob, n_tokens) || overlap(n_path, n_seq, next, n_seq) ||
      overlap(n_path, n_seq, prob, n_tokens) || overlap(next, n_seq, prob, n_tokens))
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: an output overlaps another buffer", nm);
  VerifyArgs a;
  a.logits = logits;
  a.tokens = tokens;
  a.win_off = win_off;
  a.parent = parent;
  a.draft = draft_probs;
  a.temperature = temperature;
  a.u_accept = u_accept;
  a.u_sample = u_sample;
  a.path = path;
  a.n_path = n_path;
  a.next = next;
  a.prob = prob;
  unsigned char* b = static_cast<unsigned char*>(ws);
  a.nodes = reinterpret_cast<Node*>(b + l.nodes);
  a.cmax = reinterpret_cast<float*>(b + l.cmax);
  a.csum = reinterpret_cast<double*>(b + l.csum);
  a.rest = reinterpret_cast<double*>(b + l.rest);
  a.n_tokens = n_tokens;
  a.max_window = max_window;
  a.vocab = vocab;
  a.n_chunks = (vocab + kChunk - 1) / kChunk;
  a.max_children = max_children;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // Two chunks a workgroup where there are several rounds of workgroups: what it
  // finds out before its first logit then serves both (64 rows of 248,320 with
  // three children a node 96 us, 100 with one chunk, 98 with four; five rows of
  // 128,256 25 with one, 29 with two).
  const long long chunks = static_cast<long long>(a.n_chunks) * max_window * n_seq;
  const int per = chunks >= 2048 ? 2 : 1;
  const dim3 grid((a.n_chunks + per - 1) / per, max_window, n_seq);
  hipLaunchKernelGGL(verify_rows_kernel, dim3(a.n_chunks + 1, max_window, n_seq), dim3(256), 0, s, a);
  if (int st = check_launch(nm)) return st;
  if (draft_probs)
    for (int r = 0; r < max_children && r < max_window - 1; ++r) {
      hipLaunchKernelGGL(verify_rest_kernel, grid, dim3(kRestThreads), 0, s, a, r);
      if (int st = check_launch(nm)) return st;
    }
  hipLaunchKernelGGL(verify_walk_kernel, dim3(n_seq), dim3(kWalk), 0, s, a);
  return check_launch(nm);
}

}  // extern "C"
