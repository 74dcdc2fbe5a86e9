// sg_verify.hip - which drafted tokens of a window the target's
// probabilities accept, and the token after them, from given random numbers.
//
// The vocabulary is cut into chunks.  verify_rows_kernel reads every row of
// logits once and leaves per chunk the largest logit m_c and
// sum exp((x - m_c) / temperature) (greedy: where m_c lies);
// verify_walk_kernel, one workgroup a sequence, joins the chunks of each row,
// goes down the tree and draws the last token: first its chunk, by the
// chunks' sums, then the token inside it, so that of the last row only one
// chunk is read again.  With the drafter's distributions, what a rejection
// leaves, max(R - q, 0), has to be summed over the vocabulary before the next
// sibling can be tried: verify_rest_kernel does it for all children of one
// rank of all nodes, as if their earlier siblings had been rejected.
//
// Weights and sums are fp64: the last token is found by comparing running
// sums, and with a vocabulary's worth of borders an fp32 sum would move one
// over the random number now and then.
#include "sg_window.hpp"

namespace sg {

constexpr int kChunk = 2048;      // logits of a workgroup of verify_rows_kernel
constexpr int kWalk = 1024;       // threads of verify_walk_kernel
constexpr int kMaxChildren = 16;
constexpr double kRest = 0x1p-30; // a smaller share of the mass counts as none

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));

// e^x for x <= 0, relative error below 1e-12: x = k ln2 + r, |r| <= ln2/2,
// e^r by its Taylor series to degree 11 (remainder below 7e-15).
__device__ __forceinline__ double exp_neg(double x) {
  const double k = __builtin_rint(x * 1.4426950408889634074);
  double r = __builtin_fma(k, -6.93147180369123816490e-01, x);
  r = __builtin_fma(k, -1.90821492927058770002e-10, r);
  double p = 1.0 / 39916800;
  p = __builtin_fma(p, r, 1.0 / 3628800);
  p = __builtin_fma(p, r, 1.0 / 362880);
  p = __builtin_fma(p, r, 1.0 / 40320);
  p = __builtin_fma(p, r, 1.0 / 5040);
  p = __builtin_fma(p, r, 1.0 / 720);
  p = __builtin_fma(p, r, 1.0 / 120);
  p = __builtin_fma(p, r, 1.0 / 24);
  p = __builtin_fma(p, r, 1.0 / 6);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return x < -700.0 ? 0.0 : __builtin_ldexp(p, static_cast<int>(k));
}

__device__ __forceinline__ float no_nan(float x) { return x == x ? x : -INFINITY; }

// The weight of logit x under the row's (or chunk's) largest m, which is not
// -infinity: equal logits get 1 even where both are infinite.
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  const double d = static_cast<double>(x) - static_cast<double>(m);
  return x == m ? 1.0 : d == -INFINITY ? 0.0 : exp_neg(d * inv_t);  // (0: at any temperature)
}

struct VerifyArgs {
  const float* logits;
  const int *tokens, *win_off, *parent;
  const float *draft, *temperature, *u_accept, *u_sample;
  int *path, *n_path, *next;
  float* prob;
  int2* tree;     // [token]: parent node that counts (-1: none), rank among its siblings
  float* cmax;    // [token][chunk]
  double* csum;   // [token][chunk]: sum of weights; greedy: index of the largest logit
  double* rest;   // [token][chunk]: sum of max(R - q, 0) once the node is rejected
  int n_tokens, max_window, vocab, n_chunks, max_children;
};

// The windows' trees, with draft distributions without the children past
// max_children.  One wave; node `lane`.
__device__ __forceinline__ int2 tree_node(const VerifyArgs& a, Window w, int lane) {
  int up = parent_of(a.parent, w, lane);
  int rank = 0;
  for (int j = 1; j < w.n; ++j) {
    const int pj = __shfl(up, j);
    rank += j < lane && pj == up && pj != j && up != lane;
  }
  if (a.draft && rank >= a.max_children) up = lane;
  const bool in = masks_up(up, w.n, lane) != 0;
  return make_int2(in && lane > 0 ? up : -1, rank);
}

// Grid: (chunk, node, sequence).
__global__ void __launch_bounds__(256) verify_rows_kernel(const VerifyArgs a) {
  const int s = blockIdx.z, node = blockIdx.y, c = blockIdx.x;
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  if (node >= w.n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long row = w.off + node;
  const float* x = a.logits + row * a.vocab;
  const int v0 = c * kChunk + 4 * threadIdx.x;
  float v[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = v0 + h * (kChunk / 2);
    if (at + 4 <= a.vocab) {
      const f32x4_u q = *reinterpret_cast<const f32x4_u*>(x + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = no_nan(q[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = at + i < a.vocab ? no_nan(x[at + i]) : -INFINITY;
    }
  }
  const float t = a.temperature[s];
  if (c == 0 && node == 0 && wave == 3) {
    const int2 tn = tree_node(a, w, lane);
    if (lane < w.n) a.tree[w.off + lane] = tn;
  }
  float m = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, v[i]);
  m = wave_max_dpp(m);
  __shared__ float sm[4];
  __shared__ double ss[4];
  if (lane == 0) sm[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const bool sampled = t > 0.f;
  double sum = 0.0;
  if (sampled) {
    const double inv_t = 1.0 / static_cast<double>(t);
    if (m > -INFINITY)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += weight(v[i], m, inv_t);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  } else {  // the lowest index of the largest logit, as a number
    sum = static_cast<double>(a.vocab);
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (v[i] == m) sum = fmin(sum, static_cast<double>(v0 + (i >> 2) * (kChunk / 2) + (i & 3)));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum = fmin(sum, __shfl_xor(sum, d));
  }
  if (lane == 0) ss[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    a.cmax[row * a.n_chunks + c] = m;
    a.csum[row * a.n_chunks + c] = sampled ? (ss[0] + ss[1]) + (ss[2] + ss[3])
                                           : fmin(fmin(ss[0], ss[1]), fmin(ss[2], ss[3]));
  }
}

// A row's largest logit and its sum of weights (greedy: the lowest index of
// the largest logit; -1 if all are -infinity), by one wave.
struct RowStat {
  float m;
  double s;
};
__device__ __forceinline__ RowStat row_stat(const VerifyArgs& a, long long row, bool sampled,
                                            double inv_t, int lane) {
  const float* cm = a.cmax + row * a.n_chunks;
  const double* cs = a.csum + row * a.n_chunks;
  float m = -INFINITY;
  for (int c = lane; c < a.n_chunks; c += 64) m = fmaxf(m, cm[c]);
  m = wave_max_dpp(m);
  RowStat r;
  r.m = m;
  if (sampled) {
    double s = 0.0;
    for (int c = lane; c < a.n_chunks; c += 64)
      if (cm[c] > -INFINITY) s += cs[c] * weight(cm[c], m, inv_t);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    r.s = s;
  } else {
    double s = 1e18;
    for (int c = lane; c < a.n_chunks; c += 64)
      if (cm[c] == m) s = fmin(s, cs[c]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s = fmin(s, __shfl_xor(s, d));
    r.s = m > -INFINITY ? s : -1.0;
  }
  return r;
}
// The sum of a node's rest, by one wave.
__device__ __forceinline__ double rest_sum(const VerifyArgs& a, long long row, int lane) {
  double s = 0.0;
  for (int c = lane; c < a.n_chunks; c += 64) s += a.rest[row * a.n_chunks + c];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
  return s;
}
// The target's probability of token v in a row.
__device__ __forceinline__ double target_p(RowStat r, float x, int v, bool sampled, double inv_t) {
  if (!sampled) return static_cast<double>(v) == r.s ? 1.0 : 0.0;
  return r.s > 0.0 && r.m > -INFINITY ? weight(no_nan(x), r.m, inv_t) / r.s : 0.0;
}

// The siblings of rank 0 .. n-1 below a node: rows and the sums of their rests.
struct Chain {
  int row[kMaxChildren];
  double sum[kMaxChildren];
};
// R(v) after the rejection of the first n siblings, normalized by the last
// rest that counts.  r: the target's probability.
__device__ __forceinline__ double chain_rest(const VerifyArgs& a, const Chain& ch, int n, double r,
                                             int v) {
  double s = 1.0;
  for (int i = 0; i < n; ++i) {
    if (ch.sum[i] < kRest) continue;
    const double q = a.draft[static_cast<long long>(ch.row[i]) * a.vocab + v];
    r = fmax(r / s - q, 0.0);
    s = ch.sum[i];
  }
  return r / s;
}

// Grid: (chunk, node, sequence), for the children of rank `rank`.
__global__ void __launch_bounds__(256) verify_rest_kernel(const VerifyArgs a, int rank) {
  const int s = blockIdx.z, node = blockIdx.y, c = blockIdx.x;
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  if (node >= w.n) return;
  const int2 me = a.tree[w.off + node];
  if (me.x < 0 || me.y != rank) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float t = a.temperature[s];
  const bool sampled = t > 0.f;
  const double inv_t = sampled ? 1.0 / static_cast<double>(t) : 1.0;
  __shared__ Chain ch;
  __shared__ RowStat rs;
  __shared__ double ss[4];
  if (wave == 0) {
    const RowStat r = row_stat(a, w.off + me.x, sampled, inv_t, lane);
    if (lane == 0) rs = r;
  } else if (wave == 1) {
    const int2 other = lane < w.n ? a.tree[w.off + lane] : make_int2(-1, 0);
    if (other.x == me.x && other.y < rank) ch.row[other.y] = w.off + lane;
  }
  __syncthreads();
  for (int i = wave; i < rank; i += 4) {
    const double r = rest_sum(a, ch.row[i], lane);
    if (lane == 0) ch.sum[i] = r;
  }
  __syncthreads();
  const float* x = a.logits + static_cast<long long>(w.off + me.x) * a.vocab;
  const float* q = a.draft + static_cast<long long>(w.off + node) * a.vocab;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) {
    const int v = c * kChunk + i * 256 + threadIdx.x;
    if (v < a.vocab)
      sum += fmax(chain_rest(a, ch, rank, target_p(rs, x[v], v, sampled, inv_t), v) -
                      static_cast<double>(q[v]), 0.0);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) ss[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    a.rest[static_cast<long long>(w.off + node) * a.n_chunks + c] = (ss[0] + ss[1]) + (ss[2] + ss[3]);
}

// The first i of the workgroup's values at which their running sum (from
// `before` on) passes goal and the value is positive; *total: their sum.
// Values 0..kWalk-1 by thread; -1 if there is none.  *last: the last positive one.
struct Found {
  int at, last;
  double before, total;  // the sum in front of `at`, the sum of all
};
__device__ __forceinline__ Found find_in(double v, double before, double goal, double* ws, int* wi) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double run = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
  __syncthreads();
  if (lane == 63) ws[wave] = run;
  if (threadIdx.x < 2) wi[threadIdx.x] = threadIdx.x ? -1 : kWalk;
  __syncthreads();
  double base = before, all = 0.0;
#pragma unroll
  for (int i = 0; i < kWalk / 64; ++i) {
    if (i == wave) base = before + all;
    all += ws[i];
  }
  if (v > 0.0) {
    if (base + run > goal) atomicMin(&wi[0], static_cast<int>(threadIdx.x));
    atomicMax(&wi[1], static_cast<int>(threadIdx.x));
  }
  __syncthreads();
  Found f;
  f.at = wi[0] < kWalk ? wi[0] : -1;
  f.last = wi[1];
  f.total = all;
  f.before = 0.0;
  if (f.at == static_cast<int>(threadIdx.x)) ws[kWalk / 64] = base + run - v;
  __syncthreads();
  if (f.at >= 0) f.before = ws[kWalk / 64];
  return f;
}

// One workgroup a sequence.
__global__ void __launch_bounds__(kWalk) verify_walk_kernel(const VerifyArgs a) {
  const int s = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
  __shared__ double left[kMaxWindow];   // a rejected node's rest
  __shared__ int kids[kMaxWindow][2];   // the end's rejected children: row, token
  __shared__ int s_end, s_kids;
  __shared__ double ws[kWalk / 64 + 1];
  __shared__ int wi[2];
  __shared__ Chain chain;
  const float t = a.temperature[s];
  const bool sampled = t > 0.f;
  const double inv_t = sampled ? 1.0 / static_cast<double>(t) : 1.0;
  const int2 tn = lane < w.n ? a.tree[w.off + lane] : make_int2(-1, 0);
  for (int i = wave; i < w.n; i += kWalk / 64) {
    const RowStat r = row_stat(a, w.off + i, sampled, inv_t, lane);
    double rest = 0.0;
    if (a.draft && __shfl(tn.x, i) >= 0) rest = rest_sum(a, w.off + i, lane);
    if (lane == 0) {
      stat[i] = r;
      left[i] = rest;
    }
  }
  __syncthreads();
  if (wave == 0) {
    // Node `lane`: its token's share of R at its parent, as far as the node
    // alone tells.
    const bool in = tn.x >= 0;
    const int up = in ? tn.x : 0;
    const int tok = lane < w.n ? a.tokens[w.off + lane] : -1;
    const bool real = in && tok >= 0 && tok < a.vocab;
    double r = 0.0, q = 1.0;
    if (real)
      r = target_p(stat[up], a.logits[static_cast<long long>(w.off + up) * a.vocab + tok], tok,
                   sampled, inv_t);
    const float u = in ? a.u_accept[w.off + lane] : 1.f;
    const double full = stat[up].m > -INFINITY ? 1.0 : 0.0;
    uint64_t same = 0, sib = 0;  // earlier siblings with this token, earlier siblings
    for (int j = 1; j < w.n; ++j) {
      const int pj = __shfl(tn.x, j), tj = __shfl(tok, j);
      if (j < lane && in && pj == up && pj >= 0) {
        sib |= 1ull << j;
        if (tj == tok) same |= 1ull << j;
      }
    }
    double mass = full;  // sum of R
    if (a.draft) {
      q = real ? a.draft[static_cast<long long>(w.off + lane) * a.vocab + tok] : 0.0;
      double norm = full;
      for (uint64_t b = sib; b; b &= b - 1) {
        const int j = __builtin_ctzll(b);
        if (left[j] < kRest) continue;
        const double qj =
            real ? a.draft[static_cast<long long>(w.off + j) * a.vocab + tok] : 0.0;
        r = fmax((norm > 0.0 ? r / norm : 0.0) - qj, 0.0);
        norm = left[j];
      }
      mass = norm;
    } else {
      // A point mass: a rejected sibling takes its token's share away.  Node
      // by node, since each depends on what its earlier siblings left.
      double m = lane < w.n && stat[lane < w.n ? lane : 0].m > -INFINITY ? 1.0 : 0.0;
      uint64_t gone = 0;  // rejected nodes whose share is taken
      for (int j = 1; j < w.n; ++j) {
        const int p = __shfl(tn.x, j);
        if (p < 0) continue;
        const uint64_t sm = __shfl(same, j);
        const double rj = sm & gone ? 0.0 : __shfl(r, j);
        const double mp = __shfl(m, p);
        if (lane == j) {
          r = rj;
          mass = mp;
        }
        if (mp - rj >= kRest * mp) {
          if (lane == p) m = mp - rj;
          gone |= 1ull << j;
        }
      }
      if (lane < w.n) left[lane] = gone >> lane & 1 ? 1.0 : 0.0;
    }
    const double bar = q * mass;
    const bool take = in && static_cast<double>(u) * bar < r;
    if (a.prob && lane < w.n)
      a.prob[w.off + lane] =
          lane == 0 ? 1.f : !in ? 0.f : r >= bar ? (r > 0.0 ? 1.f : 0.f)
                                                 : static_cast<float>(r / bar);
    // down the tree: the first accepted child of each node
    const uint64_t yes = __ballot(take);
    int at = 0, n = 0, mine = -1;
    while (true) {
      if (lane == n) mine = at;
      ++n;
      const uint64_t kid = __ballot(in && up == at) & yes;
      if (!kid) break;
      at = __builtin_ctzll(kid);
    }
    if (lane < a.max_window) path[lane] = mine;
    const uint64_t kid = __ballot(in && up == at);
    if (in && up == at) {
      const int k = __popcll(kid & ((1ull << lane) - 1));
      kids[k][0] = w.off + lane;
      kids[k][1] = left[lane] > 0.0 ? tok : -1;
      if (a.draft) {
        chain.row[k] = w.off + lane;
        chain.sum[k] = left[lane];
      }
    }
    if (lane == 0) {
      s_end = at;
      s_kids = __popcll(kid);
      a.n_path[s] = n;
    }
  }
  __syncthreads();

  // The last token: R at the end of the path, in units of the row's weights.
  const int end = s_end, nk = s_kids;
  const RowStat st = stat[end];
  if (st.m == -INFINITY) {
    if (threadIdx.x == 0) a.next[s] = -1;
    return;
  }
  const long long row = w.off + end;
  const float* x = a.logits + row * a.vocab;
  int from = -1;  // the rejected child whose rest is what is left
  if (a.draft)
    for (int i = 0; i < nk; ++i)
      if (chain.sum[i] >= kRest) from = chain.row[i];
  if (!sampled) {  // all the mass is on one token, whether or not a rejection left some of it
    if (threadIdx.x == 0) a.next[s] = static_cast<int>(st.s);
    return;
  }
  // the sum of a chunk
  auto chunk = [&](int c) {
    if (c >= a.n_chunks) return 0.0;
    if (from >= 0) return a.rest[static_cast<long long>(from) * a.n_chunks + c];
    const float cm = a.cmax[row * a.n_chunks + c];
    if (!(cm > -INFINITY)) return 0.0;
    double v = a.csum[row * a.n_chunks + c] * weight(cm, st.m, inv_t);
    if (!a.draft)
      for (int i = 0; i < nk; ++i) {
        const int tok = kids[i][1];
        bool again = false;
        for (int j = 0; j < i; ++j) again |= kids[j][1] == tok;
        if (tok >= 0 && tok < a.vocab && tok / kChunk == c && !again)
          v -= weight(no_nan(x[tok]), st.m, inv_t);
      }
    return fmax(v, 0.0);
  };
  double total = 0.0;
  for (int c0 = 0; c0 < a.n_chunks; c0 += kWalk) {
    const Found f = find_in(chunk(c0 + threadIdx.x), 0.0, 0.0, ws, wi);
    total += f.total;
  }
  const double goal = static_cast<double>(a.u_sample[s]) * total;
  int c_at = -1, c_last = 0;
  double before = 0.0, run = 0.0;
  for (int c0 = 0; c0 < a.n_chunks && c_at < 0; c0 += kWalk) {
    const Found f = find_in(chunk(c0 + threadIdx.x), run, goal, ws, wi);
    if (f.at >= 0) {
      c_at = c0 + f.at;
      before = f.before;
    }
    if (f.last >= 0) c_last = c0 + f.last;
    run += f.total;
  }
  const bool past = c_at < 0;  // u_sample is 1 or more, or the sums round so
  if (past) c_at = c_last;
  int tok = -1, last = 0;
  run = before;
  for (int v0 = 0; v0 < kChunk && tok < 0; v0 += kWalk) {
    const int v = c_at * kChunk + v0 + threadIdx.x;
    double r = 0.0;
    if (v < a.vocab) {
      if (a.draft) {
        r = chain_rest(a, chain, nk, target_p(st, x[v], v, sampled, inv_t), v);
        // (chunk sums are of the unnormalized rest, or of the row's weights)
        if (from >= 0) {
          double last_sum = 1.0;
          for (int i = 0; i < nk; ++i)
            if (chain.sum[i] >= kRest) last_sum = chain.sum[i];
          r *= last_sum;
        } else {
          r *= st.s;
        }
      } else {
        r = weight(no_nan(x[v]), st.m, inv_t);
        for (int i = 0; i < nk; ++i)
          if (kids[i][1] == v) r = 0.0;
      }
    }
    const Found f = find_in(r, run, past ? INFINITY : goal, ws, wi);
    if (f.at >= 0) tok = c_at * kChunk + v0 + f.at;
    if (f.last >= 0) last = c_at * kChunk + v0 + f.last;
    run += f.total;
  }
  if (threadIdx.x == 0) a.next[s] = tok >= 0 ? tok : last;
}

static size_t up16(size_t n) { return (n + 15) / 16 * 16; }
struct VerifyWs {
  size_t tree, cmax, csum, rest, bytes;
};
static VerifyWs verify_ws(int n_tokens, int vocab, int max_children) {
  const size_t t = n_tokens, c = (vocab + kChunk - 1) / kChunk;
  VerifyWs w;
  w.tree = 0;
  w.cmax = w.tree + up16(t * sizeof(int2));
  w.csum = w.cmax + up16(t * c * sizeof(float));
  w.rest = w.csum + up16(t * c * sizeof(double));
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
  a.tree = reinterpret_cast<int2*>(b + l.tree);
  a.cmax = reinterpret_cast<float*>(b + l.cmax);
  a.csum = reinterpret_cast<double*>(b + l.csum);
  a.rest = reinterpret_cast<double*>(b + l.rest);
  a.n_tokens = n_tokens;
  a.max_window = max_window;
  a.vocab = vocab;
  a.n_chunks = (vocab + kChunk - 1) / kChunk;
  a.max_children = max_children;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(a.n_chunks, max_window, n_seq);
  hipLaunchKernelGGL(verify_rows_kernel, grid, dim3(256), 0, s, a);
  if (int st = check_launch(nm)) return st;
  if (draft_probs)
    for (int r = 0; r < max_children && r < max_window - 1; ++r) {
      hipLaunchKernelGGL(verify_rest_kernel, grid, dim3(256), 0, s, a, r);
      if (int st = check_launch(nm)) return st;
    }
  hipLaunchKernelGGL(verify_walk_kernel, dim3(n_seq), dim3(kWalk), 0, s, a);
  return check_launch(nm);
}

}  // extern "C"
