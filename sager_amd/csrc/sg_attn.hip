// sg_attn.hip - the windows' attention over a paged fp16 cache, and the
// accepted tokens' way into it.
//
// For a kv head, the rows of a product are (node, query head of the group).
// A workgroup takes a block of rows and a part of a sequence's keys, 64 keys
// a step through two LDS buffers: S^T = K Q^T, then O^T = V^T P^T.  With keys
// as the first product's rows, a lane of v_mfma_f32_16x16x32_f16 gets four
// consecutive keys of one query row; and since the order of a product's 32
// terms is free, V's operand is, per lane, one column of V at four and four
// consecutive keys, which ds_read_b64_tr_b16 reads from V's rows as they lie
// in memory.  Two kernels:
//
//   attn_few_kernel   blocks of 16 or 32 rows: the four waves share the keys
//                     of the first product and the columns of the second, P
//                     goes through LDS between them.  K and V are read from
//                     LDS once, no wave holds more than a quarter of O, and
//                     nothing is joined at the end but the rows' sums.
//   attn_rows_kernel  blocks of 256 rows: each of eight waves has 32 rows of
//                     its own and reads all of K and V from LDS; P stays in
//                     its lanes, and one barrier a step orders the copies.
//
// A row's running maximum is a reference point `mref`, set 8 (in powers of 2)
// below the largest score of its step, that moves only when a score passes it
// by 15: p = 2^(s - mref) is at most 2^15, which fits fp16.  p is rounded to
// fp16 for the product: 2^-11 of a weight, no more than the output's own
// rounding, down to 2^-22 of the largest; below it 2^-33 of the largest, so
// that smaller weights bring nothing (131,072 keys that all have just that
// little together 2^-16).  l = sum p is fp32, of the unrounded p.
#include <algorithm>

#include "sg_attn.hpp"

namespace sg {

// ---- blocks of 16 or 32 rows ---------------------------------------------------------------
// LDS: K and V of two steps, P, the rows' maxima and sums of the four waves,
// the nodes' ancestors, the flags.
template <int D, int RT>
struct FewLds {
  static constexpr uint32_t kRows = 16 * RT;
  static constexpr uint32_t kP = 4 * Part<D>::kStep;
  static constexpr uint32_t kMax = kP + kRows * kKeys * 2;
  static constexpr uint32_t kSeen = kMax + 4 * kRows * 4;
  static constexpr uint32_t kFlags = kSeen + kMaxWindow * 8;
  static constexpr uint32_t kBytes = kFlags + 16;
};

// RT: tiles of 16 rows.  Wave w brings keys 16 w.. of a step, has them in the
// first product, and has columns w D/4 .. of all keys in the second.
// Bound by memory where the caches are long (24 sequences of one token, 77 to
// 4,001 cached, 8 kv heads of 128: 200 MB in 37 us, 5.4 TB/s within the
// launch) and by the rounds of latency where they are short: lengths, pages,
// copies, the two products (4 tokens over 4,099: 10 us for 8.5 MB).  Up to 128
// rows it is the faster form, though blocks of 32 read the keys again, from
// the XCD's L2: 64 rows over 32,768 tokens of dimension 256 28.0 us against
// 32.6, 128 rows 37.8 against 40.9; 200 rows 59.9 against 45.9.
template <int D, int RT>
__global__ void __launch_bounds__(256) attn_few_kernel(const AttnArgs a) {
  typedef Part<D> P;
  typedef FewLds<D, RT> L;
  constexpr int DQ = D / 64;  // 16-column tiles of a wave's part of O
  constexpr int kRows = L::kRows;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  P t{a};
  if (!t.start(lds)) return;
  const int lane = t.lane, col = t.col, grp = t.grp, row0 = t.rb * kRows;
  // flags of odd and even steps: 1 + the last step whose reference points move, and the last
  // with infinities or NaN in its window's V
  int* rise = reinterpret_cast<int*>(lds + L::kFlags);
  int* odds = rise + 2;
  float* mx = reinterpret_cast<float*>(lds + L::kMax);
  uint64_t* seen = reinterpret_cast<uint64_t*>(lds + L::kSeen);  // node: whom it sees

  int step = t.begin;
  int page = t.page_of(step, wave), page_next = 0;
  if (step < t.end) {
    t.template issue<true>(step, wave, page, 0);
    page_next = t.page_of(step + 1, wave);
  }
  if (threadIdx.x < 4) rise[threadIdx.x] = 0;
  if (wave == 3) seen[lane] = ancestors(a.parent, t.win, lane);

  h8 qf[RT][P::KK];
  f4 acc[RT][DQ];
  // lim: the score, less mref, above which mref moves: kRise once it is set
  float mref[RT], l[RT], lim[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    t.load_q(row0 + rt * 16 + col, qf[rt]);
    mref[rt] = 0.f;
    l[rt] = 0.f;
    lim[rt] = -INFINITY;
#pragma unroll
    for (int d = 0; d < DQ; ++d) acc[rt][d] = (f4){0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t koff0 = t.k_offset() + wave * 16 * D * 2, voff0 = t.v_offset();
  uint32_t koff[P::KO], voff[DQ];
#pragma unroll
  for (int i = 0; i < P::KO; ++i) koff[i] = P::k_piece(koff0, i);
#pragma unroll
  for (int d = 0; d < DQ; ++d) voff[d] = t.v_tile(voff0, wave * DQ + d);
  // P: [row][two halves of 32 keys][grp][two blocks of 16 keys][4], 16-B pieces
  // swizzled over the row's eight
  unsigned char* const pl = lds + L::kP;
  const int psw = (col >> 1) & 7;
  unsigned char* const p_out =
      pl + col * 128 + ((((wave >> 1) * 4 + grp) ^ psw) << 4) + (wave & 1) * 8;

  bar();  // the flags are cleared
  for (; step < t.end; ++step) {
    const int par = step & 1;
    const uint32_t there = t.present(step, wave, page);
    const bool plain = t.plain(step, wave, page);
    wait_vm();
    if (!plain && t.fix_v(step, wave, there)) odds[par] = step + 1;
    bar();  // everybody's copies of this step are here, and nobody reads the other buffers or P
    if (step + 1 < t.end) t.template issue<true>(step + 1, wave, page_next, 0);
    page = page_next;
    if (step + 2 < t.end) page_next = t.page_of(step + 2, wave);

    f4 s[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < P::KK; ++st) {
      const h8 kf = t.k_frag(koff[st % P::KO] + par * 2 * P::kStep, st);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        s[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][st], s[rt], 0, 0, 0);
    }
    float e[RT][4], top[RT], sum[RT];
    auto weigh = [&](int rt, float by) {  // row tile rt's p = 2^(e - by), into LDS
      float p[4];
      h4 ph;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = __builtin_amdgcn_exp2f(e[rt][i] - by);
        ph[i] = static_cast<_Float16>(p[i]);
      }
      sum[rt] = (p[0] + p[1]) + (p[2] + p[3]);
      *reinterpret_cast<h4*>(p_out + rt * 16 * 128) = ph;
    };
    bool move = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[rt][i] = __builtin_fmaf(s[rt][i], a.scale_log2, -mref[rt]);
      if (!plain) {
        const uint32_t see = t.seen_bits(step, wave, there, seen[t.node_of(row0 + rt * 16 + col)]);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[rt][i] = see & 1u << i ? e[rt][i] : -INFINITY;
      }
      top[rt] = max3(max3(e[rt][0], e[rt][1], e[rt][2]), e[rt][3], e[rt][3]);
      move |= top[rt] > lim[rt];
      weigh(rt, 0.f);
    }
    if (__any(move)) rise[par] = step + 1;
    bar();  // P is here

    if (rise[par] == step + 1) {
      // The reference points move: the rows' maxima over the waves, then P once more.
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float m = fmaxf(top[rt], __shfl_xor(top[rt], 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        if (grp == 0) mx[wave * kRows + rt * 16 + col] = m;
      }
      bar();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float* mr = mx + rt * 16 + col;
        const float m = fmaxf(fmaxf(mr[0], mr[kRows]), fmaxf(mr[2 * kRows], mr[3 * kRows]));
        const bool set = m > lim[rt], begun = lim[rt] > 0.f;
        const float by = set ? m - kBelow : 0.f;
        const float f = !set ? 1.f : begun ? __builtin_amdgcn_exp2f(-by) : 0.f;
        mref[rt] += by;
        l[rt] *= f;
#pragma unroll
        for (int d = 0; d < DQ; ++d) acc[rt][d] *= f;
        lim[rt] = set ? kRise : lim[rt];
        weigh(rt, by);
      }
      bar();
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] += sum[rt];

    if (odds[par] == step + 1) {  // one by one, to the rows that see them
#pragma unroll 1
      for (int r = 0; r < kKeys; ++r) {
        const int node = step * kKeys + r - t.len;
        if (node < 0 || node >= t.win.n) continue;
        const int piece = (r >> 5) * 4 + ((r & 15) >> 2);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float w = half_bits_to_float(*reinterpret_cast<const uint16_t*>(
              pl + (rt * 16 + col) * 128 + ((piece ^ psw) << 4) + (r >> 4 & 1) * 8 + (r & 3) * 2));
          const bool see = seen[t.node_of(row0 + rt * 16 + col)] >> node & 1;
#pragma unroll
          for (int d = 0; d < DQ; ++d)
            t.add_odd(acc[rt][d], node, (wave * DQ + d) * 16 + 4 * grp, w, see);
        }
      }
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      h8 pf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        pf[rt] = *reinterpret_cast<const h8*>(pl + (rt * 16 + col) * 128 +
                                              (((st * 4 + grp) ^ psw) << 4));
#pragma unroll
      for (int d = 0; d < DQ; ++d) {
        const h8 vf = t.v_frag(voff[d] + par * 2 * P::kStep, st);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt], acc[rt][d], 0, 0, 0);
      }
    }
  }

  // the rows' sums over the waves, and out
  bar();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    if (grp == 0) mx[wave * kRows + rt * 16 + col] = l[rt];
  }
  bar();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + col;
    const float* lr = mx + rt * 16 + col;
    float lt = (lr[0] + lr[kRows]) + (lr[2 * kRows] + lr[3 * kRows]);
    if (!seen[t.node_of(r)]) lt = 0.f;  // an absent node
    t.template store<DQ, 16>(r, wave * (D / 4) + 4 * grp, acc[rt], mref[rt], lt,
                             wave == 0 && grp == 0);
  }
}

// ---- blocks of 256 rows ---------------------------------------------------------------------
constexpr int kRowWaves = 8, kRowTiles = 2;  // 16-row tiles of a wave
template <int D>
struct RowsLds {
  static constexpr uint32_t kSeen = 4 * Part<D>::kStep;
  static constexpr uint32_t kThere = kSeen + kMaxWindow * 8;
  static constexpr uint32_t kFlags = kThere + 16;
  static constexpr uint32_t kBytes = kFlags + 16;
};

// Each wave brings 16 keys of K (the first four) or V.
// Bound by the matrix cores and the vector instructions between the products:
// a wave's registers (128 of O, 64 of Q at dimension 256) leave two waves a
// SIMD.  64 tokens of 16 heads over 131,071 cached ones, 2 kv heads of 256: 137
// GFLOP in 166 us under the profiler, 830 TFLOP/s (a large matrix product here:
// 1,190; a pass of this launch and the join among others 162 us); the matrix
// cores are busy 45 % of the cycles, vector instructions some 30 %, the LDS
// 23 %.  (Wave priorities around either phase: 2 to 20 us more; half of the
// waves a phase behind the others, with a second barrier a step: 8 more.)
template <int D>
__global__ void __launch_bounds__(64 * kRowWaves) attn_rows_kernel(const AttnArgs a) {
  typedef Part<D> P;
  typedef RowsLds<D> L;
  constexpr int RT = kRowTiles, NW = kRowWaves, DT = D / 16;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blk = wave & 3, kv = 1 + (wave >> 2);
  P t{a};
  if (!t.start(lds)) return;
  const int lane = t.lane, col = t.col, grp = t.grp;
  const int row0 = (t.rb * NW + wave) * 16 * RT;
  int* odds = reinterpret_cast<int*>(lds + L::kFlags);  // 1 + the last odd (even) step with any
  uint64_t* seen = reinterpret_cast<uint64_t*>(lds + L::kSeen);

  int step = t.begin;
  int page = t.page_of(step, blk), page_next = 0;
  if (step < t.end) {
    t.template issue<false>(step, blk, page, kv);
    page_next = t.page_of(step + 1, blk);
  }
  if (threadIdx.x < 2) odds[threadIdx.x] = 0;
  if (wave == NW - 1) seen[lane] = ancestors(a.parent, t.win, lane);

  h8 qf[RT][P::KK];
  f4 acc[RT][DT];
  // lim: the score, less mref, above which mref moves: kRise once it is set
  float mref[RT], l[RT], lim[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    t.load_q(row0 + rt * 16 + col, qf[rt]);
    mref[rt] = 0.f;
    l[rt] = 0.f;
    lim[rt] = -INFINITY;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[rt][d] = (f4){0.f, 0.f, 0.f, 0.f};
  }
  uint32_t kbase = t.k_offset() + (step & 1) * 2 * P::kStep;  // of the present step's buffer
  uint32_t vbase = t.v_offset() + (step & 1) * 2 * P::kStep;
  // which of a step's keys are there, by step parity and block of 16
  uint16_t* there_of = reinterpret_cast<uint16_t*>(lds + L::kThere);

  P::settle_q(qf);
  bar();  // the flags are cleared
  for (; step < t.end; ++step) {
    const int par = step & 1;
    const uint32_t mine = t.present(step, blk, page);
    if (wave < 4) there_of[par * 4 + blk] = mine;
    wait_vm();
    if (kv != 1 && !t.plain(step, blk, page) && t.fix_v(step, blk, mine)) odds[par] = step + 1;
    bar();  // everybody's copies of this step are here, and nobody reads the other buffers
    const uint64_t there = reinterpret_cast<const uint64_t*>(there_of)[par];
    if (step + 1 < t.end) t.template issue<false>(step + 1, blk, page_next, kv);
    page = page_next;
    if (step + 2 < t.end) page_next = t.page_of(step + 2, blk);
    // (the same in every lane: into scalar registers)
    const uint32_t there_lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(there));
    const uint32_t there_hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(there >> 32));
    const bool plain = (step + 1) * kKeys <= t.len && (there_lo & there_hi) == 0xFFFFFFFFu;
    const bool odd = !plain && odds[par] == step + 1;

#pragma unroll 1
    for (int st = 0; st < 2; ++st) {
      f4 s[2][RT];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[b][rt] = (f4){0.f, 0.f, 0.f, 0.f};
      // (the two blocks' pieces one step ahead; the fences keep the compiler from
      // reading further ahead: registers)
      h8 kn[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) kn[b] = t.k_frag(P::k_piece(kbase, 0), 0, b);
#pragma unroll
      for (int ks = 0; ks < P::KK; ++ks) {
        const h8 kf[2] = {kn[0], kn[1]};
        if (ks + 1 < P::KK) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
            kn[b] = t.k_frag(P::k_piece(kbase, (ks + 1) % P::KO), ks + 1, b);
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            s[b][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b], qf[rt][ks], s[b][rt], 0, 0, 0);
      }
      bool move = false;
      float top[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[b][rt][i] = __builtin_fmaf(s[b][rt][i], a.scale_log2, -mref[rt]);
          if (!plain) {
            const uint32_t see =
                t.seen_bits(step, 2 * st + b, (st ? there_hi : there_lo) >> (16 * b) & 0xFFFFu,
                            seen[t.node_of(row0 + rt * 16 + col)]);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[b][rt][i] = see & 1u << i ? s[b][rt][i] : -INFINITY;
          }
        }
        top[rt] = max3(max3(s[0][rt][0], s[0][rt][1], s[0][rt][2]),
                       max3(s[0][rt][3], s[1][rt][0], s[1][rt][1]),
                       max3(s[1][rt][2], s[1][rt][3], s[1][rt][3]));
        move |= top[rt] > lim[rt];
      }
      if (__any(move)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float m = fmaxf(top[rt], __shfl_xor(top[rt], 16));
          m = fmaxf(m, __shfl_xor(m, 32));
          const bool set = m > lim[rt], begun = lim[rt] > 0.f;
          const float by = set ? m - kBelow : 0.f;
          const float f = !set ? 1.f : begun ? __builtin_amdgcn_exp2f(-by) : 0.f;
          mref[rt] += by;
          l[rt] *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[rt][d] *= f;
          lim[rt] = set ? kRise : lim[rt];
#pragma unroll
          for (int b = 0; b < 2; ++b) s[b][rt] -= by;
        }
      }
      h8 pf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[b][rt][i] = __builtin_amdgcn_exp2f(s[b][rt][i]);
            pf[rt][4 * b + i] = static_cast<_Float16>(s[b][rt][i]);
          }
        l[rt] += ((s[0][rt][0] + s[0][rt][1]) + (s[0][rt][2] + s[0][rt][3])) +
                 ((s[1][rt][0] + s[1][rt][1]) + (s[1][rt][2] + s[1][rt][3]));
      }
      if (odd) {
#pragma unroll 1
        for (int r = 0; r < 32; ++r) {  // one by one, to the rows that see them
          const int node = step * kKeys + 32 * st + r - t.len;
          if (node < 0 || node >= t.win.n) continue;
          const int from = col + 16 * ((r & 15) >> 2);  // the lane that has key r's weight
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            float mine = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              mine = i == (r >> 4) * 4 + (r & 3) ? s[i >> 2][rt][i & 3] : mine;
            const float w = __shfl(mine, from);
            const bool see = seen[t.node_of(row0 + rt * 16 + col)] >> node & 1;
#pragma unroll
            for (int d = 0; d < DT; ++d) t.add_odd(acc[rt][d], node, d * 16 + 4 * grp, w, see);
          }
        }
      }
      h8 next[2] = {t.v_frag(P::v_tile(vbase, 0), 0), t.v_frag(P::v_tile(vbase, 1), 0)};
#pragma unroll
      for (int d = 0; d < DT; ++d) {  // two tiles read ahead
        const h8 vf = next[d % 2];
        asm volatile("" ::: "memory");
        if (d + 2 < DT) next[d % 2] = t.v_frag(P::v_tile(vbase, d + 2), 0);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt], acc[rt][d], 0, 0, 0);
      }
      kbase += 32 * D * 2;
      vbase += 32 * D * 2;
    }
    // the other buffer
    kbase += (par ? -2 : 2) * static_cast<int>(P::kStep) - 64 * D * 2;
    vbase += (par ? -2 : 2) * static_cast<int>(P::kStep) - 64 * D * 2;
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + col;
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    const float lt = seen[t.node_of(r)] ? l[rt] : 0.f;  // 0: an absent node
    t.template store<DT, 16>(r, 4 * grp, acc[rt], mref[rt], lt, grp == 0);
  }
}

// ---- the accepted tokens into the cache, or whole windows (no path) -----------
struct CommitArgs {
  const uint16_t *k, *v;
  long long k_stride, v_stride, k_layer, v_layer, layer_stride;
  uint16_t *kc, *vc;
  const int *pages, *length, *win_off, *path, *n_path;
  int* length_out;
  int n_tokens, max_window, n_layers, n_kv, dim, n_pages, page_log2, pages_per_seq;
};

// Grid: (16-B pieces of a window's K and V rows, sequence, kCommitLayers
// layers).  A thread looks its piece's place up once and then copies it in
// every layer, whose loads are under way together.  One window of 4 over 10
// layers takes 3.2 us, four dependent rounds (the path's length, its node, the
// page, the copy); 32 windows of up to 16 over 40 layers, 65 MB, 19 us, 3.4
// TB/s (a layer a thread: 26.8 us).
constexpr int kCommitLayers = 8;
__global__ void __launch_bounds__(256) kv_commit_kernel(const CommitArgs a) {
  const int s = blockIdx.y, l0 = blockIdx.z * kCommitLayers;
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  const int n = a.path ? min(max(a.n_path[s], 0), a.max_window) : w.n;
  const int len = a.length[s];
  if (a.length_out && blockIdx.x == 0 && l0 == 0 && threadIdx.x == 0) a.length_out[s] = len + n;
  const int pieces = a.n_kv * (a.dim / 8);
  int x = blockIdx.x * 256 + threadIdx.x;
  const bool is_v = x & 1;  // K's and V's piece of one place by neighbours
  x >>= 1;
  const int i = x / pieces;
  if (i >= n) return;
  x -= i * pieces;
  const int h = x / (a.dim / 8), c = x - h * (a.dim / 8);
  const int node = a.path ? a.path[static_cast<long long>(s) * a.max_window + i] : i;
  const long long pos = static_cast<long long>(len) + i;
  if (len < 0 || node < 0 || node >= w.n || pos >> a.page_log2 >= a.pages_per_seq) return;
  const int page = a.pages[static_cast<long long>(s) * a.pages_per_seq + (pos >> a.page_log2)];
  if (page < 0 || page >= a.n_pages) return;
  const long long step = is_v ? a.v_layer : a.k_layer;
  const uint16_t* src = (is_v ? a.v + (w.off + node) * a.v_stride : a.k + (w.off + node) * a.k_stride) +
                        h * a.dim + c * 8 + l0 * step;
  const long long slot = ((static_cast<long long>(page) * a.n_kv + h) << a.page_log2) +
                         (pos & ((1 << a.page_log2) - 1));
  uint16_t* dst = (is_v ? a.vc : a.kc) + l0 * a.layer_stride + slot * a.dim + c * 8;
  if (l0 + kCommitLayers <= a.n_layers) {
    u32x4 v[kCommitLayers];
#pragma unroll
    for (int l = 0; l < kCommitLayers; ++l) v[l] = *reinterpret_cast<const u32x4_u*>(src + l * step);
#pragma unroll
    for (int l = 0; l < kCommitLayers; ++l) *reinterpret_cast<u32x4*>(dst + l * a.layer_stride) = v[l];
  } else {
    for (int l = 0; l0 + l < a.n_layers; ++l)
      *reinterpret_cast<u32x4*>(dst + l * a.layer_stride) =
          *reinterpret_cast<const u32x4_u*>(src + l * step);
  }
}

// ---- host -----------------------------------------------------------------------

// How a call is laid out: rows of a workgroup, the most units.
struct Layout {
  int block_rows, row_blocks, max_units, goal;
  bool cut;
  int few[2];                         // the most sequences for less than one round, and two
  size_t plan_bytes, o_bytes, bytes;  // of the workspace
};
static Layout attn_layout(int n_seq, int max_window, int max_len, int group, int n_kv, int dim) {
  Layout l;
  const long long rows = static_cast<long long>(max_window) * group;
  // (one token of 32 heads over 8 kv heads, 16,384 cached: 14.4 us by blocks of
  // 16, 15.2 by 32; 96 rows of 6 sequences 27.0 by 32, 33.7 by 256; 200 rows
  // over 32,768 45.9 by 256, 59.9 by 32)
  l.block_rows = rows > 128 ? 256 : rows > 16 ? 32 : 16;
  l.row_blocks = static_cast<int>((rows + l.block_rows - 1) / l.block_rows);
  const long long units = static_cast<long long>(n_seq) * n_kv;
  const long long most = (static_cast<long long>(max_len) + max_window + kKeys - 1) / kKeys;
  // workgroups that the card holds at once (by their LDS), and units: a unit's
  // row blocks are on one of the 8 XCDs, and 11 units of three on the 32 CUs of
  // an XCD would take two rounds
  const int each = dim == 256 || l.block_rows == 256 ? 1 : dim == 128 ? 2 : 4;
  const long long slots = 256 * each;
  const long long per = 32 * each >= l.row_blocks ? 32 * each / l.row_blocks * 8 : 8;
  // Heads of sequences for less than two rounds of workgroups: parts of equal
  // length.  More: only what is longer than a round's share is cut, the others
  // are written without a join (200 sequences of 1,500 tokens, 8 kv heads of
  // 128: 244 us, 290 with all in equal parts; of 300 tokens and one of 30,000:
  // 83 us, 515 without a cut; 75 sequences of 100 to 3,000, which is 1.2
  // rounds: 102 us in equal parts, 112 with only the longest cut).  A full
  // round of at most 8 steps is not cut (200 sequences of 10 to 400: 45 us, 66).
  const bool rounds = units >= 2 * slots;
  for (int i = 0; i < 2; ++i) l.few[i] = static_cast<int>(((i + 1) * slots - 1) / n_kv);
  long long n = units;
  l.cut = most > 1 && (units < slots || most > 8);
  l.goal = 1;
  if (l.cut && !rounds) {
    n = (2 * units + per - 1) / per * per;
    // (a part a head lost to rounding; one in a thousand less: parts_of rounds)
    l.goal = static_cast<int>(n_seq <= 64 ? n : n - units - ((n - units) >> 10));
  } else if (l.cut) {
    n = units + per;
    l.goal = static_cast<int>(per - ((per + 1023) >> 10));
  }
  l.max_units = n > 0x7FFFFF00 ? 0x7FFFFF00 : static_cast<int>(n);
  const size_t part_rows =
      static_cast<size_t>((l.max_units + 7LL) / 8 * 8) * l.row_blocks * l.block_rows;
  l.plan_bytes = l.cut ? (static_cast<size_t>(n_seq) * sizeof(int2) + 15) / 16 * 16 : 0;
  l.o_bytes = l.cut ? part_rows * dim * sizeof(float) : 0;
  l.bytes = l.plan_bytes + l.o_bytes + (l.cut ? part_rows * sizeof(float2) : 0);
  return l;
}

template <int D>
static int attn_launch(const AttnArgs& a, hipStream_t s, const char* nm) {
  const dim3 grid(static_cast<unsigned>((a.max_units + 7LL) / 8 * 8 * a.row_blocks));
  if (a.block_rows == 256)
    hipLaunchKernelGGL(attn_rows_kernel<D>, grid, dim3(64 * kRowWaves), RowsLds<D>::kBytes, s, a);
  else if (a.block_rows == 32)
    hipLaunchKernelGGL((attn_few_kernel<D, 2>), grid, dim3(256), (FewLds<D, 2>::kBytes), s, a);
  else
    hipLaunchKernelGGL((attn_few_kernel<D, 1>), grid, dim3(256), (FewLds<D, 1>::kBytes), s, a);
  if (int st = check_launch(nm)) return st;
  if (a.cut) {
    hipLaunchKernelGGL(attn_join_kernel<D>, dim3(a.n_seq * a.max_window * a.n_heads),
                       dim3(kJoinThreads<D>), 0, s, a);
    return check_launch(nm);
  }
  return SG_OK;
}

static int commit(const uint16_t* k, const uint16_t* v, long long k_stride, long long v_stride,
                  long long k_layer_stride, long long v_layer_stride, const sg_kv_cache* cache,
                  const int* win_off, const int* path, const int* n_path, int* length_out,
                  int n_seq, int n_tokens, int max_window, int most, void* stream, const char* nm) {
  if (!k || !v || !win_off) return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (int st = check_cache(cache, n_seq, n_tokens, max_window, nm, most)) return st;
  const long long row = static_cast<long long>(cache->n_kv_heads) * cache->head_dim;
  if (k_stride < row || v_stride < row)
    return set_error(SG_ERR_GEOMETRY, "%s: a token stride is less than a token", nm);
  if (reinterpret_cast<uintptr_t>(k) % 2 || reinterpret_cast<uintptr_t>(v) % 2)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: k and v must be 2-B aligned", nm);
  const long long pieces = 2LL * max_window * (row / 8);
  if (n_seq > 65535 || cache->n_layers > 65535 || pieces > 0x7FFFFFFF - 256)
    return set_error(SG_ERR_UNSUPPORTED, "%s: n_seq=%d n_layers=%d n_kv_heads=%d", nm, n_seq,
                     cache->n_layers, cache->n_kv_heads);
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
  CommitArgs a;
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.k_layer = k_layer_stride;
  a.v_layer = v_layer_stride;
  a.layer_stride = cache->layer_stride;
  a.kc = cache->k;
  a.vc = cache->v;
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
  hipLaunchKernelGGL(kv_commit_kernel,
                     dim3(static_cast<unsigned>((pieces + 255) / 256), n_seq,
                          (cache->n_layers + kCommitLayers - 1) / kCommitLayers),
                     dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return check_launch(nm);
}

}  // namespace sg

extern "C" {

size_t sg_attn_tree_workspace_bytes(int n_seq, int max_window, int max_len, int n_heads,
                                    int n_kv_heads, int head_dim) {
  if (n_seq <= 0 || max_window <= 0 || max_len < 0 || n_kv_heads <= 0 ||
      n_heads <= 0 || n_heads % n_kv_heads != 0)
    return 0;
  // Enough for every smaller call too: within a way of cutting fewer sequences
  // have no more units, but fewer may be cut where more are not, and parts of
  // fewer row blocks may be more of them.  (A shorter cache is cut no sooner.)
  const int group = n_heads / n_kv_heads;
  auto layout = [&](int n, int window) {
    return sg::attn_layout(n, window, max_len, group, n_kv_heads, head_dim);
  };
  size_t bytes = 0;
  for (int window = std::min(max_window, sg::kMaxWindow); window > 0; --window) {
    const sg::Layout l = layout(n_seq, window);
    bytes = std::max(bytes, l.bytes);
    for (int few : l.few)
      if (few > 0 && few < n_seq) bytes = std::max(bytes, layout(few, window).bytes);
  }
  return bytes;
}

int sg_attn_tree_f16(const uint16_t* q, const uint16_t* k, const uint16_t* v, long long q_stride,
                     long long k_stride, long long v_stride, const sg_kv_cache* cache, int layer,
                     const int* win_off, const int* parent, uint16_t* out, void* ws,
                     size_t ws_bytes, int n_seq, int n_tokens, int max_window, int max_len,
                     int n_heads, float scale, void* stream) {
  const char* nm = "sg_attn_tree_f16";
  using namespace sg;
  if (!q || !k || !v || !win_off || !out)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (int st = check_cache(cache, n_seq, n_tokens, max_window, nm)) return st;
  const int n_kv = cache->n_kv_heads, dim = cache->head_dim;
  if (layer < 0 || layer >= cache->n_layers || max_len < 0 || n_heads <= 0 || n_heads % n_kv != 0)
    return set_error(SG_ERR_GEOMETRY, "%s: layer=%d of %d, max_len=%d, n_heads=%d of %d kv heads",
                     nm, layer, cache->n_layers, max_len, n_heads, n_kv);
  if (max_len > 0x7FFFF000)
    return set_error(SG_ERR_UNSUPPORTED, "%s: max_len=%d is too long", nm, max_len);
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 || k_stride % 8 ||
      v_stride % 8 || reinterpret_cast<uintptr_t>(q) % 2 || reinterpret_cast<uintptr_t>(out) % 8)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: k and v must be 16-B aligned, out 8-B", nm);
  if (q_stride < static_cast<long long>(n_heads) * dim ||
      k_stride < static_cast<long long>(n_kv) * dim || v_stride < static_cast<long long>(n_kv) * dim)
    return set_error(SG_ERR_GEOMETRY, "%s: a token stride is less than a token", nm);
  const long long units = static_cast<long long>(n_seq) * n_kv;
  const long long join = static_cast<long long>(n_seq) * max_window * n_heads;
  const long long rows = static_cast<long long>(max_window) * (n_heads / n_kv);
  // a launch has less than 2^32 threads, two units to a kv head
  if (units * (rows / 16 + 1) > 0x1FFFFF || join * 2 * dim > 0xFFFFFFFFLL)
    return set_error(SG_ERR_UNSUPPORTED, "%s: too many sequences", nm);
  // (workgroups read the inputs while others write)
  const long long last = n_tokens - 1, n_out = static_cast<long long>(n_tokens) * n_heads * dim;
  if (overlap(out, n_out, q, last * q_stride + n_heads * dim) ||
      overlap(out, n_out, k, last * k_stride + n_kv * dim) ||
      overlap(out, n_out, v, last * v_stride + n_kv * dim))
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: out overlaps q, k or v", nm);
  const Layout l = attn_layout(n_seq, max_window, max_len, n_heads / n_kv, n_kv, dim);
  if (l.bytes && (!ws || ws_bytes < l.bytes || reinterpret_cast<uintptr_t>(ws) % 16))
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: the workspace needs %zu bytes, 16-B aligned", nm,
                     l.bytes);
  const uint16_t* const kc = cache->k + layer * cache->layer_stride;
  const uint16_t* const vc = cache->v + layer * cache->layer_stride;
  const long long cached = static_cast<long long>(cache->n_pages) * n_kv * cache->page_size * dim;
  if (overlap(out, n_out, kc, cached) || overlap(out, n_out, vc, cached) ||
      overlap(out, n_out, cache->pages, static_cast<long long>(n_seq) * cache->pages_per_seq) ||
      overlap(out, n_out, cache->length, n_seq) || overlap(out, n_out, win_off, n_seq + 1LL) ||
      overlap(out, n_out, parent, n_tokens) ||
      overlap(out, n_out, static_cast<unsigned char*>(ws), static_cast<long long>(l.bytes)))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: out overlaps the cache, win_off, parent or the workspace", nm);
  AttnArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.kc = kc;
  a.vc = vc;
  a.pages = cache->pages;
  a.length = cache->length;
  a.win_off = win_off;
  a.parent = parent;
  a.out = out;
  unsigned char* const w = static_cast<unsigned char*>(ws);
  a.seq_plan = reinterpret_cast<int2*>(w);
  a.part_o = reinterpret_cast<float*>(w + l.plan_bytes);
  a.part_ml = reinterpret_cast<float2*>(w + l.plan_bytes + l.o_bytes);
  a.n_seq = n_seq;
  a.n_tokens = n_tokens;
  a.max_window = max_window;
  a.n_heads = n_heads;
  a.n_kv = n_kv;
  a.group = n_heads / n_kv;
  a.n_pages = cache->n_pages;
  a.page_log2 = log2_of(cache->page_size);
  a.pages_per_seq = cache->pages_per_seq;
  a.row_blocks = l.row_blocks;
  a.block_rows = l.block_rows;
  a.max_units = l.max_units;
  a.goal = l.goal;
  a.cut = l.cut;
  a.scale_log2 = scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dim == 64) return attn_launch<64>(a, s, nm);
  if (dim == 128) return attn_launch<128>(a, s, nm);
  return attn_launch<256>(a, s, nm);
}

int sg_kv_commit_f16(const uint16_t* k, const uint16_t* v, long long k_stride, long long v_stride,
                     long long k_layer_stride, long long v_layer_stride, const sg_kv_cache* cache,
                     const int* win_off, const int* path, const int* n_path, int* length_out,
                     int n_seq, int n_tokens, int max_window, void* stream) {
  const char* nm = "sg_kv_commit_f16";
  if (!path || !n_path) return sg::set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  return sg::commit(k, v, k_stride, v_stride, k_layer_stride, v_layer_stride, cache, win_off, path,
                    n_path, length_out, n_seq, n_tokens, max_window, sg::kMaxWindow, stream, nm);
}

int sg_kv_append_f16(const uint16_t* k, const uint16_t* v, long long k_stride, long long v_stride,
                     long long k_layer_stride, long long v_layer_stride, const sg_kv_cache* cache,
                     const int* win_off, int* length_out, int n_seq, int n_tokens, int max_window,
                     void* stream) {
  return sg::commit(k, v, k_stride, v_stride, k_layer_stride, v_layer_stride, cache, win_off,
                    nullptr, nullptr, length_out, n_seq, n_tokens, max_window, 0x7FFFF000, stream,
                    "sg_kv_append_f16");
}

}  // extern "C"
