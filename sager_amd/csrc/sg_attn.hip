// sg_attn.hip - the windows' attention over a paged fp16 cache, and the
// accepted tokens' way into it.
//
// For a kv head, the rows of a product are (node, query head of the group).
// A workgroup takes a block of rows and a part of a sequence's keys, 64 keys
// a step, in rows' groups of four waves:
//   S^T = K Q^T   wave w has keys 16w..16w+15 and all rows of its group (Q in
//                 registers);
//   P             goes through LDS to the group's other waves;
//   O^T = V^T P^T wave w has columns w D/4 .. of all keys.
// So K and V are read from LDS once per group, no wave holds more than a
// quarter of O, and nothing is joined at the end but the rows' sums.  With
// keys as the first product's rows, a lane of v_mfma_f32_16x16x32_f16 gets
// four consecutive keys of one query row, 8 B of P; and since the order of a
// product's 32 terms is free, V's operand is, per lane, one column of V at
// four and four consecutive keys, which ds_read_b64_tr_b16 reads from V's
// rows as they lie in memory.
//
// The running maximum is a reference point `mref` per row, common to the
// group's waves, that moves only when a score passes it by 2^15: p =
// 2^(s - mref) fits fp16 (its largest value is 2^16), and 2^(8+15) below it
// is still a normal number.  Until a score does, the waves share nothing but
// P; then all of them stop for it.  p is rounded to fp16 for the product
// (2^-11 of each weight, below the output's own rounding to fp16 once a few
// keys are averaged); l = sum p is fp32, of the unrounded p.
#include "sg_window.hpp"

namespace sg {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4* lds_s4_p;
// read through the scalar cache, whatever is stored in between
typedef const __attribute__((address_space(4))) int* const_int_p;

constexpr int kKeys = 64;          // keys of a step
constexpr float kRise = 15.f;      // log2 above mref at which mref moves
constexpr float kBelow = 8.f;      // log2 by which mref lies below the maximum it is set from
constexpr float kLog2e = 1.44269504088896340736f;

struct AttnArgs {
  const uint16_t *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  const uint16_t *kc, *vc;
  const int *pages, *length, *win_off, *parent;
  uint16_t* out;
  float* part_o;   // [split][token][head][D]
  float2* part_ml; // [split][token][head]: mref (log2), l
  int n_tokens, max_window, n_heads, n_kv, group, n_pages, page_log2, pages_per_seq;
  int n_split, split_keys, row_blocks, units;
  float scale_log2;
};

// The cached tokens of a sequence that the page table can hold.
__device__ __forceinline__ int cached_len(int length, int page_log2, int pages_per_seq) {
  const long long cap = static_cast<long long>(pages_per_seq) << page_log2;
  return static_cast<int>(length < 0 ? 0 : length > cap ? cap : length);
}

// Where chunk c (16 B) of row r lies in its row: rows are a multiple of 128 B
// apart, so 16 rows read at one chunk would share their banks.
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 64 ? (r >> 1) & 7 : r & 15;
}

// 16 B per lane from base + voff (bytes) into LDS at lds + 16 * lane.  As
// dma16 of sg_common.hpp: ordered by the kernel's own waits.
__device__ __forceinline__ void dma16_base(uint32_t lds, uint32_t voff, const void* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(base)
               : "memory");
}
__device__ __forceinline__ void dma16_ptr(uint32_t lds, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src)
               : "memory");
}

// Bytes of LDS: K and V of two steps, P, the rows' maxima and sums of the four
// waves, the nodes' ancestors, and the flags.
template <int D, int RT, int RW>
struct AttnLds {
  static constexpr uint32_t kStep = kKeys * D * 2;
  static constexpr uint32_t kRows = 16 * RT * RW;
  static constexpr uint32_t kP = 4 * kStep;
  static constexpr uint32_t kMax = kP + kRows * kKeys * 2;
  static constexpr uint32_t kSeen = kMax + 4 * kRows * 4;
  static constexpr uint32_t kFlags = kSeen + kMaxWindow * 8;
  static constexpr uint32_t kBytes = kFlags + 32;
};

// RT: tiles of 16 rows of a group; RW: groups of four waves.
template <int D, int RT, int RW>
__global__ void __launch_bounds__(256 * RW) attn_tree_kernel(const AttnArgs a) {
  typedef AttnLds<D, RT, RW> L;
  constexpr int CH = D / 8;       // 16-B chunks of a row
  constexpr int RPI = 64 / CH;    // rows of a copy instruction
  constexpr int NI = 16 / RPI;    // copy instructions of a wave's 16 keys
  constexpr int KK = D / 32;      // steps of the first product
  constexpr int DQ = D / 64;      // 16-column tiles of a wave's part of O
  constexpr int kRows = L::kRows;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds));
  int* flags = reinterpret_cast<int*>(lds + L::kFlags);  // by step parity: rise of either group, odd
  float* mx = reinterpret_cast<float*>(lds + L::kMax);
  uint64_t* seen = reinterpret_cast<uint64_t*>(lds + L::kSeen);  // node: whom it sees
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave & 3, rg = wave >> 2;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;

  // The row blocks of a unit (part, kv head, sequence) are 8 workgroups apart:
  // on one XCD, whose L2 then reads the unit's keys once.
  const int id = blockIdx.x;
  const int oct = id / (8 * a.row_blocks), in = id - oct * 8 * a.row_blocks;
  const int rb = in >> 3;
  int unit = oct * 8 + (in & 7);
  if (unit >= a.units) return;
  const int split = unit % a.n_split;
  unit /= a.n_split;
  const int h = unit % a.n_kv, seq = unit / a.n_kv;
  const Window win = window_of(a.win_off, seq, a.n_tokens, a.max_window);
  const int rows = win.n * a.group;
  if (rb * kRows >= rows) return;
  const int len = cached_len(((const_int_p)a.length)[seq], a.page_log2, a.pages_per_seq);
  const int total = len + win.n;
  const const_int_p table = (const_int_p)(a.pages + static_cast<long long>(seq) * a.pages_per_seq);
  const int steps = (total + kKeys - 1) / kKeys;
  const int per = a.split_keys / kKeys;
  const long long first = static_cast<long long>(split) * per;
  const int s_end = split == a.n_split - 1 || first + per > steps ? steps
                                                                  : static_cast<int>(first + per);
  int step = first < s_end ? static_cast<int>(first) : s_end;

  // ---- copies: wave kw brings keys 16 kw.. of a step (of two groups, the
  // first brings V's, the second K's) ----
  const uint32_t blk = kw * 16 * D * 2;
  auto page_of = [&](int s) {
    const int j = s * kKeys + 16 * kw;
    return j < len ? table[j >> a.page_log2] : -1;
  };
  auto page_ok = [&](int p) { return static_cast<uint32_t>(p) < static_cast<uint32_t>(a.n_pages); };
  // Brings a step's K and V; with two groups, V or K.
  auto issue = [&](int s, int page, bool v) {
    const int j = s * kKeys + 16 * kw;
    const uint32_t buf = lds0 + (s & 1) * 2 * L::kStep + blk + (RW == 2 && v ? L::kStep : 0);
    const long long at =
        (((static_cast<long long>(page) * a.n_kv + h) << a.page_log2) +
         (j & ((1 << a.page_log2) - 1))) * D;
    const uint16_t* const c1 = RW == 2 && v ? a.vc : a.kc;
    if (j + 16 <= len && page_ok(page)) {
      const uint16_t* b1 = uniform_ptr(c1 + at);
      const uint16_t* b2 = uniform_ptr(a.vc + at);
      int ln = lane;
      if (RT >= 3) asm("" : "+v"(ln));  // (the offsets made anew: registers are short)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + ln / CH;
        const uint32_t off = row * (D * 2) + (((ln % CH) ^ swz<D>(row)) << 4);
        dma16_base(buf + i * 1024, off, b1);
        if (RW == 1) dma16_base(buf + L::kStep + i * 1024, off, b2);
      }
    } else if (j < total) {
      // rows of the cache, then of the window; what is not there reads a
      // window row and is masked
      const int n_cache = page_ok(page) ? min(len - j, 16) : 0;
      const uint16_t* const w1 = RW == 2 && v ? a.v : a.k;
      const long long ws1 = RW == 2 && v ? a.v_stride : a.k_stride;
#pragma unroll 1
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + lane / CH;
        const int c = ((lane % CH) ^ swz<D>(row)) * 8;
        const long long w = win.off + min(max(j + row - len, 0), win.n - 1);
        const bool cached = row < n_cache;
        dma16_ptr(buf + i * 1024, (cached ? c1 + at + row * D : w1 + w * ws1 + h * D) + c);
        if (RW == 1)
          dma16_ptr(buf + L::kStep + i * 1024,
                    (cached ? a.vc + at + row * D : a.v + w * a.v_stride + h * D) + c);
      }
    }
  };
  // bit r: key 16 kw + r of the step is there
  auto present = [&](int s, int page) {
    const int j = s * kKeys + 16 * kw;
    const int nc = min(max(len - j, 0), 16), nw = min(max(total - j, 0), 16);
    const uint32_t c = (1u << nc) - 1;
    return ((1u << nw) - 1) & (page_ok(page) ? 0xFFFFu : ~c);
  };

  int page = page_of(step), page_next = 0;
  if (step < s_end) {
    issue(step, page, rg == 0);
    page_next = page_of(step + 1);
  }
  if (threadIdx.x < 8) flags[threadIdx.x] = 0;

  // ---- Q's rows, while the first copies are under way ----
  if (wave == 4 * RW - 1) seen[lane] = ancestors(a.parent, win, lane);
  const int row0 = rb * kRows + rg * 16 * RT;
  auto node_of = [&](int rt) { return min(row0 + rt * 16 + col, rows - 1) / a.group; };
  h8 qf[RT][KK];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = min(row0 + rt * 16 + col, rows - 1);  // (a row past the end repeats the last)
    const int node = r / a.group, g = r - node * a.group;
    const uint16_t* qp = a.q + static_cast<long long>(win.off + node) * a.q_stride +
                         (h * a.group + g) * D;
#pragma unroll
    for (int s = 0; s < KK; ++s) {
      const u32x4 w = *reinterpret_cast<const u32x4_u*>(qp + s * 32 + grp * 8);
      qf[rt][s] = __builtin_bit_cast(h8, w);
    }
  }

  f4 acc[RT][DQ];
  float mref[RT], l[RT];
  bool begun[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    mref[rt] = 0.f;
    l[rt] = 0.f;
    begun[rt] = false;
#pragma unroll
    for (int d = 0; d < DQ; ++d) acc[rt][d] = (f4){0.f, 0.f, 0.f, 0.f};
  }
  // P: [row][two halves of 32 keys][grp][two blocks of 16 keys][4], 16-B pieces
  // swizzled over the row's eight
  unsigned char* const pl = lds + L::kP + rg * 16 * RT * 128;
  const int psw = (col >> 1) & 7;
  // K's pieces st * 4 + grp of row col, swizzled: four offsets, the rest is added.  V's: columns
  // kw D/4 + 16 d.. of row 4 grp + col / 4 of a 16-key block.
  constexpr int KO = KK < 4 ? KK : 4;
  uint32_t koff[KO], voff[DQ];
#pragma unroll
  for (int i = 0; i < KO; ++i)
    koff[i] = blk + col * (D * 2) + (((i * 4) ^ grp ^ swz<D>(col)) << 4);
#pragma unroll
  for (int d = 0; d < DQ; ++d)
    voff[d] = lds0 + L::kStep + (4 * grp + (col >> 2)) * (D * 2) +
              (((2 * d) ^ (kw * (CH / 4) + ((col & 3) >> 1)) ^ swz<D>(4 * grp + (col >> 2))) << 4) +
              (col & 1) * 8;
  unsigned char* const p_out = pl + col * 128 + ((((kw >> 1) * 4 + grp) ^ psw) << 4) + (kw & 1) * 8;

  // Rows of V that nobody sees become 0 (0 times what lies there need not be
  // 0).  Window rows, which some queries see and others do not, are looked
  // through for infinities and NaN.  Each wave does the rows it has copied.
  auto fix_v = [&](int s, uint32_t there) {
    const int j = s * kKeys + 16 * kw;
    unsigned char* vb = lds + (s & 1) * 2 * L::kStep + L::kStep + blk;
    bool odd = false;
#pragma unroll 1
    for (int i = 0; i < NI; ++i) {
      const int row = i * RPI + lane / CH;
      u32x4* at = reinterpret_cast<u32x4*>(vb + i * 1024 + 16 * lane);
      if (!(there >> row & 1)) {
        *at = (u32x4){0, 0, 0, 0};
      } else if (j + row >= len && win.n > 1) {
        const u32x4 w = *at;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          odd |= (w[c] & 0x7C00u) == 0x7C00u || (w[c] & 0x7C000000u) == 0x7C000000u;
      }
    }
    if (__any(odd) && lane == 0) flags[4 + (s & 1)] = 1;
  };
  auto plain_step = [&](int s, uint32_t there) {
    return s * kKeys + 16 * kw + 16 <= len && there == 0xFFFFu;
  };

  float e[RT][4], top[RT], sum[RT];
  // e: the scores of a step's keys 16 kw.. above mref, log2; top: their largest per row
  auto scores = [&](int step_, uint32_t there, bool plain) {
    const unsigned char* kb = lds + (step_ & 1) * 2 * L::kStep;
    f4 s[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < KK; ++st) {
      const h8 kf = *reinterpret_cast<const h8*>(kb + koff[st % KO] + st / KO * 256);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        s[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][st], s[rt], 0, 0, 0);
      if (RW == 2 && st % 4 == 3) asm volatile("" ::: "memory");  // (no more reads ahead: registers)
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[rt][i] = __builtin_fmaf(s[rt][i], a.scale_log2, -mref[rt]);
      if (!plain) {
        // bit r of `see`: key r is there and this lane's row sees it
        const uint64_t up = seen[node_of(rt)];
        const int w0 = step_ * kKeys + 16 * kw - len;  // key 0's window node, if not negative
        const uint32_t tree = w0 >= 0    ? static_cast<uint32_t>(up >> (w0 & 63))
                              : w0 > -16 ? static_cast<uint32_t>(up << -w0) | ((1u << -w0) - 1)
                                         : 0xFFFFu;
        const uint32_t see = (there & tree) >> (4 * grp);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[rt][i] = see & 1u << i ? e[rt][i] : -INFINITY;
      }
      top[rt] = fmaxf(fmaxf(e[rt][0], e[rt][1]), fmaxf(e[rt][2], e[rt][3]));
    }
  };
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
  auto first_part = [&](int* rise_flag) {  // after scores()
    bool rise = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      rise |= top[rt] > kRise || (!begun[rt] && top[rt] > -INFINITY);
      weigh(rt, 0.f);
    }
    if (__any(rise) && lane == 0) *rise_flag = 1;
  };
  // The reference points move: the rows' maxima over the group's waves, then P
  // once more.  Every wave of the workgroup comes to the two barriers.
  auto move_refs = [&](bool mine) {
    if (mine)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float m = fmaxf(top[rt], __shfl_xor(top[rt], 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        if (grp == 0) mx[kw * kRows + (rg * RT + rt) * 16 + col] = m;
      }
    bar();
    if (mine)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float* mr = mx + (rg * RT + rt) * 16 + col;
        const float m = fmaxf(fmaxf(mr[0], mr[kRows]), fmaxf(mr[2 * kRows], mr[3 * kRows]));
        const bool set = m > kRise || (!begun[rt] && m > -INFINITY);
        const float by = set ? m - kBelow : 0.f;
        const float f = !set ? 1.f : begun[rt] ? __builtin_amdgcn_exp2f(-by) : 0.f;
        mref[rt] += by;
        l[rt] *= f;
#pragma unroll
        for (int d = 0; d < DQ; ++d) acc[rt][d] *= f;
        begun[rt] |= set;
        weigh(rt, by);
      }
    bar();
  };
  auto second_part = [&](int s) {
    const unsigned char* vb = lds + (s & 1) * 2 * L::kStep + L::kStep;
    const bool odd = flags[4 + (s & 1)] != 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] += sum[rt];
    if (odd) {
      // Infinities and NaN in the window's V: added one by one to the rows
      // that see them, and taken as 0 below.
#pragma unroll 1
      for (int r = 0; r < kKeys; ++r) {
        const int node = s * kKeys + r - len;
        if (node < 0 || node >= win.n) continue;
        const int piece = (r >> 5) * 4 + ((r & 15) >> 2);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float w = half_bits_to_float(*reinterpret_cast<const uint16_t*>(
              pl + (rt * 16 + col) * 128 + ((piece ^ psw) << 4) + (r >> 4 & 1) * 8 + (r & 3) * 2));
          const bool see = seen[node_of(rt)] >> node & 1;
#pragma unroll
          for (int d = 0; d < DQ; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int c = kw * (D / 4) + d * 16 + 4 * grp + i;
              const uint16_t b = *reinterpret_cast<const uint16_t*>(
                  vb + r * (D * 2) + (((c >> 3) ^ swz<D>(r)) << 4) + (c & 7) * 2);
              acc[rt][d][i] += see && (b & 0x7C00) == 0x7C00 ? w * half_bits_to_float(b) : 0.f;
            }
        }
      }
    }
    const uint32_t vl = (s & 1) * 2 * L::kStep;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      h8 pf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        pf[rt] = *reinterpret_cast<const h8*>(pl + (rt * 16 + col) * 128 +
                                              (((st * 4 + grp) ^ psw) << 4));
#pragma unroll
      for (int d = 0; d < DQ; ++d) {
        s4 x[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          x[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_p)(static_cast<uintptr_t>(
              vl + voff[d] + (st * 2 + b) * 16 * D * 2)));
          if (odd) {
            const int j = s * kKeys + (st * 2 + b) * 16 + 4 * grp;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[b][i] = j + i >= len && (x[b][i] & 0x7C00) == 0x7C00 ? 0 : x[b][i];
          }
        }
        const h8 vf = __builtin_bit_cast(
            h8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt], acc[rt][d], 0, 0, 0);
      }
      if (RW == 2) asm volatile("" ::: "memory");
    }
  };

  bar();  // the flags are cleared
  if (RW == 1) {
    for (; step < s_end; ++step) {
      const int par = step & 1;
      const uint32_t there = present(step, page);
      wait_vm();
      if (!plain_step(step, there)) fix_v(step, there);
      bar();  // everybody's copies of this step are here, and nobody reads the other buffers or P
      if (step + 1 < s_end) issue(step + 1, page_next, false);
      const int page_then = step + 2 < s_end ? page_of(step + 2) : -1;
      if (threadIdx.x == 0) flags[par ^ 1] = flags[4 + (par ^ 1)] = 0;
      scores(step, there, plain_step(step, there));
      first_part(flags + par);
      bar();  // P is here
      if (flags[par]) move_refs(true);
      second_part(step);
      page = page_next;
      page_next = page_then;
    }
  } else {
    // Two groups half a step apart: while one takes a step's first part
    // (scores and weights), the other takes the second part of the step before
    // and brings the next step's copies, since the first part is the longer
    // way: K in even halves (the second group), V in odd ones (the first).  In
    // half t, group t & 1 takes the first part of step t / 2, the other the
    // second part of step (t - 1) / 2.
    const int n = s_end - step, begin = step;
    uint32_t there = 0, there_before = 0;
#pragma unroll 1
    for (int t = 0; t <= 2 * n; ++t) {
      const int who = t & 1, s1 = begin + (t >> 1), s2 = begin + ((t - 1) >> 1);
      const bool lead = who == rg, more = s1 < s_end;
      if (who == 0) {
        there_before = there;
        there = present(s1, page);
      }
      if (!lead && more) {
        wait_vm();
        if (who == 1 && !plain_step(s1, there)) fix_v(s1, there);
      }
      bar();  // K (V) of s1 is here, and the other group's P
      const int moved = t > 0 ? flags[2 * (who ^ 1) + (s2 & 1)] : 0;
      if (lead) {
        if (more) scores(s1, there, plain_step(s1, there));
        if (moved) move_refs(false);
        if (more) first_part(flags + 2 * who + (s1 & 1));
      } else {
        if (moved) {  // (K of s2 is still there)
          scores(s2, who ? there : there_before, false);
          move_refs(true);
        }
        if (s1 + 1 < s_end) issue(s1 + 1, page_next, who == 1);
        if (t > 0) second_part(s2);
      }
      if (threadIdx.x == 0) {
        flags[2 * who + ((s1 & 1) ^ 1)] = 0;
        if (who == 1) flags[4 + ((s1 & 1) ^ 1)] = 0;
      }
      if (who == 1) {
        page = page_next;
        if (s1 + 2 < s_end) page_next = page_of(s1 + 2);
      }
    }
  }

  // ---- the rows' sums over the group's waves, and out ----
  bar();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    if (grp == 0) mx[kw * kRows + (rg * RT + rt) * 16 + col] = l[rt];
  }
  bar();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + col;
    const float* lr = mx + (rg * RT + rt) * 16 + col;
    float lt = (lr[0] + lr[kRows]) + (lr[2 * kRows] + lr[3 * kRows]);
    if (!seen[node_of(rt)]) lt = 0.f;  // an absent node
    if (r < rows) {
      const int node = r / a.group, g = r - node * a.group;
      const long long at = static_cast<long long>(win.off + node) * a.n_heads + h * a.group + g;
      const int c0 = kw * (D / 4) + 4 * grp;
      if (a.n_split == 1) {
        const float inv = lt != 0.f ? 1.f / lt : 0.f;
#pragma unroll
        for (int d = 0; d < DQ; ++d) {
          h4 y;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[i] = lt != 0.f ? static_cast<_Float16>(acc[rt][d][i] * inv) : static_cast<_Float16>(0);
          *reinterpret_cast<h4*>(a.out + at * D + c0 + d * 16) = y;
        }
      } else {
        const long long pa = static_cast<long long>(split) * a.n_tokens * a.n_heads + at;
#pragma unroll
        for (int d = 0; d < DQ; ++d)
          *reinterpret_cast<f4*>(a.part_o + pa * D + c0 + d * 16) = acc[rt][d];
        if (kw == 0 && grp == 0) a.part_ml[pa] = make_float2(mref[rt], lt);
      }
    }
  }
}

// The parts of a row's keys, joined: a workgroup per (token, head), each
// wave's 16-B lanes taking whole parts in turn.  A part whose l is 0 has no
// key that the row sees, and what its O holds is not read as a number.
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
  constexpr int LP = D / 4;        // lanes of a part
  constexpr int SP = 256 / LP;     // parts at once
  constexpr int U = 8;             // loads under way per lane
  const int per = a.max_window * a.n_heads;
  const int seq = blockIdx.x / per;
  const int rest = blockIdx.x - seq * per;
  const int node = rest / a.n_heads, head = rest - node * a.n_heads;
  const Window w = window_of(a.win_off, seq, a.n_tokens, a.max_window);
  if (node >= w.n) return;
  const long long at = static_cast<long long>(w.off + node) * a.n_heads + head;
  const long long step = static_cast<long long>(a.n_tokens) * a.n_heads;
  const int t = threadIdx.x, sub = t / LP, c = (t % LP) * 4;
  const float* po = a.part_o + at * D + c;
  // every lane group joins its parts about a maximum of its own
  float m = -INFINITY, sum = 0.f;
  f4 o = (f4){0.f, 0.f, 0.f, 0.f};
  for (int s0 = sub; s0 < a.n_split; s0 += SP * U) {
    f4 v[U];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u * SP, a.n_split - 1);
      ml[u] = a.part_ml[at + s * step];
      v[u] = *reinterpret_cast<const f4*>(po + s * step * D);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * SP >= a.n_split) ml[u].y = 0.f;
      top = ml[u].y != 0.f ? fmaxf(top, ml[u].x) : top;
    }
    const float f0 = m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 0.f;
    sum *= f0;
    o *= f0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool some = ml[u].y != 0.f;
      const float f = some ? __builtin_amdgcn_exp2f(ml[u].x - top) : 0.f;
      sum += some ? ml[u].y * f : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += some ? v[u][i] * f : 0.f;
    }
    m = top;
  }
  __shared__ f4 so[256];
  __shared__ float sm[SP], ss[SP];
  so[t] = o;
  if (t % LP == 0) {
    sm[sub] = m;
    ss[sub] = sum;
  }
  __syncthreads();
  if (sub == 0) {
    float top = sm[0];
#pragma unroll
    for (int i = 1; i < SP; ++i) top = fmaxf(top, sm[i]);
    float total = 0.f;
    f4 y = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SP; ++i) {
      const bool some = ss[i] != 0.f;
      const float f = some ? __builtin_amdgcn_exp2f(sm[i] - top) : 0.f;
      total += some ? ss[i] * f : 0.f;
      const f4 x = so[i * LP + t];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] += some ? x[j] * f : 0.f;
    }
    const float inv = total != 0.f ? 1.f / total : 0.f;
    h4 z;
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = static_cast<_Float16>(y[j] * inv);
    *reinterpret_cast<h4*>(a.out + at * D + c) = z;
  }
}

// ---- the accepted tokens into the cache --------------------------------------
struct CommitArgs {
  const uint16_t *k, *v;
  long long k_stride, v_stride, k_layer, v_layer, layer_stride;
  uint16_t *kc, *vc;
  const int *pages, *length, *win_off, *path, *n_path;
  int* length_out;
  int n_tokens, max_window, n_kv, dim, n_pages, page_log2, pages_per_seq;
};

// Grid: (16-B pieces of a window's K and V rows, sequence, layer).
__global__ void __launch_bounds__(256) kv_commit_kernel(const CommitArgs a) {
  const int s = blockIdx.y, layer = blockIdx.z;
  const Window w = window_of(a.win_off, s, a.n_tokens, a.max_window);
  const int n = min(max(a.n_path[s], 0), a.max_window);
  const int len = a.length[s];
  if (a.length_out && blockIdx.x == 0 && layer == 0 && threadIdx.x == 0) a.length_out[s] = len + n;
  const int pieces = a.n_kv * (a.dim / 8);
  int x = blockIdx.x * 256 + threadIdx.x;
  const bool is_v = x & 1;  // K's and V's piece of one place by neighbours: both tables' pages once
  x >>= 1;
  const int i = x / pieces;
  if (i >= n) return;
  x -= i * pieces;
  const int h = x / (a.dim / 8), c = x - h * (a.dim / 8);
  const int node = a.path[static_cast<long long>(s) * a.max_window + i];
  const long long pos = static_cast<long long>(len) + i;
  if (len < 0 || node < 0 || node >= w.n || pos >> a.page_log2 >= a.pages_per_seq) return;
  const int page = a.pages[static_cast<long long>(s) * a.pages_per_seq + (pos >> a.page_log2)];
  if (page < 0 || page >= a.n_pages) return;
  const uint16_t* src = (is_v ? a.v + layer * a.v_layer + (w.off + node) * a.v_stride
                              : a.k + layer * a.k_layer + (w.off + node) * a.k_stride) +
                        h * a.dim + c * 8;
  const long long slot = ((static_cast<long long>(page) * a.n_kv + h) << a.page_log2) +
                         (pos & ((1 << a.page_log2) - 1));
  uint16_t* dst = (is_v ? a.vc : a.kc) + layer * a.layer_stride + slot * a.dim + c * 8;
  *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4_u*>(src);
}

// ---- host -----------------------------------------------------------------------

static int log2_of(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

static int check_cache(const sg_kv_cache* c, int n_seq, int n_tokens, int max_window,
                       const char* nm) {
  if (!c || !c->k || !c->v || !c->pages || !c->length)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null cache", nm);
  if (n_seq <= 0 || n_tokens <= 0 || max_window <= 0 || c->n_layers <= 0 || c->n_pages <= 0 ||
      c->pages_per_seq <= 0 || c->n_kv_heads <= 0)
    return set_error(SG_ERR_GEOMETRY,
                     "%s: n_seq=%d n_tokens=%d max_window=%d n_layers=%d n_pages=%d "
                     "pages_per_seq=%d n_kv_heads=%d must be positive",
                     nm, n_seq, n_tokens, max_window, c->n_layers, c->n_pages, c->pages_per_seq,
                     c->n_kv_heads);
  if (max_window > kMaxWindow)
    return set_error(SG_ERR_UNSUPPORTED, "%s: max_window=%d is over %d", nm, max_window,
                     kMaxWindow);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return set_error(SG_ERR_UNSUPPORTED, "%s: head_dim=%d is not 64, 128 or 256", nm, c->head_dim);
  if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) != 0)
    return set_error(SG_ERR_UNSUPPORTED, "%s: page_size=%d is no power of two from 16 on", nm,
                     c->page_size);
  // token positions are 32-bit
  if ((static_cast<long long>(c->pages_per_seq) << log2_of(c->page_size)) > 0x7FFFF000LL)
    return set_error(SG_ERR_UNSUPPORTED, "%s: a sequence of %d pages of %d tokens is too long", nm,
                     c->pages_per_seq, c->page_size);
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 ||
      c->layer_stride % 8)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: the cache is not 16-B aligned", nm);
  return SG_OK;
}

// How a call is cut: rows of a workgroup, parts of the caches.
struct Cut {
  int rt, rw, row_blocks, n_split, split_keys;
};
static Cut attn_cut(int n_seq, int max_window, int max_len, int group, int n_kv, int dim) {
  Cut c;
  const long long rows = static_cast<long long>(max_window) * group;
  c.rt = rows > 32 ? 4 : rows > 16 ? 2 : 1;
  c.rw = rows > 64 ? 2 : 1;
  if (c.rw == 2 && dim == 256) c.rt = 2;
  c.row_blocks = static_cast<int>((rows + 16 * c.rt * c.rw - 1) / (16 * c.rt * c.rw));
  const long long keys = static_cast<long long>(max_len) + max_window;
  const long long most = (keys + kKeys - 1) / kKeys;
  const long long units = static_cast<long long>(n_seq) * n_kv * c.row_blocks;
  const long long slots = 256 * (dim == 256 || c.rw == 2 ? 1 : 2);
  long long n = units >= slots ? 1 : slots / units;
  if (n > most) n = most;
  c.split_keys = static_cast<int>((most + n - 1) / n * kKeys);
  c.n_split = static_cast<int>((keys + c.split_keys - 1) / c.split_keys);
  return c;
}
static size_t part_bytes(const Cut& c, int n_tokens, int n_heads, int dim) {
  if (c.n_split == 1) return 0;
  return static_cast<size_t>(c.n_split) * n_tokens * n_heads * (dim * 4 + 8);
}

template <int D, int RT, int RW>
static void attn_go(const AttnArgs& a, long long grid, hipStream_t s) {
  hipLaunchKernelGGL((attn_tree_kernel<D, RT, RW>), dim3(static_cast<unsigned>(grid)),
                     dim3(256 * RW), (AttnLds<D, RT, RW>::kBytes), s, a);
}
template <int D>
static int attn_launch(const AttnArgs& a, const Cut& c, int n_seq, hipStream_t s, const char* nm) {
  const long long grid = (a.units + 7LL) / 8 * 8 * c.row_blocks;
  if (c.rw == 2)
    attn_go<D, D == 256 ? 2 : 4, 2>(a, grid, s);
  else if (c.rt == 4)
    attn_go<D, 4, 1>(a, grid, s);
  else if (c.rt == 2)
    attn_go<D, 2, 1>(a, grid, s);
  else
    attn_go<D, 1, 1>(a, grid, s);
  if (int st = check_launch(nm)) return st;
  if (c.n_split > 1) {
    hipLaunchKernelGGL(attn_join_kernel<D>, dim3(n_seq * a.max_window * a.n_heads), dim3(256), 0, s,
                       a);
    return check_launch(nm);
  }
  return SG_OK;
}

}  // namespace sg

extern "C" {

size_t sg_attn_tree_workspace_bytes(int n_seq, int n_tokens, int max_window, int max_len,
                                    int n_heads, int n_kv_heads, int head_dim) {
  if (n_seq <= 0 || n_tokens <= 0 || max_window <= 0 || max_len < 0 || n_kv_heads <= 0 ||
      n_heads <= 0 || n_heads % n_kv_heads != 0)
    return 0;
  // enough for every smaller batch too: fewer sequences are cut into more parts
  size_t most = 0;
  for (int s = 1; s <= n_seq; ++s) {
    const sg::Cut c =
        sg::attn_cut(s, max_window, max_len, n_heads / n_kv_heads, n_kv_heads, head_dim);
    const size_t b = sg::part_bytes(c, n_tokens, n_heads, head_dim);
    if (b > most) most = b;
    if (c.n_split == 1) break;
  }
  return most;
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
  const Cut c = attn_cut(n_seq, max_window, max_len, n_heads / n_kv, n_kv, dim);
  const size_t need = part_bytes(c, n_tokens, n_heads, dim);
  if (need && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16))
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: the workspace needs %zu bytes, 16-B aligned", nm,
                     need);
  const long long units = static_cast<long long>(n_seq) * n_kv * c.n_split;
  const long long join = static_cast<long long>(n_seq) * max_window * n_heads;
  if ((units + 8) * c.row_blocks > 0x7FFFFFFF || join > 0x7FFFFFFF)
    return set_error(SG_ERR_UNSUPPORTED, "%s: too many sequences", nm);
  AttnArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.kc = cache->k + layer * cache->layer_stride;
  a.vc = cache->v + layer * cache->layer_stride;
  a.pages = cache->pages;
  a.length = cache->length;
  a.win_off = win_off;
  a.parent = parent;
  a.out = out;
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(
      a.part_o + static_cast<size_t>(c.n_split) * n_tokens * n_heads * dim);
  a.n_tokens = n_tokens;
  a.max_window = max_window;
  a.n_heads = n_heads;
  a.n_kv = n_kv;
  a.group = n_heads / n_kv;
  a.n_pages = cache->n_pages;
  a.page_log2 = log2_of(cache->page_size);
  a.pages_per_seq = cache->pages_per_seq;
  a.n_split = c.n_split;
  a.split_keys = c.split_keys;
  a.row_blocks = c.row_blocks;
  a.units = static_cast<int>(units);
  a.scale_log2 = scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dim == 64) return attn_launch<64>(a, c, n_seq, s, nm);
  if (dim == 128) return attn_launch<128>(a, c, n_seq, s, nm);
  return attn_launch<256>(a, c, n_seq, s, nm);
}

int sg_kv_commit_f16(const uint16_t* k, const uint16_t* v, long long k_stride, long long v_stride,
                     long long k_layer_stride, long long v_layer_stride, const sg_kv_cache* cache,
                     const int* win_off, const int* path, const int* n_path, int* length_out,
                     int n_seq, int n_tokens, int max_window, void* stream) {
  const char* nm = "sg_kv_commit_f16";
  using namespace sg;
  if (!k || !v || !win_off || !path || !n_path)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (int st = check_cache(cache, n_seq, n_tokens, max_window, nm)) return st;
  if (length_out == cache->length)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: length_out is the cache's own length", nm);
  const long long row = static_cast<long long>(cache->n_kv_heads) * cache->head_dim;
  if (k_stride < row || v_stride < row)
    return set_error(SG_ERR_GEOMETRY, "%s: a token stride is less than a token", nm);
  if (reinterpret_cast<uintptr_t>(k) % 2 || reinterpret_cast<uintptr_t>(v) % 2)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: k and v must be 2-B aligned", nm);
  const long long pieces = 2LL * max_window * (row / 8);
  if (n_seq > 65535 || cache->n_layers > 65535 || pieces > 0x7FFFFFFF - 256)
    return set_error(SG_ERR_UNSUPPORTED, "%s: n_seq=%d n_layers=%d n_kv_heads=%d", nm, n_seq,
                     cache->n_layers, cache->n_kv_heads);
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
  a.n_kv = cache->n_kv_heads;
  a.dim = cache->head_dim;
  a.n_pages = cache->n_pages;
  a.page_log2 = log2_of(cache->page_size);
  a.pages_per_seq = cache->pages_per_seq;
  hipLaunchKernelGGL(kv_commit_kernel,
                     dim3(static_cast<unsigned>((pieces + 255) / 256), n_seq, cache->n_layers),
                     dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return check_launch(nm);
}

}  // extern "C"
