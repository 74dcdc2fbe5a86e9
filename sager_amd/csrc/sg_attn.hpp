// sg_attn.hpp - what the attentions over a paged cache share: how a batch is
// cut into units, K's and V's steps in LDS, the operands read from there, and
// the join of a row's parts.
#pragma once

#include "sg_cache.hpp"

namespace sg {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4* lds_s4_p;
typedef __attribute__((address_space(3))) unsigned char* lds_char_p;
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
  // Parts of cut units, by unit, row block and row: O, and mref (log2) and l.
  // seq_plan: per sequence its first unit and the parts of its units.
  float* part_o;
  float2* part_ml;
  int2* seq_plan;
  int n_tokens, max_window, n_heads, n_kv, group, n_pages, page_log2, pages_per_seq;
  int n_seq, row_blocks, block_rows, max_units, goal;
  bool cut;
  float scale_log2;
};

// The arguments once more from where the launch put them, for paths taken now
// and then: what only they need then holds no scalar registers between.
typedef const __attribute__((address_space(4))) AttnArgs* kernarg_p;
__device__ __forceinline__ kernarg_p cold_args() {
  kernarg_p p = (kernarg_p)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// The cached tokens of a sequence that the page table can hold.
__device__ __forceinline__ int cached_len(int length, int page_log2, int pages_per_seq) {
  const long long cap = static_cast<long long>(pages_per_seq) << page_log2;
  return static_cast<int>(length < 0 ? 0 : length > cap ? cap : length);
}

// How a batch is cut, from the caches' lengths, which only the device knows.
// A unit is a part of a sequence's keys for one kv head; a sequence's steps of
// 64 keys are cut into parts of `part` steps: `goal` of them if they came out
// even, and up to 64 sequences more a part until the units are no more than
// max_units, so that the units of a ragged batch are equally long and the
// launch ends in one round.  Every wave finds this by itself: a sequence a
// lane, the sum, a few guesses at `part`, the running sum.
__device__ __forceinline__ int parts_of(int steps, int part) {
  // (fp32: a part more or less changes nothing, the last one takes what is left)
  const float inv = __builtin_amdgcn_rcpf(static_cast<float>(part));
  return steps > 0 ? max(1, static_cast<int>(ceilf(static_cast<float>(steps) * inv))) : 0;
}
__device__ __forceinline__ int steps_of(const AttnArgs& a, int seq, int* len, Window* win) {
  if (seq >= a.n_seq) return 0;
  *win = window_of(a.win_off, seq, a.n_tokens, a.max_window);
  *len = cached_len(a.length[seq], a.page_log2, a.pages_per_seq);
  return win->n > 0 ? (*len + win->n + kKeys - 1) / kKeys : 0;
}
__device__ __forceinline__ int wave_run_sum_i(int v) {  // lane l: of lanes 0..l
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}
struct Unit {
  int seq, h, k, parts, part;  // part k of `parts`, `part` steps each
  int len, steps;
  Window win;
};
// Finds unit `unit`; false if there is none.  plan: leaves the plan for the join.
// (A: whose steps_of counts a sequence's steps)
template <class A>
__device__ __forceinline__ bool find_unit(const A& a, int unit, int lane, bool plan, Unit& u) {
  int len = 0;
  Window win{0, 0};
  int steps = steps_of(a, lane, &len, &win);
  int part = 0x7FFFFFFF;
  if (a.cut) {
    long long sum = __builtin_amdgcn_readlane(wave_run_sum_i(steps), 63);
    const int n_seq = a.n_seq;
    for (int s = lane + 64; s - lane < n_seq; s += 64) {
      int l;
      Window w;
      sum += __builtin_amdgcn_readlane(wave_run_sum_i(steps_of(a, s, &l, &w)), 63);
    }
    part = max(1, static_cast<int>(min((sum * a.n_kv + a.goal - 1) / a.goal, 0x7FFFFFFFLL)));
    if (n_seq <= 64)
      while (__builtin_amdgcn_readlane(wave_run_sum_i(parts_of(steps, part)), 63) * a.n_kv >
             a.max_units)
        part += max(1, part >> 3);
  }
  int base = 0;
  bool found = false;
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    if (s0 > 0) steps = steps_of(a, s0 + lane, &len, &win);
    const int n = a.cut ? parts_of(steps, part) : steps > 0;
    const int run = wave_run_sum_i(n) * a.n_kv;  // units up to this sequence's end
    if (plan && s0 + lane < a.n_seq) a.seq_plan[s0 + lane] = make_int2(base + run - n * a.n_kv, n);
    const uint64_t past = __ballot(base + run > unit);
    if (past && !found) {
      const int l = __builtin_ctzll(past);
      found = true;
      u.seq = s0 + l;
      u.parts = __builtin_amdgcn_readlane(n, l);
      const int in = unit - (base + __builtin_amdgcn_readlane(run, l) - u.parts * a.n_kv);
      u.h = in / u.parts;
      u.k = in - u.h * u.parts;
      u.part = part;
      u.len = __builtin_amdgcn_readlane(len, l);
      u.steps = __builtin_amdgcn_readlane(steps, l);
      u.win.off = __builtin_amdgcn_readlane(win.off, l);
      u.win.n = __builtin_amdgcn_readlane(win.n, l);
      if (!plan) break;
    }
    base += __builtin_amdgcn_readlane(run, 63);
  }
  return found;
}

// Where chunk c (16 B) of row r lies in its row: at c ^ swz(r), linear in r's
// bits.  Rows are a multiple of 128 B apart; K's reads (16 rows at a chunk,
// the next four lanes' rows at the next) and V's (eight rows at a pair of
// chunks) find no bank twice, whichever quarter or half of the wave goes
// together.  (With rows r and r + 8 in one pair of chunks a third of the LDS'
// cycles were conflicts.)
template <int D>
__device__ __forceinline__ int swz(int r) {
  const int up = r >> 3 & 1;
  return D == 64 ? ((r & 6) ^ up << 2) | up : ((r & 7) << 1 ^ up << 3) | up;
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
// The larger of three, a NaN passed over (fmaxf twice, without the
// canonicalization of its arguments that the compiler adds).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ bool fp16_odd(uint32_t b) { return (b & 0x7C00) == 0x7C00; }

// What both kernels know of their part of the work.  K and V of step s lie at
// (s & 1) * 2 kStep and kStep after it, 64 rows of D values each, their 16-B
// chunks at chunk ^ swz(row).
template <int D>
struct Part {
  static constexpr int CH = D / 8;       // 16-B chunks of a row
  static constexpr int RPI = 64 / CH;    // rows of a copy instruction
  static constexpr int NI = 16 / RPI;    // copy instructions of 16 keys
  static constexpr int KK = D / 32;      // steps of the first product
  static constexpr int KO = KK < 4 ? KK : 4;
  static constexpr uint32_t kStep = kKeys * D * 2;

  const AttnArgs& a;
  int lane, col, grp;
  int unit, parts, rb, h;
  Window win;
  int rows, len, total;  // rows of the window; cached keys, cached and window's
  int begin, end;        // steps
  const_int_p table;
  unsigned char* lds;
  uint32_t lds0;

  // The row blocks of a unit are 8 workgroups apart: on one XCD, whose L2 then
  // reads the unit's keys once.
  __device__ __forceinline__ bool start(unsigned char* l) {
    lds = l;
    lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char_p)l));
    lane = threadIdx.x & 63;
    col = lane & 15;
    grp = lane >> 4;
    const int id = blockIdx.x;
    const int oct = id / (8 * a.row_blocks), in = id - oct * 8 * a.row_blocks;
    rb = in >> 3;
    unit = oct * 8 + (in & 7);
    Unit u;
    const bool plan = a.cut && id == 0 && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) == 0;
    if (!find_unit(a, unit, lane, plan, u)) return false;
    auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // (the same in every lane)
    h = one(u.h);
    parts = one(u.parts);
    win = Window{one(u.win.off), one(u.win.n)};
    rows = win.n * a.group;
    if (rb * a.block_rows >= rows) return false;
    len = one(u.len);
    total = len + win.n;
    table = (const_int_p)(a.pages + static_cast<long long>(one(u.seq)) * a.pages_per_seq);
    const int k = one(u.k), part = one(u.part), steps = one(u.steps);
    const long long first = static_cast<long long>(k) * part;
    begin = first < steps ? static_cast<int>(first) : steps;
    end = k == parts - 1 || first + part > steps ? steps : static_cast<int>(first + part);
    return true;
  }
  // The page of keys 16 b.. of step s (pages hold a multiple of 16 keys).
  __device__ __forceinline__ int page_of(int s, int b) const {
    const int j = s * kKeys + 16 * b;
    return j < len ? table[j >> a.page_log2] : -1;
  }
  __device__ __forceinline__ bool page_ok(int p) const {
    return static_cast<uint32_t>(p) < static_cast<uint32_t>(a.n_pages);
  }
  // bit r: key 16 b + r of step s is there
  __device__ __forceinline__ uint32_t present(int s, int b, int page) const {
    const int j = s * kKeys + 16 * b;
    const int nc = min(max(len - j, 0), 16), nw = min(max(total - j, 0), 16);
    return ((1u << nw) - 1) & (page_ok(page) ? 0xFFFFu : ~((1u << nc) - 1));
  }
  // whether all 16 keys are the cache's, and there
  __device__ __forceinline__ bool plain(int s, int b, int page) const {
    return s * kKeys + 16 * b + 16 <= len && page_ok(page);
  }
  // Brings keys 16 b.. of step s: K and V (kBoth), or K (kv 1) or V (2).
  // Row i * RPI + r of a copy (r < RPI: its lane's) has swz(i * RPI) ^ swz(r):
  // every copy's offset is the first one's, one xor and one sum away.
  template <bool kBoth>
  __device__ __forceinline__ void issue(int s, int b, int page, int kv) const {
    const int j = s * kKeys + 16 * b;
    const bool v_only = !kBoth && kv == 2;
    const uint32_t buf = lds0 + (s & 1) * 2 * kStep + b * 16 * D * 2 + (v_only ? kStep : 0);
    const long long at =
        (((static_cast<long long>(page) * a.n_kv + h) << a.page_log2) +
         (j & ((1 << a.page_log2) - 1))) * D;
    const uint16_t* const c1 = v_only ? a.vc : a.kc;
    int ln = lane;
    asm("" : "+v"(ln));  // (the offsets made anew: registers are short)
    if (plain(s, b, page)) {
      const uint16_t* b1 = uniform_ptr(c1 + at);
      const uint16_t* b2 = uniform_ptr(a.vc + at);
      const uint32_t off0 = (ln / CH) * (D * 2) + (((ln % CH) ^ swz<D>(ln / CH)) << 4);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint32_t off = (off0 ^ (swz<D>(i * RPI) << 4)) + i * 1024;
        dma16_base(buf + i * 1024, off, b1);
        if (kBoth) dma16_base(buf + kStep + i * 1024, off, b2);
      }
    } else if (j < total) {
      // rows of the cache, then of the window; what is not there reads a
      // window row and is masked
      const int n_cache = page_ok(page) ? min(len - j, 16) : 0;
      const kernarg_p ca = cold_args();
      const uint16_t* const w1 = v_only ? ca->v : ca->k;
      const uint16_t* const w2 = ca->v;
      const long long ws1 = v_only ? ca->v_stride : ca->k_stride, ws2 = ca->v_stride;
#pragma unroll 1
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + ln / CH;
        const int c = ((ln % CH) ^ swz<D>(row)) * 8;
        const long long w = win.off + min(max(j + row - len, 0), win.n - 1);
        const bool cached = row < n_cache;
        dma16_ptr(buf + i * 1024, (cached ? c1 + at + row * D : w1 + w * ws1 + h * D) + c);
        if (kBoth)
          dma16_ptr(buf + kStep + i * 1024,
                    (cached ? a.vc + at + row * D : w2 + w * ws2 + h * D) + c);
      }
    }
  }
  // Rows of V that nobody sees become 0 (0 times what lies there need not be
  // 0), and so do infinities and NaN in the window's rows, which some queries
  // see and others do not: true if there are any, to be added by odd_v.  For
  // the 16 keys that the calling wave has brought.
  __device__ __forceinline__ bool fix_v(int s, int b, uint32_t there) const {
    const int j = s * kKeys + 16 * b;
    unsigned char* vb = lds + (s & 1) * 2 * kStep + kStep + b * 16 * D * 2;
    bool odd = false;
#pragma unroll 1
    for (int i = 0; i < NI; ++i) {
      const int row = i * RPI + lane / CH;
      u32x4* at = reinterpret_cast<u32x4*>(vb + i * 1024 + 16 * lane);
      if (!(there >> row & 1)) {
        *at = (u32x4){0, 0, 0, 0};
      } else if (j + row >= len && win.n > 1) {
        u32x4 w = *at;
        bool mine = false;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const bool lo = fp16_odd(w[c]), hi = fp16_odd(w[c] >> 16);
          mine |= lo || hi;
          w[c] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
        }
        if (mine) *at = w;
        odd |= mine;
      }
    }
    return __any(odd);
  }
  // bit i: key 16 b + 4 grp + i of step s is there and seen by a node with these ancestors
  __device__ __forceinline__ uint32_t seen_bits(int s, int b, uint32_t there, uint64_t up) const {
    const int w0 = s * kKeys + 16 * b - len;  // key 0's window node, if not negative
    const uint32_t tree = w0 >= 0    ? static_cast<uint32_t>(up >> (w0 & 63))
                          : w0 > -16 ? static_cast<uint32_t>(up << -w0) | ((1u << -w0) - 1)
                                     : 0xFFFFu;
    return (there & tree) >> (4 * grp);
  }
  __device__ __forceinline__ int node_of(int r) const {
    return min(r, rows - 1) / cold_args()->group;
  }
  // The 16-B pieces of Q's row r that a lane holds (a row past the end: the last).
  __device__ __forceinline__ void load_q(int r, h8 (&q)[KK]) const {
    r = min(r, rows - 1);
    const int node = r / a.group, g = r - node * a.group;
    const uint16_t* qp =
        a.q + static_cast<long long>(win.off + node) * a.q_stride + (h * a.group + g) * D;
#pragma unroll
    for (int s = 0; s < KK; ++s) {
      const u32x4 w = *reinterpret_cast<const u32x4_u*>(qp + s * 32 + grp * 8);
      q[s] = __builtin_bit_cast(h8, w);
    }
  }
  // Waits for Q before the loop: left to the compiler, the waits stand at Q's
  // uses inside it, where they wait for the copies just issued as well. Over
  // many steps that costs (a pass of a tree of 64 over 131,071 tokens: 167 us
  // against 162); the small blocks do few steps, and there the first step's
  // start weighs more (four tokens over 4,099: 14.1 us against 14.6 with it).
  template <int RT>
  static __device__ __forceinline__ void settle_q(h8 (&q)[RT][KK]) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int s = 0; s < KK; ++s) asm volatile("" : "+v"(q[rt][s]));
  }
  // Piece st * 4 + grp of K's row col of a 16-key block; at: k_offset plus
  // the block's place, multiples of 256 B.
  __device__ __forceinline__ uint32_t k_offset() const {
    return col * (D * 2) + ((grp ^ swz<D>(col)) << 4);
  }
  static __device__ __forceinline__ uint32_t k_piece(uint32_t at, int i) { return at ^ (i << 6); }
  // at: k_piece(.., st % 4)
  __device__ __forceinline__ h8 k_frag(uint32_t at, int st, int block = 0) const {
    return *reinterpret_cast<const h8*>(lds + at + (block * 16 * D * 2 + (st >> 2) * 256));
  }
  // V's columns 0..15 of row 4 grp + col / 4 of a 16-key block; tile c of
  // columns is at v_tile(that plus the block's place, c).
  __device__ __forceinline__ uint32_t v_offset() const {
    const int row = 4 * grp + (col >> 2);
    return kStep + row * (D * 2) + ((((col & 3) >> 1) ^ swz<D>(row)) << 4) + (col & 1) * 8;
  }
  static __device__ __forceinline__ uint32_t v_tile(uint32_t at, int c) {
    return (at ^ ((c & 7) << 5)) + (c >> 3) * 256;
  }
  // V's operand: 16 columns (at: v_tile) at keys 32 st.. of a step
  __device__ __forceinline__ h8 v_frag(uint32_t at, int st) const {
    s4 x[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
      x[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s4_p)((lds_char_p)lds + at + (st * 2 + b) * 16 * D * 2));
    return __builtin_bit_cast(h8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // Adds what weight w (0: not seen) brings to columns c.. (4) from fix_v's infinities and NaN
  // of window node `node`.
  __device__ __forceinline__ void add_odd(f4& o, int node, int c, float w, bool see) const {
    const kernarg_p ca = cold_args();
    const uint64_t b = *reinterpret_cast<const uint64_t*>(
        ca->v + static_cast<long long>(win.off + node) * ca->v_stride + h * D + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = static_cast<uint32_t>(b >> (16 * i)) & 0xFFFFu;
      o[i] += see && fp16_odd(x) ? w * half_bits_to_float(x) : 0.f;
    }
    asm volatile("" : "+v"(o)::"memory");  // (one after the other: registers)
  }
  // Row r's columns c.. (4), and its sum l about mref.
  template <int N, int kStride>
  __device__ __forceinline__ void store(int r, int c, const f4 (&o)[N], float mref, float l,
                                        bool first) const {
    if (r >= rows) return;
    const kernarg_p a = cold_args();
    if (parts == 1) {
      const int node = r / a->group, g = r - node * a->group;
      const long long at = static_cast<long long>(win.off + node) * a->n_heads + h * a->group + g;
      const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
      for (int d = 0; d < N; ++d) {
        h4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = l != 0.f ? static_cast<_Float16>(o[d][i] * inv) : static_cast<_Float16>(0);
        *reinterpret_cast<h4*>(a->out + at * D + c + d * kStride) = y;
      }
    } else {
      const long long pa =
          (static_cast<long long>(unit) * a->row_blocks + rb) * a->block_rows + r - rb * a->block_rows;
#pragma unroll
      for (int d = 0; d < N; ++d)
        *reinterpret_cast<f4*>(a->part_o + pa * D + c + d * kStride) = o[d];
      if (first) a->part_ml[pa] = make_float2(mref, l);
    }
  }
};

// The parts of a row's keys, joined: a workgroup per (token, head), each
// 16-B lanes taking whole parts in turn.  A part whose l is 0 has no key that
// the row sees, and what its O holds is not read as a number.  Latency decides
// for few rows (four tokens of 16 heads in 128 parts: 4.3 us; a tree of 64 in
// 64 parts: 14 us for 67 MB).  (256 threads of eight loads whatever D: 1 us
// more at D 64 and 256.)
template <int D>
constexpr int kJoinThreads = 2 * D;  // (counted on by the call's limit)
template <int D>
__global__ void __launch_bounds__(kJoinThreads<D>) attn_join_kernel(const AttnArgs a) {
  constexpr int LP = D / 4;                 // lanes of a part
  constexpr int SP = kJoinThreads<D> / LP;  // parts at once
  constexpr int U = 4;                      // loads under way per lane
  const int per = a.max_window * a.n_heads;
  const int seq = blockIdx.x / per;
  const int rest = blockIdx.x - seq * per;
  const int node = rest / a.n_heads, head = rest - node * a.n_heads;
  const Window w = window_of(a.win_off, seq, a.n_tokens, a.max_window);
  const int2 plan = a.seq_plan[seq];  // the first unit, the parts
  if (node >= w.n || plan.y <= 1) return;
  const int h = head / a.group, r = node * a.group + head - h * a.group;
  const int rb = r / a.block_rows;
  // the row in the unit's first part; from part to part:
  const long long at =
      (static_cast<long long>(plan.x + h * plan.y) * a.row_blocks + rb) * a.block_rows + r -
      rb * a.block_rows;
  const long long step = static_cast<long long>(a.row_blocks) * a.block_rows;
  const int t = threadIdx.x, sub = t / LP, c = (t % LP) * 4;
  const float* po = a.part_o + at * D + c;
  // every lane group joins its parts about a maximum of its own
  float m = -INFINITY, sum = 0.f;
  f4 o = (f4){0.f, 0.f, 0.f, 0.f};
  for (int s0 = sub; s0 < plan.y; s0 += SP * U) {
    f4 v[U];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u * SP, plan.y - 1);
      ml[u] = a.part_ml[at + s * step];
      v[u] = *reinterpret_cast<const f4*>(po + s * step * D);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * SP >= plan.y) ml[u].y = 0.f;
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
  __shared__ f4 so[kJoinThreads<D>];
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
    const long long row = static_cast<long long>(w.off + node) * a.n_heads + head;
    *reinterpret_cast<h4*>(a.out + row * D + c) = z;
  }
}

}  // namespace sg
