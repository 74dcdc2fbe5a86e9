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
  // seq_plan: per sequence its first unit and the parts of its units; then the
  // steps of a part.
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
__device__ __forceinline__ bool find_unit(const AttnArgs& a, int unit, int lane, bool plan, Unit& u) {
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
       overlap(length_out, n_seq, cache->pages, pages)))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: length_out overlaps the cache's lengths or pages, n_path, path or win_off",
                     nm);
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
  // Enough for every smaller batch too: within a way of cutting fewer sequences
  // have no more units, but fewer may be cut where more are not.
  const int group = n_heads / n_kv_heads;
  const sg::Layout l = sg::attn_layout(n_seq, max_window, max_len, group, n_kv_heads, head_dim);
  size_t bytes = l.bytes;
  for (int few : l.few)
    if (few > 0 && few < n_seq) {
      const size_t b =
          sg::attn_layout(few, max_window, max_len, group, n_kv_heads, head_dim).bytes;
      bytes = b > bytes ? b : bytes;
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
