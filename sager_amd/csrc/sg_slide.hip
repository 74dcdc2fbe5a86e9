// sg_slide.hip - attention over a 16-bit or a quantised cache, over all of it
// or over a sliding window and the first tokens (the sinks).
//
// A token at position p sees its ancestors (in a chain: all before it) and
// itself, as far as they are less than `reach` positions back or among the
// first `sinks` positions.  The keys come in steps of 64: the cache's steps,
// then the window's own, so that a step is all of one kind; the steps that no
// row of a block sees are passed over.  The two products, the running
// reference point of a row's weights and the cut of a batch into units are
// those of sg_attn.hip.
//
// slide_few_kernel: blocks of 16 or 32 rows.  Four waves share the keys of the
// first product and the columns of the second, as there, but K and V come
// through registers: a wave's keys are nobody else's, so K needs no LDS at
// all, and V's columns go through a corner of LDS that is the wave's own,
// where ds_read_b64_tr_b16 turns them.  Only P is exchanged, so a step has one
// barrier, and a step's loads are under way during the one before.
//
// A code times its scale has up to 18 bits, and rounding it to a factor of the
// products costs more than all else: keys of 2^-12 of their size off move
// scores, and so weights, by several times the output's own rounding.  So a
// quantised value is two 16-bit numbers, rounded and rest, and each product is
// made with both; the matrix cores have the time.
//
// V at infinity or NaN where some rows see it and others do not: a product
// with a weight of 0 would spread it.  In the steps that not every row sees in
// full such values are 0 in the product; if there were any, they are added at
// the end to the rows that see them (what they are multiplied by does not
// matter any more).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "sg_attn.hpp"

namespace sg {

// 16 and 4 B of global memory, at any address that the buffers' own alignment allows
typedef const __attribute__((address_space(1))) unsigned char* gmem;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x4 load16(gmem p, uint32_t off = 0) {
  return *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(p + off);
}
__device__ __forceinline__ uint32_t load4(gmem p, uint32_t off = 0) {
  return *reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(p + off);
}

// Here the loads of x are waited for, and not before: left to the compiler, some
// of what is made of them moves up to where the step before has just issued them.
template <typename T, int N>
__device__ __forceinline__ void settle(T (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// Two weights more in a row's sum.  Weights are rounded to 16 bits, since the
// matrix cores take such factors: 2^-11 of a weight at the most, as the output's
// own rounding; in two parts they would double the second product.  The sum is of
// the rounded weights, those that the product with V is made with: what rounding a
// large weight takes from one it then takes from the other.  (Against 64 bits the
// errors are 1.0 to 1.26 times those of 32-bit weights: 2.0e-4 to 2.6e-4 of the
// outputs' size and 1.9e-4 to 2.1e-4, in batches of one token to a chunk of 4,096.)
__device__ __forceinline__ float weight_sum(h2 p, float sum) {
  const h2 one = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
  return __builtin_amdgcn_fdot2(p, one, sum, false);
}

struct SlideArgs : AttnArgs {
  const uint16_t *ks, *vs;  // scales of the quantised cache (kc, vc: its codes)
  int reach, sinks;
  int spread;  // how workgroups are mapped to row blocks
  int turn_units;  // units, as far as the host knows
};
enum { kSpreadUnits, kSpreadTurns, kSpreadRuns };

// As cold_args, for paths taken now and then.
typedef const __attribute__((address_space(4))) SlideArgs* slide_p;
__device__ __forceinline__ slide_p cold_slide() {
  slide_p p = (slide_p)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// The steps that a sequence's nodes first .. last see: [0, sink) and [low,
// high), the window's steps from `cached` on.
struct Steps {
  int cached, sink, low, high;
  __device__ __forceinline__ int count() const { return low > sink ? sink + high - low : high; }
  __device__ __forceinline__ int at(int v) const {  // the v-th of them
    return low > sink && v >= sink ? v - sink + low : v;
  }
  __device__ __forceinline__ int skip(int s) const {  // s, or the next that is seen
    return s >= sink && s < low ? low : s;
  }
};
__device__ __forceinline__ Steps steps_seen(int len, int n, int first, int last, int reach,
                                            int sinks) {
  Steps t;
  t.cached = (len + kKeys - 1) / kKeys;
  t.high = t.cached + last / kKeys + 1;
  const int s = min(sinks, len + n);
  t.sink = min(s <= len ? (s + kKeys - 1) / kKeys : t.cached + (s - len + kKeys - 1) / kKeys, t.high);
  const long long l = static_cast<long long>(len) + first - reach + 1;  // the first position seen
  t.low = l <= 0 ? 0
                 : static_cast<int>(l < len ? l / kKeys : t.cached + (l - len) / kKeys);
  return t;
}
__device__ __forceinline__ int steps_of(const SlideArgs& a, int seq, int* len, Window* win) {
  if (seq >= a.n_seq) return 0;
  *win = window_of(a.win_off, seq, a.n_tokens, a.max_window);
  *len = cached_len(a.length[seq], a.page_log2, a.pages_per_seq);
  return win->n > 0 ? steps_seen(*len, win->n, 0, win->n - 1, a.reach, a.sinks).count() : 0;
}

template <int D>
struct SlidePart : Part<D> {
  typedef Part<D> B;
  const SlideArgs& sa;
  Steps steps;
  int first, last;  // nodes of the block

  __device__ __forceinline__ explicit SlidePart(const SlideArgs& s) : B{s}, sa(s) {}

  // Finds the block's work; its steps are steps.skip(begin) .. end - 1.
  __device__ __forceinline__ bool start(unsigned char* l) {
    this->lds = l;
    this->lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char_p)l));
    const int lane = threadIdx.x & 63;
    this->lane = lane;
    this->col = lane & 15;
    this->grp = lane >> 4;
    const int id = blockIdx.x;
    if (sa.spread == kSpreadTurns) {
      // Many row blocks that see all before them: over the XCDs in turn, the last
      // rows of all units, which see most, first, so that short blocks fill up what
      // long ones leave (4,096 tokens over none, 32 heads on 8 of 128: 159 us, unit
      // after unit 258).
      // (units that the host does not count on follow likewise)
      const int turn = sa.turn_units, run = turn * sa.row_blocks;
      const bool past = id >= run;
      const int units = past ? max(sa.max_units - turn, 1) : turn, in = past ? id - run : id;
      const int row = in / units;
      int k = in - row * units;
      this->unit = k + (past ? turn : 0);
      this->rb = sa.row_blocks - 1 - row;
      if (this->rb < 0) return false;  // (behind the last one)
    } else if (sa.spread == kSpreadRuns) {
      // That see a window: an XCD has neighbours, whose windows are the same keys
      // but for a few, and reads them once (4,096 tokens of 32 heads on 8 of 128 over
      // windows of 2,048: 210 us, 255 quantised; in turn 221 and 327).
      // (past the last unit there is none)
      const int at = (id & 7) * (gridDim.x >> 3) + (id >> 3);
      this->unit = at / sa.row_blocks;
      this->rb = at - this->unit * sa.row_blocks;
    } else {
      // The row blocks of a unit are 8 workgroups apart: on one XCD, whose L2
      // then reads the unit's keys once.
      const int oct = id / (8 * sa.row_blocks), in = id - oct * 8 * sa.row_blocks;
      this->rb = in >> 3;
      this->unit = oct * 8 + (in & 7);
    }
    auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // (the same in every lane)
    this->unit = one(this->unit);
    this->rb = one(this->rb);
    Unit u;
    const bool plan = sa.cut && id == 0 && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) == 0;
    if (!find_unit(sa, this->unit, lane, plan, u)) return false;
    this->h = one(u.h);
    this->parts = one(u.parts);
    this->win = Window{one(u.win.off), one(u.win.n)};
    this->rows = this->win.n * sa.group;
    if (this->rb * sa.block_rows >= this->rows) return false;
    this->len = one(u.len);
    this->total = this->len + this->win.n;
    this->table =
        (const_int_p)(sa.pages + static_cast<long long>(one(u.seq)) * sa.pages_per_seq);
    const int n = this->win.n;
    first = one(sa.parent ? 0 : this->rb * sa.block_rows / sa.group);
    last = one(sa.parent ? n - 1 : min((this->rb + 1) * sa.block_rows - 1, this->rows - 1) / sa.group);
    const Steps all = steps_seen(this->len, n, 0, n - 1, sa.reach, sa.sinks);
    steps = steps_seen(this->len, n, first, last, sa.reach, sa.sinks);
    const int k = one(u.k), part = one(u.part), count = one(u.steps);
    const long long from = static_cast<long long>(k) * part;
    const int v0 = from < count ? static_cast<int>(from) : count;
    const int v1 = k == this->parts - 1 || from + part > count ? count : static_cast<int>(from + part);
    this->begin = v0 < v1 ? steps.skip(all.at(v0)) : 0;
    this->end = v0 < v1 ? min(all.at(v1 - 1) + 1, steps.high) : 0;
    return true;
  }
  // A part of which the block's rows see no step: says so, and true, for the join.
  __device__ __forceinline__ bool empty() const {
    if (this->begin < this->end || this->parts == 1) return false;
    const slide_p a = cold_slide();
    const int in = threadIdx.x;
    if (in < a->block_rows)
      a->part_ml[(static_cast<long long>(this->unit) * a->row_blocks + this->rb) * a->block_rows + in] =
          make_float2(0.f, 0.f);
    return true;
  }
  // Where the rows of a cached step's blocks of 16 keys begin, in values.
  struct Rows {
    long long at[4];
    uint32_t ok;  // bit b: block b's page is there
  };
  __device__ __forceinline__ Rows rows_of(int s) const {
    Rows r;
    r.ok = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int j = s * kKeys + 16 * b;
      int p = j < this->len ? this->table[j >> sa.page_log2] : -1;
      if (this->page_ok(p))
        r.ok |= 1u << b;
      else
        p = 0;  // (any page: what is read there is not used)
      r.at[b] = (((static_cast<long long>(p) * sa.n_kv + this->h) << sa.page_log2) +
                 (j & ((1 << sa.page_log2) - 1))) * D;
    }
    return r;
  }
  // Whether every row of the block sees every key of step s: of the cache,
  __device__ __forceinline__ bool full(int s, uint32_t ok) const {
    return ok == 15u && (s + 1) * kKeys <= this->len &&
           ((s + 1) * kKeys <= sa.sinks ||
            s * kKeys > static_cast<long long>(this->len) + last - sa.reach);
  }
  // and of a chain's window.
  __device__ __forceinline__ bool full_window(int s) const {
    const int w = (s - steps.cached) * kKeys;
    return !sa.parent && w + kKeys - 1 <= first &&
           (this->len + w + kKeys <= sa.sinks || w > static_cast<long long>(last) - sa.reach);
  }
  // Which of step s's keys are there.
  __device__ __forceinline__ uint64_t present(int s, uint32_t ok) const {
    const int n = s < steps.cached ? this->len - s * kKeys
                                   : this->win.n - (s - steps.cached) * kKeys;
    uint64_t m = n >= kKeys ? ~0ull : (1ull << n) - 1;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (!(ok >> b & 1)) m &= ~(0xFFFFull << (16 * b));
    return m;
  }
  // bit i: key k + i of step s (i < 4) is there and seen by a node at position pos;
  // up: whom of the window's tree it sees (with a parent).
  __device__ __forceinline__ uint32_t seen4(int s, int k, uint64_t there, int pos,
                                            uint64_t up) const {
    uint32_t m = static_cast<uint32_t>(there >> k) & 15u;
    const bool cached = s < steps.cached;
    const slide_p ca = cold_slide();
    const int sinks = ca->sinks;
    const uint32_t reach = ca->reach;
    if (!cached && ca->parent) return m & static_cast<uint32_t>(up >> k);
    // (positions as unsigned differences: no further than pos, and less than reach)
    const int p0 = (cached ? s * kKeys : this->len + (s - steps.cached) * kKeys) + k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t back = pos - (p0 + i);
      const uint32_t most = p0 + i < sinks ? 0x7FFFFFFFu : reach - 1;
      m &= back <= most ? ~0u : ~(1u << i);
    }
    return m;
  }
};

// Eight 16-bit values, or a group's scale, of which infinities and NaN, and
// all if they are not there, become 0: whether there were any of those.
__device__ __forceinline__ bool finite8(u32x4& w, bool there) {
  bool odd = false;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const bool lo = fp16_odd(w[c]), hi = fp16_odd(w[c] >> 16);
    odd |= there && (lo || hi);
    w[c] &= there ? (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u) : 0u;
  }
  return odd;
}
__device__ __forceinline__ bool finite_scale(uint32_t& scale, bool there) {
  const bool odd = there && fp16_odd(scale);
  scale = there && !odd ? scale : 0u;
  return odd;
}

// Adds the infinities and NaN that the products were made without: of each key
// of a step that not all rows see in full, to columns c + 16 d (4) of the rows
// that see it, at positions pos and with the tree's up.
template <int D, bool Q8, int RT, int N>
__device__ __forceinline__ void add_odds(const SlidePart<D>& t, f4 (&acc)[RT][N], int c,
                                         const int (&pos)[RT], const uint64_t (&up)[RT]) {
  const slide_p a = cold_slide();
  for (int s = t.begin; s < t.end; s = t.steps.skip(s + 1)) {
    const bool window = s >= t.steps.cached;
    typename SlidePart<D>::Rows rows;
    rows.ok = 15u;
    if (!window) rows = t.rows_of(s);
    if (window ? t.full_window(s) : t.full(s, rows.ok)) continue;
    const uint64_t there = t.present(s, rows.ok);
#pragma unroll 1
    for (int r = 0; r < kKeys; ++r) {
      if (!(there >> r & 1)) continue;
      const int b = r >> 4;
      const long long at =
          window ? static_cast<long long>(t.win.off + (s - t.steps.cached) * kKeys + r) * a->v_stride +
                       t.h * D
                 : (b == 0 ? rows.at[0] : b == 1 ? rows.at[1] : b == 2 ? rows.at[2] : rows.at[3]) +
                       (r & 15) * D;
      const uint16_t* const row = (window ? a->v : a->vc) + at;
      int c0 = c;
      asm("" : "+v"(c0));  // (the addresses made anew: registers)
      bool see[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) see[rt] = t.seen4(s, r, there, pos[rt], up[rt]) & 1;
#pragma unroll
      for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = c0 + 16 * d + i;
          // (a group of codes that is not finite is so throughout)
          const float x =
              half_bits_to_float(Q8 && !window ? a->vs[(at + k) / kKvGroup] : row[k]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt][d][i] += see[rt] && !isfinite(x) ? x : 0.f;
        }
    }
  }
}

// The nodes' positions, and whom of their window each sees, by one wave.
__device__ __forceinline__ void see_tree(const SlideArgs& a, Window w, int len, int lane, int* pos,
                                         uint64_t* seen) {
  uint64_t up = ancestors(a.parent, w, lane);
  const int depth = __popcll(up) - 1;
  pos[lane] = len + max(depth, 0);
  if (a.reach < w.n) {
    uint64_t near = 0;
    for (int j = 0; j < w.n; ++j) {
      const int d = __builtin_amdgcn_readlane(depth, j);
      if (depth - d < a.reach || len + d < a.sinks) near |= 1ull << j;
    }
    up &= near;
  }
  seen[lane] = up;
}

// LDS: V of the four waves, P of two steps, the rows' maxima and sums of the
// four waves, the nodes' positions and what they see, the flags.
template <int D, int RT, bool Q8>
struct SlideFewLds {
  static constexpr uint32_t kRows = 16 * RT;
  // A wave's row of V: slots of 16 columns, of a quantised cache rounded values
  // and rests in turn.  Row r has slot i at i ^ swz(r), so that the 32 B of four
  // or eight rows that are read transposed together lie in different banks.
  static constexpr uint32_t kSlots = D / 64 * (Q8 ? 2 : 1);
  static constexpr uint32_t kRow = kSlots * 32;
  static __device__ __forceinline__ uint32_t swz(uint32_t r) {
    return r / (8 / kSlots) & (kSlots - 1);
  }
  static constexpr uint32_t kWave = kKeys * kRow;
  static constexpr uint32_t kP = 4 * kWave;
  static constexpr uint32_t kStepP = kRows * kKeys * 2;
  static constexpr uint32_t kMax = kP + 2 * kStepP;
  static constexpr uint32_t kSeen = kMax + 4 * kRows * 4;
  static constexpr uint32_t kPos = kSeen + kMaxWindow * 8;
  static constexpr uint32_t kFlags = kPos + kMaxWindow * 4;
  static constexpr uint32_t kBytes = kFlags + 16;
};

// Waves of a SIMD, that is, workgroups of a CU.
constexpr int slide_waves(int dim, int tiles) {
  return dim == 256 ? 2 : dim == 128 ? (tiles == 2 ? 3 : 4) : tiles == 2 ? 4 : 5;
}

// RT: tiles of 16 rows.  Wave w has keys 16 w.. of a step in the first product,
// and columns w D/4 .. of all keys in the second.  Bound by the cache's bytes
// where batches are large (32 sequences of one token over 4,000, 8 kv heads of
// 128: 525 MB in 16 bits in 102 us, 5.2 TB/s; quantised 279 MB in 63 us, 4.4
// TB/s, with vector instructions for the values as the other half of the time),
// and by the length of a step, some 2 us of loads, exponentials and barriers,
// where few workgroups have work.
template <int D, int RT, bool Q8>
__global__ void __launch_bounds__(256, slide_waves(D, RT)) slide_few_kernel(const SlideArgs a) {
  typedef SlidePart<D> P;
  typedef SlideFewLds<D, RT, Q8> L;
  constexpr int KK = D / 32, DQ = D / 64, kRows = L::kRows;
  // A wave's columns of V: LP lanes of 8 values a row, RP rows at once; of
  // codes, 16 a lane.
  constexpr int LP = D / 32, RP = 64 / LP, LQ = D / 64, RQ = 64 / LQ;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  P t(a);
  if (!t.start(lds) || t.empty()) return;
  const int lane = t.lane, col = t.col, grp = t.grp, row0 = t.rb * kRows;
  int* rise = reinterpret_cast<int*>(lds + L::kFlags);  // odd and even: 1 + the last step that moves
  float* mx = reinterpret_cast<float*>(lds + L::kMax);
  uint64_t* seen = reinterpret_cast<uint64_t*>(lds + L::kSeen);
  int* place = reinterpret_cast<int*>(lds + L::kPos);
  unsigned char* const vl = lds + wave * L::kWave;

  // K: lane (col, grp) has key 16 wave + col; its pieces of 8 values lie at
  // 32 i + 8 grp, of a quantised cache at 64 (i / 2) + 16 grp + 8 (i % 2).
  auto piece = [&](int i) {
    return Q8 ? 64 * (i / 2) + 16 * grp + 8 * (i % 2) : 32 * i + 8 * grp;
  };
  // A step's raw K and V, of a window or of the cache: 16 B a register quad.
  struct Raw {
    u32x4 k[KK], v[KK];
  };
  struct Codes {
    u32x4 k[KK / 2], v[LQ];
    uint32_t ks[KK / 2], vs[LQ];
  };
  typedef typename std::conditional<Q8, Codes, Raw>::type Cached;
  typedef typename P::Rows Rows;
  const gmem kc = (gmem)a.kc, vc = (gmem)a.vc, ksc = (gmem)a.ks, vsc = (gmem)a.vs;
  auto load_k = [&](Cached& x, const Rows& rows) {
    const long long at = wave == 0 ? rows.at[0] : wave == 1 ? rows.at[1] : wave == 2 ? rows.at[2] : rows.at[3];
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < KK / 2; ++i) x.k[i] = load16(kc + at, col * D + 64 * i + 16 * grp);
      // the row's scales, two a register
      const gmem sc = ksc + at / (kKvGroup / 2);
      if constexpr (KK == 8) {
        const u32x4 w = load16(sc, col * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.ks[i] = w[i];
      } else {
#pragma unroll
        for (int i = 0; i < KK / 2; ++i) x.ks[i] = load4(sc, col * KK * 2 + 4 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < KK; ++i) x.k[i] = load16(kc + 2 * at, (col * D + piece(i)) * 2);
    }
  };
  auto load_v = [&](Cached& x, const Rows& rows) {
    // (values of the wave's columns; a block of 16 rows or more at once)
    constexpr int N = Q8 ? LQ : KK, L1 = Q8 ? LQ : LP, R1 = Q8 ? RQ : RP;
    // (out of their array: a choice among its elements would put it into scratch memory)
    long long from[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      from[b] = rows.at[b];
      asm("" : "+s"(from[b]));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      constexpr int kBlocks = R1 <= 16 ? 1 : R1 / 16;
      const int b0 = i * R1 / 16, in = lane / L1;
      long long at = from[b0];
      if constexpr (kBlocks == 2) at = in < 16 ? at : from[b0 + 1];
      if constexpr (kBlocks == 4)
        at = in < 32 ? (in < 16 ? from[0] : from[1]) : (in < 48 ? from[2] : from[3]);
      const uint32_t row = i * R1 % 16 + in % 16;
      const uint32_t off = row * D + wave * (D / 4) + (lane % L1) * (Q8 ? 16 : 8);
      if constexpr (Q8) {
        x.v[i] = load16(vc + at, off);
        // (the two scales that the wave's are among)
        x.vs[i] = load4(vsc + at / (kKvGroup / 2), row * (D / 16) + (wave * D / 4 / 64) * 4);
      } else {
        x.v[i] = load16(vc + 2 * at, 2 * off);
      }
    }
  };
  // which of the two scales of load_v a lane's 16 columns have
  const int vhalf = 16 * ((wave * (D / 4) + (lane % LQ) * 16) / kKvGroup & 1);
  auto load_window = [&](Raw& x, int s) {
    const int w0 = (s - t.steps.cached) * kKeys;
    const gmem kp =
        (gmem)(a.k + static_cast<long long>(t.win.off + min(w0 + 16 * wave + col, t.win.n - 1)) * a.k_stride +
               t.h * D);
#pragma unroll
    for (int i = 0; i < KK; ++i) x.k[i] = load16(kp, piece(i) * 2);
#pragma unroll
    for (int i = 0; i < KK; ++i) {
      const int w = min(w0 + i * RP + lane / LP, t.win.n - 1);
      x.v[i] = load16((gmem)(a.v + static_cast<long long>(t.win.off + w) * a.v_stride + t.h * D +
                             wave * (D / 4) + (lane % LP) * 8));
    }
  };

  // The block's steps of the cache and of the window.
  const int cached_end = min(t.end, t.steps.cached);
  int step = t.begin, wstep = t.steps.skip(max(t.begin, t.steps.cached));
  Raw own;
  if (wstep < t.end) load_window(own, wstep);
  if (threadIdx.x < 2) rise[threadIdx.x] = 0;
  if (wave == 3 && a.parent) see_tree(a, t.win, t.len, lane, place, seen);

  h8 qf[RT][KK];
  f4 acc[RT][DQ];
  // lim: the score, less mref, above which mref moves: kRise once it is set
  float mref[RT], l[RT], lim[RT];
  int node[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = min(row0 + rt * 16 + col, t.rows - 1);
    node[rt] = r / a.group;
    const uint16_t* qp = a.q + static_cast<long long>(t.win.off + node[rt]) * a.q_stride +
                         (t.h * a.group + r - node[rt] * a.group) * D;
#pragma unroll
    for (int i = 0; i < KK; ++i)
      qf[rt][i] = __builtin_bit_cast(h8, static_cast<u32x4>(*reinterpret_cast<const u32x4_u*>(qp + piece(i))));
    mref[rt] = 0.f;
    l[rt] = 0.f;
    lim[rt] = -INFINITY;
#pragma unroll
    for (int d = 0; d < DQ; ++d) acc[rt][d] = (f4){0.f, 0.f, 0.f, 0.f};
  }
  // P: [row][two halves of 32 keys][grp][two blocks of 16 keys][4], 16-B pieces
  // swizzled over the row's eight
  const int psw = (col >> 1) & 7;
  const uint32_t p_out =
      L::kP + col * 128 + ((((wave >> 1) * 4 + grp) ^ psw) << 4) + (wave & 1) * 8;
  // V's columns 0..15 of row 4 grp + col / 4 of a 16-key block; slot i is at v_in ^ 32 i
  const uint32_t v_row = 4 * grp + (col >> 2);
  const uint32_t v_in = wave * L::kWave + v_row * L::kRow + L::swz(v_row) * 32 + (col & 3) * 8;

  int it = 0;
  bool odd = false;
  // A step's scores from K, its weights and V into LDS, the second product.
  // scores(s): the products with K; spread(odd): V into the wave's corner;
  // each issues the next step's loads once it is through with its own.
  auto run = [&](int step, bool full, uint64_t there, auto n_parts, auto&& scores,
                 auto&& spread) {
    constexpr int parts = decltype(n_parts)::value;  // of V's values
    const int par = it++ & 1;
    f4 s[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt] = (f4){0.f, 0.f, 0.f, 0.f};
    scores(s);

    float e[RT][4], top[RT], sum[RT];
    auto weigh = [&](int rt, float by) {  // row tile rt's p = 2^(e - by), into LDS
      h4 ph;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        ph[i] = static_cast<_Float16>(__builtin_amdgcn_exp2f(e[rt][i] - by));
      sum[rt] = weight_sum((h2){ph[0], ph[1]}, weight_sum((h2){ph[2], ph[3]}, 0.f));
      *reinterpret_cast<h4*>(lds + p_out + par * L::kStepP + rt * 16 * 128) = ph;
    };
    bool move = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[rt][i] = __builtin_fmaf(s[rt][i], a.scale_log2, -mref[rt]);
      if (!full) {
        const uint32_t see = t.seen4(step, 16 * wave + 4 * grp, there,
                                     a.parent ? place[node[rt]] : t.len + node[rt],
                                     a.parent ? seen[node[rt]] : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[rt][i] = see >> i & 1 ? e[rt][i] : -INFINITY;
      }
      top[rt] = max3(max3(e[rt][0], e[rt][1], e[rt][2]), e[rt][3], e[rt][3]);
      move |= top[rt] > lim[rt];
      weigh(rt, 0.f);
    }
    if (__any(move)) rise[par] = step + 1;
    odd |= spread();
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

    const unsigned char* const pl = lds + L::kP + par * L::kStepP;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      h8 pf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        pf[rt] = *reinterpret_cast<const h8*>(pl + (rt * 16 + col) * 128 +
                                              (((st * 4 + grp) ^ psw) << 4));
#pragma unroll
      for (int d = 0; d < DQ; ++d)
#pragma unroll
        for (int part = 0; part < (parts == 2 ? 2 : 1); ++part) {
          const uint32_t at = v_in ^ 32 * (Q8 ? 2 * d + part : d);
          s4 x[2];
#pragma unroll
          for (int b = 0; b < 2; ++b)
            x[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s4_p)((lds_char_p)lds + at + (st * 2 + b) * 16 * L::kRow));
          const h8 vf = __builtin_bit_cast(
              h8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt], acc[rt][d], 0, 0, 0);
        }
    }
  };
  // 16-bit K and V of a step as they were loaded
  auto raw_scores = [&](const Raw& x, f4 (&s)[RT]) {
#pragma unroll
    for (int i = 0; i < KK; ++i)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        s[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x.k[i]), qf[rt][i],
                                                       s[rt], 0, 0, 0);
  };
  auto raw_spread = [&](const Raw& x, bool full, uint64_t there) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < KK; ++i) {
      const int r = i * RP + lane / LP;
      u32x4 w = x.v[i];
      if (!full) odd |= finite8(w, there >> r & 1);
      const uint32_t p = lane % LP, slot = (Q8 ? 2 : 1) * (p >> 1);
      *reinterpret_cast<u32x4*>(vl + r * L::kRow + (slot ^ L::swz(r)) * 32 + (p & 1) * 16) = w;
    }
    return __any(odd);
  };

  bar();  // the flags are cleared, the tree is there
  while (wstep < t.end) {  // (one step, but for chains of more than 64 tokens)
    const bool full = t.full_window(wstep);
    const uint64_t there = full ? ~0ull : t.present(wstep, 15u);
    run(
        wstep, full, there, std::integral_constant<int, 1>(),
        [&](f4 (&s)[RT]) { raw_scores(own, s); },
        [&] { return raw_spread(own, full, there); });
    wstep = t.steps.skip(wstep + 1);
    if (wstep < t.end) load_window(own, wstep);
  }
  // (no load of the window is under way any more: else the loop would wait for all of its own)
  settle(own.k);
  settle(own.v);
  if (step < cached_end) {
    // A step's loads are under way during the step before, and only one step's:
    // more workgroups on a CU bring more than a second step's registers (32
    // sequences of one token over 4,000 quantised ones, 8 kv heads of 128: 62 us,
    // 71 with two).  (The window's K and V have had these registers before.)
    Cached now;
    Rows rows = t.rows_of(step);
    load_k(now, rows);
    load_v(now, rows);
    while (step < cached_end) {
      const bool full = t.full(step, rows.ok);
      const uint64_t there = full ? ~0ull : t.present(step, rows.ok);
      // (after the last step that one once more: a load that is made or not would
      // be waited for as if it were not, with all before it)
      const int next = t.steps.skip(step + 1);
      rows = t.rows_of(next < cached_end ? next : step);
      run(
          step, full, there, std::integral_constant<int, Q8 ? 2 : 1>(),
          [&](f4 (&s)[RT]) {
            settle(now.k);
            if constexpr (Q8) {
              settle(now.ks);
#pragma unroll
              for (int i = 0; i < KK / 2; ++i) {
                const h2 d = scale2(now.ks[i] >> (grp & 2) * 8);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  uint32_t w[2][2], x[2][2];
                  decode4(now.k[i][2 * j], d, w[0], x[0]);
                  decode4(now.k[i][2 * j + 1], d, w[1], x[1]);
                  const h8 kf = __builtin_bit_cast(h8, (u32x4){w[0][0], w[0][1], w[1][0], w[1][1]});
                  const h8 kx = __builtin_bit_cast(h8, (u32x4){x[0][0], x[0][1], x[1][0], x[1][1]});
#pragma unroll
                  for (int rt = 0; rt < RT; ++rt) {
                    s[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][2 * i + j], s[rt], 0, 0, 0);
                    s[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx, qf[rt][2 * i + j], s[rt], 0, 0, 0);
                  }
                }
              }
            } else {
              raw_scores(now, s);
            }
            load_k(now, rows);
          },
          [&] {
            bool odd = false;
            settle(now.v);
            if constexpr (Q8) {
              settle(now.vs);
#pragma unroll
              for (int i = 0; i < LQ; ++i) {
                const int r = i * RQ + lane / LQ;
                uint32_t scale = now.vs[i] >> vhalf;
                if (!full) odd |= finite_scale(scale, there >> r & 1);
                const h2 d = scale2(scale);
                uint32_t w[4][2], x[4][2];
#pragma unroll
                for (int j = 0; j < 4; ++j) decode4(now.v[i][j], d, w[j], x[j]);
                unsigned char* const row = vl + r * L::kRow;
                const uint32_t slot = 2 * (lane % LQ) ^ L::swz(r);
                u32x4* to = reinterpret_cast<u32x4*>(row + slot * 32);
                to[0] = (u32x4){w[0][0], w[0][1], w[1][0], w[1][1]};
                to[1] = (u32x4){w[2][0], w[2][1], w[3][0], w[3][1]};
                to = reinterpret_cast<u32x4*>(row + (slot ^ 1) * 32);
                to[0] = (u32x4){x[0][0], x[0][1], x[1][0], x[1][1]};
                to[1] = (u32x4){x[2][0], x[2][1], x[3][0], x[3][1]};
              }
              odd = __any(odd);
            } else {
              odd = raw_spread(now, full, there);
            }
            load_v(now, rows);
            return odd;
          });
      step = next;
    }
  }

  if (odd) {
    int pos[RT];
    uint64_t up[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      pos[rt] = a.parent ? place[node[rt]] : t.len + node[rt];
      up[rt] = a.parent ? seen[node[rt]] : 0;
    }
    add_odds<D, Q8>(t, acc, wave * (D / 4) + 4 * grp, pos, up);
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
    if (a.parent && !seen[node[rt]]) lt = 0.f;  // an absent node
    t.template store<DQ, 16>(r, wave * (D / 4) + 4 * grp, acc[rt], mref[rt], lt,
                             wave == 0 && grp == 0);
  }
}

// ---- blocks of 256 rows ---------------------------------------------------------------------
// LDS: K and V of two steps, or of one and the codes of two; the nodes'
// positions and what they see, the scales of two steps' codes, the flags.
template <int D>
struct SlideRowsLds {
  static constexpr uint32_t kSeen = 4 * Part<D>::kStep;
  static constexpr uint32_t kPos = kSeen + kMaxWindow * 8;
  static constexpr uint32_t kScales = kPos + kMaxWindow * 4;
  static constexpr uint32_t kScaleStep = 2 * kKeys * D / kKvGroup * 2;  // K's and V's
  static constexpr uint32_t kFlags = kScales + 2 * kScaleStep;
  static constexpr uint32_t kBytes = kFlags + 16;
};
constexpr int kSlideRowWaves = 8, kSlideRowTiles = 2;  // 16-row tiles of a wave

// Eight waves with 32 rows each, as attn_rows_kernel: K and V of a step lie in
// LDS in 16 bits, each wave brings 16 keys of one of them.  Rows of 16 bits are
// copied into one of two buffers while the other is computed on.  A step of
// codes lies in half of the second buffer; 32 of its keys at a time are turned
// into rounded values and rests of K and of V, which fill the first.  Bound by
// the matrix cores (36 % of the cycles) and the vector instructions between the
// products (34 %), which no more than two waves a SIMD, for the registers' sake, do
// in turn (4,096 tokens over 4,099 more, windows of 2,048: 16 heads on 2 of 256 155
// to 190 us, 890 to 730 TFLOP/s, 32 heads on 8 of 128 187 to 210).  Where each CU
// has one block the heaviest decides: without a cache the last, which sees twice the
// mean; over a quantised one the first, which sees little else, at 1.5 times a
// 16-bit step's time (280 us for the heads of 256; those of 128, two blocks a CU,
// 250 to 265).
template <int D, bool Q8>
__global__ void __launch_bounds__(64 * kSlideRowWaves) slide_rows_kernel(const SlideArgs a) {
  typedef SlidePart<D> P;
  typedef SlideRowsLds<D> L;
  typedef typename P::Rows Rows;
  constexpr int RT = kSlideRowTiles, NW = kSlideRowWaves, DT = D / 16, KK = D / 32;
  constexpr int CH = D / 8, RPI = 64 / CH, NI = 16 / RPI;  // as Part: 16-bit copies
  constexpr int CQ = D / 16, RQ = 64 / CQ, NQ = 16 / RQ;   // of codes
  constexpr int kAhead = 4;  // operands read ahead
  // Halves of a step (32 keys) at once: fewer waits for scores and operands, where
  // registers allow it (as below, heads of 128 without a window: 524 us, by one 595;
  // at head dimension 64 two workgroups share a CU as long as they need 128).
  constexpr int kHalves = D == 128 || (D == 64 && !Q8) ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blk = wave & 3;
  const bool is_v = wave >= 4;
  P t(a);
  if (!t.start(lds) || t.empty()) return;
  const int lane = t.lane, col = t.col, grp = t.grp;
  const int row0 = (t.rb * NW + wave) * 16 * RT;
  int* odds = reinterpret_cast<int*>(lds + L::kFlags);  // whether V had infinities or NaN
  uint64_t* seen = reinterpret_cast<uint64_t*>(lds + L::kSeen);
  int* place = reinterpret_cast<int*>(lds + L::kPos);
  // where the wave's 16 keys go in a buffer of K and V
  const uint32_t mine = (is_v ? P::kStep : 0) + blk * 16 * D * 2;

  // 16-bit rows of step s into buffer b (bytes from LDS' start)
  auto bring = [&](int s, const Rows& rows, uint32_t b) {
    int ln = lane;
    asm("" : "+v"(ln));  // (the offsets made anew: registers are short)
    const uint32_t to = t.lds0 + b + mine;
    if (!Q8 && s < t.steps.cached) {
      const long long at =
          blk == 0 ? rows.at[0] : blk == 1 ? rows.at[1] : blk == 2 ? rows.at[2] : rows.at[3];
      const uint16_t* src = uniform_ptr((is_v ? a.vc : a.kc) + at);
      const uint32_t off0 = (ln / CH) * (D * 2) + (((ln % CH) ^ swz<D>(ln / CH)) << 4);
#pragma unroll
      for (int i = 0; i < NI; ++i)
        dma16_base(to + i * 1024, (off0 ^ (swz<D>(i * RPI) << 4)) + i * 1024, src);
    } else {
      const slide_p ca = cold_slide();
      const int w0 = (s - t.steps.cached) * kKeys + 16 * blk;
      const uint16_t* const base = (is_v ? ca->v : ca->k) + t.h * D;
      const long long stride = is_v ? ca->v_stride : ca->k_stride;
      if (w0 + 16 <= t.win.n) {
        const uint16_t* src = uniform_ptr(base + (t.win.off + w0) * stride);
        const uint32_t row0 = (ln / CH) * (static_cast<uint32_t>(stride) * 2);
        const uint32_t c0 = ((ln % CH) ^ swz<D>(ln / CH)) << 4;
#pragma unroll
        for (int i = 0; i < NI; ++i)
          dma16_base(to + i * 1024, row0 + (c0 ^ (swz<D>(i * RPI) << 4)), src + i * RPI * stride);
      } else {
#pragma unroll 1
        for (int i = 0; i < NI; ++i) {
          const int row = i * RPI + ln / CH;
          const int c = ((ln % CH) ^ swz<D>(row)) * 8;
          const long long w = t.win.off + min(w0 + row, t.win.n - 1);
          dma16_ptr(to + i * 1024, base + w * stride + c);
        }
      }
    }
  };
  // codes of cached step s, and their scales, into half `half` of the second buffer
  auto bring_codes = [&](const Rows& rows, int half) {
    int ln = lane;
    asm("" : "+v"(ln));
    const long long at =
        blk == 0 ? rows.at[0] : blk == 1 ? rows.at[1] : blk == 2 ? rows.at[2] : rows.at[3];
    const unsigned char* src =
        uniform_ptr(reinterpret_cast<const unsigned char*>(is_v ? a.vc : a.kc) + at);
    const uint32_t to = t.lds0 + (2 + half) * P::kStep + (is_v ? P::kStep / 2 : 0) + blk * 16 * D;
#pragma unroll
    for (int i = 0; i < NQ; ++i) dma16_base(to + i * 1024, ln * 16 + i * 1024, src);
    if (ln < D / 16) {
      const unsigned char* sc = uniform_ptr(
          reinterpret_cast<const unsigned char*>(is_v ? a.vs : a.ks) + at / (kKvGroup / 2));
      dma16_base(t.lds0 + L::kScales + half * L::kScaleStep + (is_v ? L::kScaleStep / 2 : 0) + blk * D,
                 ln * 16, sc);
    }
  };
  // Keys 32 st.. of half `half` into the first buffer: rounded K, its rests, V
  // likewise; rows of V that are not there as 0.  A wave has eight of K's keys or
  // of V's.  True if one of V's groups is not finite and `full` is not so.
  constexpr uint32_t kPart = 32 * D * 2;
  auto turn_codes = [&](int half, int st, bool full, uint64_t there) {
    int ln = lane;
    asm("" : "+v"(ln));  // (the offsets made anew: registers are short)
    const int key0 = 32 * st + 8 * blk;
    const unsigned char* const from =
        lds + (2 + half) * P::kStep + (is_v ? P::kStep / 2 : 0) + key0 * D;
    const unsigned char* const sc = lds + L::kScales + half * L::kScaleStep +
                                    (is_v ? L::kScaleStep / 2 : 0) + key0 * (D / kKvGroup * 2);
    bool odd = false;
#pragma unroll 1
    for (int i = 0; i < (RQ < 8 ? 8 / RQ : 1); ++i) {
      const int r = i * RQ + ln / CQ, c = ln % CQ;  // of the eight keys
      if (RQ > 8 && r >= 8) break;
      const u32x4 x = *reinterpret_cast<const u32x4*>(from + r * D + c * 16);
      uint32_t scale =
          *reinterpret_cast<const uint16_t*>(sc + r * (D / kKvGroup * 2) + (c / 2) * 2);
      if (!full && is_v) odd |= finite_scale(scale, there >> (key0 + r) & 1);
      const h2 d = scale2(scale);
      uint32_t w[4][2], y[4][2];
#pragma unroll
      for (int j = 0; j < 4; ++j) decode4(x[j], d, w[j], y[j]);
      const int row = 8 * blk + r;  // of the 32 keys
      const uint32_t s0 = ((2 * c) ^ swz<D>(row & 15)) << 4, s1 = ((2 * c + 1) ^ swz<D>(row & 15)) << 4;
      unsigned char* const to = lds + (is_v ? P::kStep : 0) + row * (D * 2);
      *reinterpret_cast<u32x4*>(to + s0) = (u32x4){w[0][0], w[0][1], w[1][0], w[1][1]};
      *reinterpret_cast<u32x4*>(to + s1) = (u32x4){w[2][0], w[2][1], w[3][0], w[3][1]};
      *reinterpret_cast<u32x4*>(to + kPart + s0) = (u32x4){y[0][0], y[0][1], y[1][0], y[1][1]};
      *reinterpret_cast<u32x4*>(to + kPart + s1) = (u32x4){y[2][0], y[2][1], y[3][0], y[3][1]};
    }
    return !full && is_v && __any(odd);
  };
  // Rows of V that are not there become 0, and so do infinities and NaN: true if
  // there are any.  For the 16 rows that the calling wave has brought to buffer b.
  auto clean_v = [&](uint32_t b, uint32_t there) {
    unsigned char* vb = lds + b + mine;
    bool odd = false;
#pragma unroll 1
    for (int i = 0; i < NI; ++i) {
      u32x4* at = reinterpret_cast<u32x4*>(vb + i * 1024 + 16 * lane);
      u32x4 w = *at;
      odd |= finite8(w, there >> (i * RPI + lane / CH) & 1);
      *at = w;
    }
    return __any(odd);
  };
  if (threadIdx.x == 0) *odds = 0;
  if (wave == NW - 1 && a.parent) see_tree(a, t.win, t.len, lane, place, seen);

  h8 qf[RT][KK];
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
  const uint32_t koff = t.k_offset(), voff = t.v_offset();

  // Keys 32 st.. of a step, `halves` times 32 of them, K's and V's operands from
  // kbase and vbase on, kPart between the halves; with rests, kPart behind the values.
  auto compute = [&](int step, int st, uint32_t kbase, uint32_t vbase, bool full, uint64_t there,
                     auto rests, auto halves) {
    constexpr int kParts = decltype(rests)::value ? 2 : 1, H = decltype(halves)::value;
    asm("" : "+v"(kbase), "+v"(vbase));  // (the pieces' places made anew: registers)
    f4 s[2 * H][RT];
#pragma unroll
    for (int b = 0; b < 2 * H; ++b)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[b][rt] = (f4){0.f, 0.f, 0.f, 0.f};
    // K's pieces, of the two blocks in turn, kAhead of them under way: what LDS
    // takes to answer eight waves is longer than the products of one or two
    h8 kn[kAhead];
    constexpr int kPieces = 2 * KK * kParts * H;
    auto k_read = [&](int f) {
      const int g = f % (2 * KK), part = f / (2 * KK);  // (a half, or the rests)
      return t.k_frag(P::k_piece(kbase, (g >> 1) % P::KO) + part * kPart, g >> 1, g & 1);
    };
#pragma unroll
    for (int f = 0; f < kAhead; ++f) kn[f] = k_read(f);
#pragma unroll
    for (int f = 0; f < kPieces; ++f) {
      const h8 kf = kn[f % kAhead];
      const int g = f % (2 * KK), b = (kParts == 1 ? f / (2 * KK) * 2 : 0) + (g & 1);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        s[b][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][g >> 1], s[b][rt], 0, 0, 0);
      if (f + kAhead < kPieces) kn[f % kAhead] = k_read(f + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
    bool move = false;
    float top[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int b = 0; b < 2 * H; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[b][rt][i] = __builtin_fmaf(s[b][rt][i], a.scale_log2, -mref[rt]);
      if (!full) {
        const bool tree = cold_slide()->parent;
        const int node = t.node_of(row0 + rt * 16 + col);
        const int pos = tree ? place[node] : t.len + node;
        const uint64_t up = tree ? seen[node] : 0;
#pragma unroll
        for (int b = 0; b < 2 * H; ++b) {
          const uint32_t see = t.seen4(step, 32 * st + 16 * b + 4 * grp, there, pos, up);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[b][rt][i] = see >> i & 1 ? s[b][rt][i] : -INFINITY;
        }
      }
      top[rt] = s[0][rt][0];
#pragma unroll
      for (int b = 0; b < 2 * H; ++b) {
        top[rt] = max3(top[rt], s[b][rt][0], s[b][rt][1]);
        top[rt] = max3(top[rt], s[b][rt][2], s[b][rt][3]);
      }
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
        for (int b = 0; b < 2 * H; ++b) s[b][rt] -= by;
      }
    }
    h8 pf[H][RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            pf[h][rt][4 * b + i] = static_cast<_Float16>(__builtin_amdgcn_exp2f(s[2 * h + b][rt][i]));
#pragma unroll
        for (int i = 0; i < 8; i += 2) sum = weight_sum((h2){pf[h][rt][i], pf[h][rt][i + 1]}, sum);
      }
      l[rt] += sum;
    }
    h8 vn[kAhead];
    constexpr int kTiles = DT * kParts * H;
    auto v_read = [&](int f) {  // (tile after tile, a tile's rests behind its values; a half after the other)
      const int part = kParts == 2 ? f % 2 : f / DT, d = kParts == 2 ? f / 2 : f % DT;
      return t.v_frag(P::v_tile(vbase, d) + part * kPart, 0);
    };
#pragma unroll
    for (int f = 0; f < kAhead; ++f) vn[f] = v_read(f);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < kTiles; ++f) {
      const h8 vf = vn[f % kAhead];
      const int d = kParts == 2 ? f / 2 : f % DT, h = kParts == 2 ? 0 : f / DT;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[h][rt], acc[rt][d], 0, 0, 0);
      if (f + kAhead < kTiles) vn[f % kAhead] = v_read(f + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  P::settle_q(qf);
  int step = t.begin, it = 0;
  const int cached_end = min(t.end, t.steps.cached);
  if constexpr (Q8) {
    if (step < cached_end) {
      Rows rows = t.rows_of(step);
      bring_codes(rows, 0);
      for (; step < cached_end; ++it) {
        const uint32_t ok = rows.ok;
        const bool full = t.full(step, ok);
        const uint64_t there = full ? ~0ull : t.present(step, ok);
        const int next = t.steps.skip(step + 1);
        wait_vm();
        bar();  // the codes are here, nobody reads the first buffer (and the flags are cleared)
        if (next < cached_end) {
          rows = t.rows_of(next);
          bring_codes(rows, (it + 1) & 1);
        }
#pragma unroll 1
        for (int st = 0; st < 2; ++st) {
          if (st > 0) bar();  // nobody reads the first 32 keys any more
          if (turn_codes(it & 1, st, full, there)) *odds = 1;
          bar();  // everybody's keys are there
          compute(step, st, koff, voff, full, there, std::true_type(), std::integral_constant<int, 1>());
        }
        step = next;
      }
    }
  }
  if (step < t.end) {
    // the buffers in turn, the second first: the first may still be read
    Rows rows;
    rows.ok = 15u;
    if (!Q8 && step < t.steps.cached) rows = t.rows_of(step);
    if (Q8) bar();  // (codes in the second one are read)
    bring(step, rows, 2 * P::kStep);
    if (!Q8 || it == 0) bar();  // the flags are cleared, the tree is there
    for (uint32_t b = 2 * P::kStep; step < t.end; b ^= 2 * P::kStep, ++it) {
      const bool cached = !Q8 && step < t.steps.cached;
      const uint32_t ok = rows.ok;
      const bool full = cached ? t.full(step, ok) : t.full_window(step);
      const uint64_t there = full ? ~0ull : t.present(step, ok);
      const int next = t.steps.skip(step + 1);
      rows.ok = 15u;
      if (!Q8 && next < cached_end) rows = t.rows_of(next);
      wait_vm();
      if (is_v && !full && clean_v(b, static_cast<uint32_t>(there >> (16 * blk)) & 0xFFFFu))
        *odds = 1;
      bar();  // everybody's copies of this step are here, and nobody reads the other buffer
      if (next < t.end) bring(next, rows, b ^ 2 * P::kStep);
#pragma unroll 1
      for (int st = 0; st < 2; st += kHalves)
        compute(step, st, koff + b + st * kPart, voff + b + st * kPart, full, there,
                std::false_type(), std::integral_constant<int, kHalves>());
      step = next;
    }
  }

  // (the last step's barrier is behind the last flag)
  if (t.begin < t.end && *odds) {
    int pos[RT];
    uint64_t up[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int node = t.node_of(row0 + rt * 16 + col);
      pos[rt] = a.parent ? place[node] : t.len + node;
      up[rt] = a.parent ? seen[node] : 0;
    }
    add_odds<D, Q8>(t, acc, 4 * grp, pos, up);
  }
  int last_col = col;
  asm("" : "+v"(last_col));  // (the rows made anew: registers)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + last_col;
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    const float lt = a.parent && !seen[t.node_of(r)] ? 0.f : l[rt];  // 0: an absent node
    t.template store<DT, 16>(r, 4 * grp, acc[rt], mref[rt], lt, grp == 0);
  }
}

// The parts of many rows, joined as attn_join_kernel does it, which has a workgroup
// for each row: here D / 4 lanes have a row and read its parts one after the
// other, those in which it sees something (2,048 tokens of 16 heads of 256 in two
// to four parts, with no cache: 98 us in all, 147 by a workgroup each).
template <int D>
__global__ void __launch_bounds__(256) slide_join_kernel(const AttnArgs a) {
  constexpr int LP = D / 4, U = 4;  // lanes of a row, parts at once
  const int per = a.max_window * a.n_heads;
  const long long x = blockIdx.x * (256LL / LP) + threadIdx.x / LP;
  const int seq = static_cast<int>(x / per);
  if (seq >= a.n_seq) return;
  const int rest = static_cast<int>(x - static_cast<long long>(seq) * per);
  const int node = rest / a.n_heads, head = rest - node * a.n_heads;
  const Window w = window_of(a.win_off, seq, a.n_tokens, a.max_window);
  const int2 plan = a.seq_plan[seq];  // the first unit, the parts
  if (node >= w.n || plan.y <= 1) return;
  const int h = head / a.group, r = node * a.group + head - h * a.group;
  const int rb = r / a.block_rows;
  const long long at =
      (static_cast<long long>(plan.x + h * plan.y) * a.row_blocks + rb) * a.block_rows + r -
      rb * a.block_rows;
  const long long step = static_cast<long long>(a.row_blocks) * a.block_rows;
  const int c = threadIdx.x % LP * 4;
  const float* po = a.part_o + at * D + c;
  float m = -INFINITY, sum = 0.f;
  f4 o = (f4){0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < plan.y; s0 += U) {
    f4 v[U];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) ml[u] = a.part_ml[at + min(s0 + u, plan.y - 1) * step];
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= plan.y) ml[u].y = 0.f;
      top = ml[u].y != 0.f ? fmaxf(top, ml[u].x) : top;
      v[u] = (f4){0.f, 0.f, 0.f, 0.f};
      if (ml[u].y != 0.f) v[u] = *reinterpret_cast<const f4*>(po + (s0 + u) * step * D);
    }
    const float f0 = m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 0.f;
    sum *= f0;
    o *= f0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = ml[u].y != 0.f ? __builtin_amdgcn_exp2f(ml[u].x - top) : 0.f;
      sum += ml[u].y != 0.f ? ml[u].y * f : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += ml[u].y != 0.f ? v[u][i] * f : 0.f;
    }
    m = top;
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  h4 z;
#pragma unroll
  for (int j = 0; j < 4; ++j) z[j] = static_cast<_Float16>(o[j] * inv);
  const long long row = static_cast<long long>(w.off + node) * a.n_heads + head;
  *reinterpret_cast<h4*>(a.out + row * D + c) = z;
}

// ---- host -----------------------------------------------------------------------

// Steps at the most: of `nodes` tokens in line that see each other and `before` of the window.
static long long slide_steps(int max_len, int reach, int sinks, long long before, long long nodes) {
  const long long keys = static_cast<long long>(max_len) + before;
  const long long near = static_cast<long long>(reach) + nodes + sinks + 2 * kKeys;
  return ((keys < near ? keys : near) + kKeys - 1) / kKeys + 1;
}
// Workgroups of few rows that a CU holds at once, and units of `row_blocks` of
// them that the card does, an XCD's 32 CUs with whole ones (32 sequences of one
// token and of five over 4,000 quantised ones, 8 kv heads of 128: 59.8 and 69.4
// us by 3 a CU, 62.0 and 80.0 by 4, 58.6 and 72.6 by 2; of 64: 41 us by 4, 48 by
// 2; four tokens over 131,071, 2 kv heads of 256: 43.8 by 2, 58.3 by 4).
static int slide_few_each(int dim) { return dim == 256 ? 2 : dim == 128 ? 3 : 4; }
static long long slide_units(int each, long long row_blocks) {
  return 32 * each >= row_blocks ? 32 * each / row_blocks * 8 : 8;
}
constexpr int kMostUnits = 0x1FFFFF;    // sequences times kv heads of a call
constexpr int kMostRows = 0x7FFFF000;   // tokens of a window times query heads of a kv head
static int slide_join_steps(int dim) { return dim / 64 + 1; }  // what a join of wide blocks costs
constexpr int kFewJoinSteps = 8;                               // of blocks of few rows
static size_t slide_plan_bytes(int n_seq) {
  return (static_cast<size_t>(n_seq) * sizeof(int2) + 15) / 16 * 16;
}

// How a call is laid out: rows of a workgroup, the most units.
struct SlideLayout {
  int block_rows, row_blocks, max_units, goal;
  bool cut, by_rows;  // by_rows: how parts are joined
  int spread;
  size_t plan_bytes, o_bytes, bytes;  // of the workspace
};
static SlideLayout slide_layout(int n_seq, int max_window, int max_len, int group, int n_kv, int dim,
                                int reach, int sinks) {
  SlideLayout l;
  const long long rows = static_cast<long long>(max_window) * group;
  const long long units = static_cast<long long>(n_seq) * n_kv;
  // steps at the most: of a sequence, and of a block of 256 of its rows (a window
  // that may be a tree lies in every block's reach); and over the blocks in the mean
  auto steps = [&](long long before, long long nodes) {
    return slide_steps(max_len, reach, sinks, before, nodes);
  };
  const bool chain = max_window > kMaxWindow;
  const long long most = steps(max_window, max_window);
  const long long own = chain ? steps(max_window, 256 / group + 1) : most;
  const long long mean = chain ? steps(max_window / 2, 256 / group + 1) : most;
  // 256 rows read a step's keys once and keep the matrix cores busy, but 32 rows
  // spread little work further: by 256 as soon as each CU has two such steps (in
  // us, 32 rows and 256: 32 sequences of 64 nodes, 32 query heads on 8, over 300
  // keys of 128 quantised values 70 and 43, 4 of 32 nodes, 64 on 8, over 32,768
  // 494 and 322; 8 of 64 nodes that reach 128 keys back, 48 on 8, 24 and 32).
  const long long wide_units = 2 * 256 / ((rows + 255) / 256 * mean) + 1;
  const bool wide = rows > 128 && units >= wide_units;
  l.block_rows = wide ? 256 : rows > 16 ? 32 : 16;
  l.row_blocks = static_cast<int>((rows + l.block_rows - 1) / l.block_rows);
  const long long blocks = units * l.row_blocks;
  const bool near_only = reach / 2 < max_len / 2 + max_window / 2;
  // workgroups that the card holds at once, and units of them
  const int each = wide ? 1 : slide_few_each(dim);
  const long long slots = 256 * each;
  const long long per = slide_units(each, l.row_blocks);
  // Less work than the card holds is cut into parts if that saves more steps than
  // the parts' way through memory and the join cost, `join` of them (of a chunk's
  // blocks of 256 rows the last sees `own` steps, all together `mean` a block);
  // blocks that see few of their sequence's steps would get empty parts.  More than
  // it holds, in blocks of few rows, is cut over long caches, so that a ragged batch
  // ends together.  (28 sequences of up to 210 tokens, 56 query heads on 8 of 128,
  // that reach 63 keys back: 340 us in parts, 88 whole; 600 batches of mixed shapes:
  // twice `join` costs 1 to 2% more.)
  const long long join = wide ? slide_join_steps(dim) : kFewJoinSteps;
  const long long room = own > join ? slots * (own - join) / (wide ? mean : own) : 0;  // of blocks: below it
  const bool rounds = blocks >= 2 * slots;
  l.cut = own * 2 >= most && (blocks < room || (!wide && blocks >= slots && most > kFewJoinSteps));
  // (blocks of 256 rows: as many parts as all CUs take, of the blocks that see something
  // of a part; of four steps or more: 1,024 tokens over none, 16 heads on 2 of 256, 48
  // us, 68 with parts of two)
  const long long all_goal = slots * own / mean / l.row_blocks, most_goal = units * own / 4;
  const long long wide_goal = all_goal < most_goal ? all_goal : most_goal > units ? most_goal : units;
  if (wide && n_seq == 1 && wide_goal < 2 * units) l.cut = false;  // (it would not come to it)
  l.spread = l.row_blocks < 8 ? kSpreadUnits : near_only && !l.cut ? kSpreadRuns : kSpreadTurns;
  long long n = units;
  l.goal = 1;
  if (l.cut && wide) {
    l.goal = static_cast<int>(wide_goal);
    n = l.goal + (n_seq <= 64 ? 0 : units);
  } else if (l.cut && !rounds) {
    n = (2 * units + per - 1) / per * per;
    // (a part a head lost to rounding; one in a thousand less: parts_of rounds)
    l.goal = static_cast<int>(n_seq <= 64 ? n : n - units - ((n - units) >> 10));
  } else if (l.cut) {
    n = units + per;
    l.goal = static_cast<int>(per - ((per + 1023) >> 10));
  }
  // many rows of few parts: a workgroup of the join has several rows, one after the other
  l.by_rows = wide && l.goal < 8 * units;
  l.max_units = n > 0x7FFFFF00 ? 0x7FFFFF00 : static_cast<int>(n);
  const size_t part_rows =
      static_cast<size_t>((l.max_units + 7LL) / 8 * 8) * l.row_blocks * l.block_rows;
  l.plan_bytes = l.cut ? slide_plan_bytes(n_seq) : 0;
  l.o_bytes = l.cut ? part_rows * dim * sizeof(float) : 0;
  l.bytes = l.plan_bytes + l.o_bytes + (l.cut ? part_rows * sizeof(float2) : 0);
  return l;
}

// Bytes that no layout of at most n_seq sequences, windows of max_window and caches of max_len
// passes: a smaller call may be cut where a larger one is not, into more parts of more row blocks.
// So all numbers of row blocks are gone through, each with the most units that slide_layout has of it.
static size_t slide_workspace(int n_seq, int max_window, int max_len, int group, int n_kv, int dim,
                              int reach, int sinks) {
  n_seq = std::min(n_seq, kMostUnits / n_kv);
  max_window = std::min(max_window, kMostRows / group);
  if (n_seq == 0 || max_window == 0) return 0;  // (no such call)
  const long long rows = static_cast<long long>(max_window) * group;
  const long long near = std::min(max_window, kMaxWindow);  // of what may be a tree
  auto steps = [&](int len, long long before, long long nodes) {
    return slide_steps(len, reach, sinks, before, nodes);
  };
  long long part_rows = 0;
  auto take = [&](long long units, long long row_blocks, int block_rows) {
    part_rows = std::max(part_rows, (units + 7) / 8 * 8 * row_blocks * block_rows);
  };
  // Blocks of few rows.  Over 128 rows they have no more than 512 steps of 256 rows, those of
  // the mean row over no cache at the least.
  const long long in_line = std::max(max_window, 256 / group + 1);  // (a chain's block may count more)
  if (steps(max_len, max_window, in_line) > kFewJoinSteps) {
    const int each = slide_few_each(dim), block = rows > 16 ? 32 : 16;
    for (long long rb = (group + block - 1) / block; rb <= (rows + block - 1) / block; ++rb) {
      const long long least = (rb - 1) * block + 1, nodes = (least + group - 1) / group;
      const long long per = slide_units(each, rb);
      long long n = n_seq;
      if (least > 128) {
        long long mean = nodes > kMaxWindow ? LLONG_MAX : steps(0, nodes, nodes);
        if (max_window > kMaxWindow) {
          const long long w = std::max(nodes, kMaxWindow + 1LL);
          mean = std::min(mean, steps(0, w / 2, 256 / group + 1));
        }
        n = std::min(n, 512 / ((least + 255) / 256 * mean) / n_kv);
        if (n == 0) break;
      }
      const long long two = (2 * 256 * each - 1) / rb / n_kv;  // less than two rounds
      if (const long long few = std::min(n, two)) take((2 * few * n_kv + per - 1) / per * per, rb, block);
      if (n > two) take(n * n_kv + per, rb, block);
    }
  }
  // Blocks of 256 rows: fewer than CUs times the last block's steps over the mean's, which is
  // two at the most in a chain and one in what may be a tree.
  for (long long rb = (group + 255) / 256; rows > 128 && rb <= (rows + 255) / 256; ++rb) {
    const long long w = std::min<long long>(rb * 256 / group, max_window);
    const long long quota = w > kMaxWindow ? 512 : 256;
    long long own = steps(max_len, std::min(w, near), std::min(w, near));
    if (w > kMaxWindow) own = std::max(own, steps(max_len, w, 256 / group + 1));
    const long long n = std::min<long long>((quota - 1) / rb / n_kv, n_seq), units = n * n_kv;
    if (n == 0) break;
    const long long goal = std::min(quota / rb, std::max(units * own / 4, units));
    if (own > slide_join_steps(dim) && (n > 1 || goal >= 2 * units))
      take(goal + (n > 64 ? units : 0), rb, 256);
  }
  return part_rows == 0 ? 0
                        : slide_plan_bytes(n_seq) +
                              static_cast<size_t>(part_rows) * (dim * sizeof(float) + sizeof(float2));
}

// Workgroups of the launches, and their threads.
static long long slide_grid(const SlideLayout& l) {
  const long long n = l.spread == kSpreadUnits ? (l.max_units + 7LL) / 8 * 8 : l.max_units;
  return (n * l.row_blocks + 7) / 8 * 8;
}
static int slide_threads(const SlideLayout& l) {
  return l.block_rows == 256 ? 64 * kSlideRowWaves : 256;
}
static long long slide_join_groups(const SlideLayout& l, long long rows, int dim) {
  return l.by_rows ? (rows * (dim / 4) + 255) / 256 : rows;
}
static int slide_join_threads(const SlideLayout& l, int dim) { return l.by_rows ? 256 : 2 * dim; }

template <int D, bool Q8>
static int slide_launch(const SlideArgs& a, const SlideLayout& l, hipStream_t s, const char* nm) {
  static_assert(kJoinThreads<D> == 2 * D, "the limit of the join's launch counts on it");
  const dim3 grid(static_cast<unsigned>(slide_grid(l))), threads(slide_threads(l));
  if (a.block_rows == 256)
    hipLaunchKernelGGL((slide_rows_kernel<D, Q8>), grid, threads,
                       SlideRowsLds<D>::kBytes, s, a);
  else if (a.block_rows == 32)
    hipLaunchKernelGGL((slide_few_kernel<D, 2, Q8>), grid, threads, (SlideFewLds<D, 2, Q8>::kBytes), s,
                       a);
  else
    hipLaunchKernelGGL((slide_few_kernel<D, 1, Q8>), grid, threads, (SlideFewLds<D, 1, Q8>::kBytes), s,
                       a);
  if (int st = check_launch(nm)) return st;
  if (!l.cut) return SG_OK;
  const long long rows = static_cast<long long>(a.n_seq) * a.max_window * a.n_heads;
  const dim3 groups(static_cast<unsigned>(slide_join_groups(l, rows, D)));
  const dim3 of(slide_join_threads(l, D));
  if (l.by_rows)
    hipLaunchKernelGGL(slide_join_kernel<D>, groups, of, 0, s, static_cast<const AttnArgs&>(a));
  else
    hipLaunchKernelGGL(attn_join_kernel<D>, groups, of, 0, s, static_cast<const AttnArgs&>(a));
  return check_launch(nm);
}

// What the cache is apart from its tables: whether out lies over it, and its layer.
static bool over_layer(const uint16_t* out, long long n, const sg_kv_cache* c, long long at,
                       long long values) {
  return overlap(out, n, c->k + at, values) || overlap(out, n, c->v + at, values);
}
static bool over_layer(const uint16_t* out, long long n, const sg_kv_cache_q8* c, long long at,
                       long long values) {
  return overlap(out, n, c->k + at, values) || overlap(out, n, c->v + at, values) ||
         overlap(out, n, c->k_scale + at / kKvGroup, values / kKvGroup) ||
         overlap(out, n, c->v_scale + at / kKvGroup, values / kKvGroup);
}
static void set_layer(SlideArgs& a, const sg_kv_cache* c, long long at) {
  a.kc = c->k + at;
  a.vc = c->v + at;
  a.ks = a.vs = nullptr;
}
static void set_layer(SlideArgs& a, const sg_kv_cache_q8* c, long long at) {
  a.kc = reinterpret_cast<const uint16_t*>(c->k + at);
  a.vc = reinterpret_cast<const uint16_t*>(c->v + at);
  a.ks = c->k_scale + at / kKvGroup;
  a.vs = c->v_scale + at / kKvGroup;
}

template <typename C>
static int attn_slide(const uint16_t* q, const uint16_t* k, const uint16_t* v, long long q_stride,
                      long long k_stride, long long v_stride, const C* cache, int layer,
                      const int* win_off, const int* parent, uint16_t* out, void* ws,
                      size_t ws_bytes, int n_seq, int n_tokens, int max_window, int max_len,
                      int n_heads, float scale, int reach, int sinks, void* stream,
                      const char* nm) {
  constexpr bool kQ8 = std::is_same<C, sg_kv_cache_q8>::value;
  if (!q || !k || !v || !win_off || !out)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: null pointer", nm);
  if (int st = check_cache(cache, n_seq, n_tokens, max_window, nm, parent ? kMaxWindow : 1 << 24))
    return st;
  const int n_kv = cache->n_kv_heads, dim = cache->head_dim;
  if (layer < 0 || layer >= cache->n_layers || max_len < 0 || n_heads <= 0 || n_heads % n_kv != 0)
    return set_error(SG_ERR_GEOMETRY, "%s: layer=%d of %d, max_len=%d, n_heads=%d of %d kv heads",
                     nm, layer, cache->n_layers, max_len, n_heads, n_kv);
  if (reach < 0 || sinks < 0)
    return set_error(SG_ERR_GEOMETRY, "%s: reach=%d or sinks=%d is negative", nm, reach, sinks);
  if (max_len > 0x7FFFF000)
    return set_error(SG_ERR_UNSUPPORTED, "%s: max_len=%d is too long", nm, max_len);
  // token positions are 32-bit, the windows' too
  if ((static_cast<long long>(cache->pages_per_seq) << log2_of(cache->page_size)) + max_window >
      0x7FFFF000LL)
    return set_error(SG_ERR_UNSUPPORTED, "%s: a sequence of %d pages and a window of %d is too long",
                     nm, cache->pages_per_seq, max_window);
  // (a row's pieces of 16 B lie anywhere in memory; LDS copies need them aligned)
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 || k_stride % 8 ||
      v_stride % 8 || reinterpret_cast<uintptr_t>(q) % 2 || reinterpret_cast<uintptr_t>(out) % 8)
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: k and v must be 16-B aligned, out 8-B", nm);
  if (q_stride < static_cast<long long>(n_heads) * dim ||
      k_stride < static_cast<long long>(n_kv) * dim || v_stride < static_cast<long long>(n_kv) * dim)
    return set_error(SG_ERR_GEOMETRY, "%s: a token stride is less than a token", nm);
  // (a few tokens' rows are reached by 32-bit offsets)
  if (k_stride >= 1LL << 27 || v_stride >= 1LL << 27)
    return set_error(SG_ERR_UNSUPPORTED, "%s: a token stride of 2^27 or more", nm);
  // each launch has less than 2^32 threads (windows of max_window count, whether they are there
  // or not), each of which looks through the sequences; a window's rows are 32-bit
  const long long units = static_cast<long long>(n_seq) * n_kv;
  const long long rows = static_cast<long long>(max_window) * (n_heads / n_kv);
  if (rows > kMostRows || units > kMostUnits)
    return set_error(SG_ERR_UNSUPPORTED, "%s: too many sequences, or too long windows", nm);
  const int far = reach == 0 ? 0x7FFFFFFF : reach;
  const SlideLayout l =
      slide_layout(n_seq, max_window, max_len, n_heads / n_kv, n_kv, dim, far, sinks);
  if (slide_grid(l) > 0xFFFFFFFFLL / slide_threads(l) ||
      (l.cut && slide_join_groups(l, units * rows, dim) > 0xFFFFFFFFLL / slide_join_threads(l, dim)))
    return set_error(SG_ERR_UNSUPPORTED, "%s: too many sequences, or too long windows", nm);
  const long long last = n_tokens - 1, n_out = static_cast<long long>(n_tokens) * n_heads * dim;
  if (overlap(out, n_out, q, last * q_stride + n_heads * dim) ||
      overlap(out, n_out, k, last * k_stride + n_kv * dim) ||
      overlap(out, n_out, v, last * v_stride + n_kv * dim))
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: out overlaps q, k or v", nm);
  if (l.bytes && (!ws || ws_bytes < l.bytes || reinterpret_cast<uintptr_t>(ws) % 16))
    return set_error(SG_ERR_INVALID_ARGUMENT, "%s: the workspace needs %zu bytes, 16-B aligned", nm,
                     l.bytes);
  const long long at = layer * cache->layer_stride;
  const long long values = static_cast<long long>(cache->n_pages) * n_kv * cache->page_size * dim;
  if (over_layer(out, n_out, cache, at, values) ||
      overlap(out, n_out, cache->pages, static_cast<long long>(n_seq) * cache->pages_per_seq) ||
      overlap(out, n_out, cache->length, n_seq) || overlap(out, n_out, win_off, n_seq + 1LL) ||
      overlap(out, n_out, parent, n_tokens) ||
      overlap(out, n_out, static_cast<unsigned char*>(ws), static_cast<long long>(l.bytes)))
    return set_error(SG_ERR_INVALID_ARGUMENT,
                     "%s: out overlaps the cache, win_off, parent or the workspace", nm);
  SlideArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  set_layer(a, cache, at);
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
  a.spread = l.spread;
  a.turn_units = l.max_units / static_cast<int>(units) * static_cast<int>(units);
  a.scale_log2 = scale * kLog2e;
  a.reach = far;
  a.sinks = sinks;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dim == 64) return slide_launch<64, kQ8>(a, l, s, nm);
  if (dim == 128) return slide_launch<128, kQ8>(a, l, s, nm);
  return slide_launch<256, kQ8>(a, l, s, nm);
}

}  // namespace sg

extern "C" {

size_t sg_attn_sliding_workspace_bytes(int n_seq, int max_window, int max_len, int n_heads,
                                       int n_kv_heads, int head_dim, int reach, int sinks) {
  if (n_seq <= 0 || max_window <= 0 || max_len < 0 || n_kv_heads <= 0 || n_heads <= 0 ||
      n_heads % n_kv_heads != 0 || reach < 0 || sinks < 0)
    return 0;
  return sg::slide_workspace(n_seq, max_window, max_len, n_heads / n_kv_heads, n_kv_heads, head_dim,
                             reach == 0 ? 0x7FFFFFFF : reach, sinks);
}

int sg_attn_sliding_f16(const uint16_t* q, const uint16_t* k, const uint16_t* v, long long q_stride,
                        long long k_stride, long long v_stride, const sg_kv_cache* cache, int layer,
                        const int* win_off, const int* parent, uint16_t* out, void* ws,
                        size_t ws_bytes, int n_seq, int n_tokens, int max_window, int max_len,
                        int n_heads, float scale, int reach, int sinks, void* stream) {
  return sg::attn_slide(q, k, v, q_stride, k_stride, v_stride, cache, layer, win_off, parent, out,
                        ws, ws_bytes, n_seq, n_tokens, max_window, max_len, n_heads, scale, reach,
                        sinks, stream, "sg_attn_sliding_f16");
}

int sg_attn_sliding_q8(const uint16_t* q, const uint16_t* k, const uint16_t* v, long long q_stride,
                       long long k_stride, long long v_stride, const sg_kv_cache_q8* cache, int layer,
                       const int* win_off, const int* parent, uint16_t* out, void* ws,
                       size_t ws_bytes, int n_seq, int n_tokens, int max_window, int max_len,
                       int n_heads, float scale, int reach, int sinks, void* stream) {
  return sg::attn_slide(q, k, v, q_stride, k_stride, v_stride, cache, layer, win_off, parent, out,
                        ws, ws_bytes, n_seq, n_tokens, max_window, max_len, n_heads, scale, reach,
                        sinks, stream, "sg_attn_sliding_q8");
}

}  // extern "C"
