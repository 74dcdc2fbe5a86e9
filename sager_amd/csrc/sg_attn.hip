// sg_attn.hip - the windows' attention over a paged fp16 cache, and the
// accepted tokens' way into it.
//
// For a kv head, the rows of a product are (node, query head of the group):
// S^T = K Q^T and O^T = V^T P^T, 32 keys at a time and wave.  With keys as
// the first product's rows, a lane of v_mfma_f32_16x16x32_f16 gets four
// consecutive keys of one query row (keys 4g..4g+3 of each 16, g = lane / 16),
// and since the order of a product's 32 terms is free, those eight weights
// are the second product's operand as they are: p never leaves its lane.  V's
// operand then is, per lane, one column of V at the same eight keys, which
// ds_read_b64_tr_b16 reads from V's rows as they lie in memory.
//
// The running maximum is a reference point `mref` per row that moves only
// when a score passes it by 2^15: p = 2^(s - mref) fits fp16 (its largest
// value is 2^16), and 2^(8+15) below it is still a normal number.  l = sum p
// is kept per lane and joined at the end.
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

constexpr int kTile = 32;          // keys of a wave's step
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
  int n_split, split_keys, row_blocks;
  float scale_log2;
};

// The cached tokens of sequence s that the page table can hold.
__device__ __forceinline__ int cached_len(const int* __restrict__ length, int s, int page_log2,
                                          int pages_per_seq) {
  const long long cap = static_cast<long long>(pages_per_seq) << page_log2;
  const long long len = length[s];
  return static_cast<int>(len < 0 ? 0 : len > cap ? cap : len);
}

// Where chunk c (16 B) of key row r lies in its row: rows are a multiple of
// 128 B apart, so 16 rows read at one chunk would share their banks.
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
template <int N>
__device__ __forceinline__ void wait_vm_upto() {
  static_assert(N < 64, "the counter's range");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4 << 14));
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ const uint16_t* shfl_ptr(const uint16_t* p, int src) {
  const uint64_t v = reinterpret_cast<uintptr_t>(p);
  const uint32_t lo = __shfl(static_cast<uint32_t>(v), src);
  const uint32_t hi = __shfl(static_cast<uint32_t>(v >> 32), src);
  return reinterpret_cast<const uint16_t*>(static_cast<uintptr_t>(hi) << 32 | lo);
}

// One tile of a wave: which of its keys there are, and whether it needs more
// than the plain path (a page boundary past 16 keys, an absent page, the
// window's keys, keys past the end).
struct TileKind {
  uint32_t present;  // bit r: key r of the tile exists
  bool plain;
};

template <int D, int RT>
struct Attn {
  static constexpr int CH = D / 8;         // 16-B chunks of a row
  static constexpr int RPI = 64 / CH;      // rows of a copy instruction
  static constexpr int NI = kTile / RPI;   // copy instructions of a tile
  static constexpr int DT = D / 16;        // 16-column tiles of the output
  static constexpr int KK = D / 32;        // steps of the first product
  static constexpr uint32_t kTileBytes = kTile * D * 2;

  const AttnArgs& a;
  int lane, col, grp;
  int seq, h, len, total;  // cached keys, cached + window
  Window win;
  const int* table;
  uint32_t kbuf, vbuf;  // LDS byte addresses of this wave's buffers
  const unsigned char* lds;

  __device__ __forceinline__ const uint16_t* cache_row(const uint16_t* c, int page, int slot) const {
    const long long at =
        ((static_cast<long long>(page) * a.n_kv + h) << a.page_log2) + slot;
    return c + at * D;
  }
  __device__ __forceinline__ bool page_ok(int p) const {
    return static_cast<uint32_t>(p) < static_cast<uint32_t>(a.n_pages);
  }

  // Issues the copies of a tile's K (or V) rows; returns its kind.
  template <bool kV>
  __device__ __forceinline__ TileKind issue(int tile) const {
    const int j0 = tile * kTile;
    const uint16_t* c = kV ? a.vc : a.kc;
    const uint32_t buf = kV ? vbuf : kbuf;
    TileKind kind{0xFFFFFFFFu, false};
    if (j0 + kTile <= len) {  // pages of 16 hold half a tile, larger ones all of it
      const const_int_p ids = (const_int_p)(table);
      const int p0 = ids[j0 >> a.page_log2];
      const int p1 = ids[(j0 + 16) >> a.page_log2];
      if (page_ok(p0) && page_ok(p1)) {
        kind.plain = true;
        const int mask = (1 << a.page_log2) - 1;
        const uint16_t* b0 = uniform_ptr(cache_row(c, p0, j0 & mask));
        const uint16_t* b1 = uniform_ptr(cache_row(c, p1, (j0 + 16) & mask) - 16 * D);
        const int sub = lane / CH;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = i * RPI + sub;
          const uint32_t voff = row * (D * 2) + (((lane % CH) ^ swz<D>(row)) << 4);
          dma16_base(buf + i * 1024, voff, i * RPI < 16 ? b0 : b1);
        }
        return kind;
      }
    }
    // lane r (and r + 32) finds key r
    const int j = j0 + (lane & 31);
    const uint16_t* w = kV ? a.v : a.k;
    const long long ws = kV ? a.v_stride : a.k_stride;
    const uint16_t* src = w + static_cast<long long>(win.off) * ws + h * D;
    bool there = false;
    if (j < len) {
      const int p = table[j >> a.page_log2];
      there = page_ok(p);
      if (there) src = cache_row(c, p, j & ((1 << a.page_log2) - 1));
    } else if (j < total) {
      there = true;
      src += static_cast<long long>(j - len) * ws;
    }
    kind.present = static_cast<uint32_t>(__ballot(there));
#pragma unroll 2
    for (int i = 0; i < NI; ++i) {
      const int row = i * RPI + lane / CH;
      const uint16_t* s = shfl_ptr(src, row);
      dma16_ptr(buf + i * 1024, s + ((lane % CH) ^ swz<D>(row)) * 8);
    }
    return kind;
  }
};

// One workgroup of four waves: one part of a sequence's keys, one kv head, a
// block of 16 RT rows.  The waves take the part's tiles in turn, each with
// its own K and V buffer in LDS, so that no barrier orders them: while a
// wave multiplies by V, its next K is under way, and the other way round.
template <int D, int RT>
__global__ void __launch_bounds__(256) attn_tree_kernel(const AttnArgs a) {
  typedef Attn<D, RT> A;
  constexpr int CH = A::CH, RPI = A::RPI, NI = A::NI, DT = A::DT, KK = A::KK;
  constexpr int kRows = 16 * RT;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  A t{a};
  t.lane = threadIdx.x & 63;
  t.col = t.lane & 15;
  t.grp = t.lane >> 4;
  int id = blockIdx.x;
  const int split = id % a.n_split;
  id /= a.n_split;
  const int rb = id % a.row_blocks;
  id /= a.row_blocks;
  t.h = id % a.n_kv;
  t.seq = id / a.n_kv;
  t.win = window_of(a.win_off, t.seq, a.n_tokens, a.max_window);
  const int rows = t.win.n * a.group;
  if (rb * kRows >= rows) return;
  t.len = cached_len(a.length, t.seq, a.page_log2, a.pages_per_seq);
  t.total = t.len + t.win.n;
  t.table = a.pages + static_cast<long long>(t.seq) * a.pages_per_seq;
  t.lds = lds;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) unsigned char*)lds));
  t.kbuf = lds0 + wave * 2 * A::kTileBytes;
  t.vbuf = t.kbuf + A::kTileBytes;
  const unsigned char* kb = lds + wave * 2 * A::kTileBytes;
  unsigned char* vb = lds + wave * 2 * A::kTileBytes + A::kTileBytes;

  const int tiles = (t.total + kTile - 1) / kTile;
  const int per = a.split_keys / kTile;
  const long long first = static_cast<long long>(split) * per;
  const int t_end = split == a.n_split - 1 ? tiles
                                           : static_cast<int>(first + per < tiles ? first + per : tiles);
  int tile = first + wave < t_end ? static_cast<int>(first) + wave : t_end;

  TileKind kind{0, true};
  if (tile < t_end) {
    t.template issue<false>(tile);
    kind = t.template issue<true>(tile);
  }

  // Q's rows, while the first copies are under way
  const uint64_t up_all = ancestors(a.parent, t.win, t.lane);
  h8 qf[RT][KK];
  uint64_t up[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rb * kRows + rt * 16 + t.col;
    const int node = r / a.group, g = r - node * a.group;
    up[rt] = __shfl(up_all, r < rows ? node : 0);
    const uint16_t* qp = a.q + static_cast<long long>(t.win.off + (r < rows ? node : 0)) * a.q_stride +
                         (t.h * a.group + (r < rows ? g : 0)) * D;
#pragma unroll
    for (int s = 0; s < KK; ++s) {
      u32x4 w = *reinterpret_cast<const u32x4_u*>(qp + s * 32 + t.grp * 8);
      if (r >= rows) w = (u32x4){0, 0, 0, 0};
      qf[rt][s] = __builtin_bit_cast(h8, w);
    }
  }

  f4 acc[RT][DT];
  float mref[RT], l[RT];
  bool begun[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    mref[rt] = 0.f;
    l[rt] = 0.f;
    begun[rt] = false;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[rt][d] = (f4){0.f, 0.f, 0.f, 0.f};
  }

  while (tile < t_end) {
    const int next = tile + 4;
    wait_vm_upto<NI>();  // K is here; V's NI copies may be under way
    f4 s[2][RT];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[kt][rt] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < KK; ++st)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int row = kt * 16 + t.col;
        const h8 kf = *reinterpret_cast<const h8*>(kb + row * (D * 2) +
                                                   (((st * 4 + t.grp) ^ swz<D>(row)) << 4));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          s[kt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][st], s[kt][rt], 0, 0, 0);
      }
    const TileKind now = kind;
    wait_lds();
    if (next < t_end) t.template issue<false>(next);

    float e[RT][8];
    bool move = false;
    float top[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        e[rt][i] = __builtin_fmaf(s[i >> 2][rt][i & 3], a.scale_log2, -mref[rt]);
      if (!now.plain) {
        // bit r of `see`: key r is there and this lane's row sees it
        const int w0 = tile * kTile - t.len;  // key 0's window node, if not negative
        const uint32_t tree = w0 >= 0    ? static_cast<uint32_t>(up[rt] >> w0)
                              : w0 > -32 ? static_cast<uint32_t>(up[rt] << -w0) | ((1u << -w0) - 1)
                                         : 0xFFFFFFFFu;
        const uint32_t see = (now.present & tree) >> (4 * t.grp);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          e[rt][i] = see & 1u << ((i >> 2) * 16 + (i & 3)) ? e[rt][i] : -INFINITY;
      }
      top[rt] = e[rt][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top[rt] = fmaxf(top[rt], e[rt][i]);
      move |= top[rt] > kRise || (!begun[rt] && top[rt] > -INFINITY);
    }
    if (__any(move)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float m = fmaxf(top[rt], __shfl_xor(top[rt], 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const bool set = m > kRise || (!begun[rt] && m > -INFINITY);
        const float by = set ? m - kBelow : 0.f;
        const float f = !set ? 1.f : begun[rt] ? __builtin_amdgcn_exp2f(-by) : 0.f;
        mref[rt] += by;
        l[rt] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[rt][d] *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[rt][i] -= by;
        begun[rt] |= set;
      }
    }
    h8 p[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[rt][i] = __builtin_amdgcn_exp2f(e[rt][i]);
        p[rt][i] = static_cast<_Float16>(e[rt][i]);
      }
      l[rt] += ((e[rt][0] + e[rt][1]) + (e[rt][2] + e[rt][3])) +
               ((e[rt][4] + e[rt][5]) + (e[rt][6] + e[rt][7]));
    }

    if (next < t_end)
      wait_vm_upto<NI>();  // V is here; the next K's copies may be under way
    else
      wait_vm_upto<0>();
    if (!now.plain) {
      // Rows that no query sees become 0 (0 times what lies there need not
      // be 0).  A window row that some queries see and others do not is
      // looked through for infinities and NaN: they are taken out for the
      // product and added to the queries that see them, one by one.
      const int j0 = tile * kTile;
      bool odd = false;
#pragma unroll 2
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + t.lane / CH;
        u32x4* at = reinterpret_cast<u32x4*>(vb + i * 1024 + 16 * t.lane);
        if (!(now.present >> row & 1)) {
          *at = (u32x4){0, 0, 0, 0};
        } else if (j0 + row >= t.len && t.win.n > 1) {
          const u32x4 w = *at;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            odd |= (w[c] & 0x7C00u) == 0x7C00u || (w[c] & 0x7C000000u) == 0x7C000000u;
        }
      }
      wait_lds();
      if (__any(odd)) {
        for (int r = 0; r < kTile; ++r) {
          if (!(now.present >> r & 1) || j0 + r < t.len) continue;
          const int from = t.col + 16 * ((r & 15) >> 2);  // the lane that has key r's weight
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            float mine = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i == ((r >> 4) * 4 + (r & 3))) mine = e[rt][i];
            const float w = __shfl(mine, from);
            const bool see = up[rt] >> (j0 + r - t.len & 63) & 1;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int c = d * 16 + 4 * t.grp + i;
                const uint16_t b = *reinterpret_cast<const uint16_t*>(
                    vb + r * (D * 2) + (((c >> 3) ^ swz<D>(r)) << 4) + (c & 7) * 2);
                acc[rt][d][i] += see && (b & 0x7C00) == 0x7C00 ? w * half_bits_to_float(b) : 0.f;
              }
          }
        }
        wait_lds();
        for (int i = 0; i < NI; ++i) {
          const int row = i * RPI + t.lane / CH;
          if (j0 + row < t.len) continue;
          uint16_t* at = reinterpret_cast<uint16_t*>(vb + i * 1024 + 16 * t.lane);
          for (int c = 0; c < 8; ++c)
            if ((at[c] & 0x7C00) == 0x7C00) at[c] = 0;
        }
        wait_lds();
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      h8 vf;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int row = kt * 16 + 4 * t.grp + (t.col >> 2);
        const uint32_t off = row * (D * 2) + (((2 * d + ((t.col & 3) >> 1)) ^ swz<D>(row)) << 4) +
                             (t.col & 1) * 8;
        const h4 x = __builtin_bit_cast(
            h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s4_p)(static_cast<uintptr_t>(t.vbuf + off))));
#pragma unroll
        for (int i = 0; i < 4; ++i) vf[kt * 4 + i] = x[i];
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[rt], acc[rt][d], 0, 0, 0);
    }
    wait_lds();
    if (next < t_end) kind = t.template issue<true>(next);
    tile = next;
  }

  // Join the four waves: O = sum over waves of O_w 2^(mref_w - m).  A wave's
  // 16-B pieces of O lie at piece ^ row, against bank conflicts.
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
  }
  __syncthreads();
  float* ob = reinterpret_cast<float*>(lds);
  float* ml = ob + 4 * kRows * D;  // [wave][row]: mref, then [wave][row]: l
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rt * 16 + t.col;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<f4*>(ob + (wave * kRows + r) * D + (((d * 4 + t.grp) ^ t.col) << 2)) =
          acc[rt][d];
    if (t.grp == 0) {
      // (a row whose scores are all NaN has not begun either, but counts)
      ml[wave * kRows + r] = begun[rt] || l[rt] != l[rt] ? mref[rt] : -INFINITY;
      ml[(4 + wave) * kRows + r] = up[rt] ? l[rt] : 0.f;
    }
  }
  __syncthreads();
  constexpr int kPieces = D / 4;
  for (int x = threadIdx.x; x < kRows * kPieces; x += 256) {
    const int r = x / kPieces, piece = x % kPieces;
    const int rr = rb * kRows + r;
    if (rr >= rows) break;
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w * kRows + r]);
    f4 o = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = ml[w * kRows + r], lw = ml[(4 + w) * kRows + r];
      if (mw > -INFINITY && lw != 0.f) {
        const float f = __builtin_amdgcn_exp2f(mw - m);
        sum += lw * f;
        o += *reinterpret_cast<const f4*>(ob + (w * kRows + r) * D + ((piece ^ (r & 15)) << 2)) * f;
      }
    }
    const int node = rr / a.group, g = rr - node * a.group;
    const long long at =
        static_cast<long long>(t.win.off + node) * a.n_heads + t.h * a.group + g;
    if (a.n_split == 1) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      h4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = static_cast<_Float16>(o[i] * inv);
      *reinterpret_cast<h4*>(a.out + at * D + piece * 4) = y;
    } else {
      const long long pa = static_cast<long long>(split) * a.n_tokens * a.n_heads + at;
      if (sum != 0.f) *reinterpret_cast<f4*>(a.part_o + pa * D + piece * 4) = o;
      if (piece == 0) a.part_ml[pa] = make_float2(m, sum);
    }
  }
}

// The parts of a split, joined: one wave per (token, head).
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a, int n_seq) {
  const int lane = threadIdx.x & 63;
  const long long x = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const long long per = static_cast<long long>(a.max_window) * a.n_heads;
  if (x >= per * n_seq) return;
  const int seq = static_cast<int>(x / per);
  const int rest = static_cast<int>(x - seq * per);
  const int node = rest / a.n_heads, head = rest - node * a.n_heads;
  const Window w = window_of(a.win_off, seq, a.n_tokens, a.max_window);
  if (node >= w.n) return;
  const long long at = static_cast<long long>(w.off + node) * a.n_heads + head;
  const long long step = static_cast<long long>(a.n_tokens) * a.n_heads;
  float m = -INFINITY;
  for (int s = lane; s < a.n_split; s += 64) {
    const float2 v = a.part_ml[at + s * step];
    if (v.y != 0.f) m = fmaxf(m, v.x);
  }
  m = wave_max_dpp(m);
  constexpr int E = D / 64;
  float o[E], sum = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  for (int s = 0; s < a.n_split; ++s) {
    const float2 v = a.part_ml[at + s * step];
    if (v.y == 0.f) continue;
    const float f = __builtin_amdgcn_exp2f(v.x - m);
    sum += v.y * f;
    const float* p = a.part_o + (at + s * step) * D + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] += p[i] * f;
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) a.out[at * D + lane * E + i] = f16b(o[i] * inv);
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
  int rt, row_blocks, n_split, split_keys;
};
static Cut attn_cut(int n_seq, int max_window, int max_len, int group, int n_kv, int dim) {
  Cut c;
  const int rows = max_window * group;
  c.rt = rows > 16 ? 2 : 1;
  c.row_blocks = (rows + 16 * c.rt - 1) / (16 * c.rt);
  const long long keys = static_cast<long long>(max_len) + max_window;
  const long long step = 4 * kTile;
  const long long most = (keys + step - 1) / step;
  const long long groups = static_cast<long long>(n_seq) * n_kv * c.row_blocks;
  const long long slots = 256 * (dim == 256 ? 1 : 2);
  long long n = groups >= slots ? 1 : slots / groups;
  if (n > most) n = most;
  c.split_keys = static_cast<int>((most + n - 1) / n * step);
  c.n_split = static_cast<int>((keys + c.split_keys - 1) / c.split_keys);
  return c;
}
static size_t part_bytes(const Cut& c, int n_tokens, int n_heads, int dim) {
  if (c.n_split == 1) return 0;
  return static_cast<size_t>(c.n_split) * n_tokens * n_heads * (dim * 4 + 8);
}

template <int D>
static int attn_launch(const AttnArgs& a, const Cut& c, int n_seq, long long grid, hipStream_t s,
                       const char* nm) {
  const size_t lds = 4 * 16 * c.rt * D * 4 + 2 * 4 * 16 * c.rt * 4;
  const size_t bufs = 4 * 2 * Attn<D, 1>::kTileBytes;
  const size_t bytes = lds > bufs ? lds : bufs;
  if (c.rt == 1)
    hipLaunchKernelGGL((attn_tree_kernel<D, 1>), dim3(static_cast<unsigned>(grid)), dim3(256),
                       bytes, s, a);
  else
    hipLaunchKernelGGL((attn_tree_kernel<D, 2>), dim3(static_cast<unsigned>(grid)), dim3(256),
                       bytes, s, a);
  if (int st = check_launch(nm)) return st;
  if (c.n_split > 1) {
    const long long waves = static_cast<long long>(n_seq) * a.max_window * a.n_heads;
    hipLaunchKernelGGL(attn_join_kernel<D>, dim3(static_cast<unsigned>((waves + 3) / 4)),
                       dim3(256), 0, s, a, n_seq);
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
  const long long grid = static_cast<long long>(n_seq) * n_kv * c.row_blocks * c.n_split;
  const long long join = static_cast<long long>(n_seq) * max_window * n_heads;
  if (grid > 0x7FFFFFFF || join > 0x7FFFFFFF)
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
  a.scale_log2 = scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dim == 64) return attn_launch<64>(a, c, n_seq, grid, s, nm);
  if (dim == 128) return attn_launch<128>(a, c, n_seq, grid, s, nm);
  return attn_launch<256>(a, c, n_seq, grid, s, nm);
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
