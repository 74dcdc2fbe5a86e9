// sg_window.hpp - the windows of a speculative batch: which rows a sequence
// has, and who is whose ancestor in its tree of drafts.
#pragma once

#include "sg_common.hpp"

namespace sg {

constexpr int kMaxWindow = 64;  // nodes of a window: one lane, one mask bit each

// Rows of sequence s: [off, off + n), inside the buffers whatever win_off says.
struct Window {
  int off, n;
};
__device__ __forceinline__ Window window_of(const int* __restrict__ win_off, int s, int n_tokens,
                                            int max_window) {
  const int a = win_off[s], b = win_off[s + 1];
  Window w;
  w.off = a;
  w.n = a < 0 || a >= n_tokens || b <= a ? 0 : min(min(b - a, max_window), n_tokens - a);
  return w;
}

// The ancestors of node `lane` and itself as a mask of nodes, for the calling
// wave; 0 for a node that does not hang on the root (node 0).  `up` is the
// node's parent, or the node itself where it has none that counts.
// Pointer doubling: after r rounds a mask holds 2^r steps of the way up.
__device__ __forceinline__ uint64_t masks_up(int up, int n, int lane) {
  uint64_t m = 1ull << lane;
  for (int r = 1; r < n; r <<= 1) {
    m |= __shfl(m, up);
    up = __shfl(up, up);
  }
  return lane < n && (m & 1) ? m : 0;
}
// The parent of node `lane` in window w (itself: none).  parent NULL: a chain.
__device__ __forceinline__ int parent_of(const int* __restrict__ parent, Window w, int lane) {
  if (lane == 0 || lane >= w.n) return lane;
  if (!parent) return lane - 1;
  const int p = parent[w.off + lane];
  return p >= 0 && p < lane ? p : lane;
}
__device__ __forceinline__ uint64_t ancestors(const int* __restrict__ parent, Window w, int lane) {
  if (!parent) return lane < w.n ? (2ull << lane) - 1 : 0;
  return masks_up(parent_of(parent, w, lane), w.n, lane);
}

}  // namespace sg
