// draft.h -- the decoding operators' shared device code: the drafted tree, the paged cache's
// addresses.  Included once by draft.hip.
//
// A tree has N <= DRAFT_MAX_NODES nodes.  Node 0 is the last decided token: present when
// parents[0] == -1, else the whole sequence is absent.  Node i > 0 hangs on parents[i] when
// that is a present node of [0, i), else it is absent.
#pragma once

#include <stdint.h>

namespace gb {

constexpr int DRAFT_MAX_NODES = 128;
constexpr int DRAFT_MAX_POSITIONS = 0x7ffff000;  // a sequence's; some tiles of keys more stay an int32

// A node on the climb to the root: the nodes passed so far as bits of w, itself included, and where it goes on: up >= 0 at
// that node, -1: the root was reached, -2: none leads there.  All nodes climb at once, each on to where the one above it
// has got by then, so a way of up to 127 steps is done after 7 turns.  (Node by node a chain of 54 took 6 us.)
struct DraftNode {
  int up;
  uint32_t w[DRAFT_MAX_NODES / 32];
};
__device__ inline DraftNode draft_node(int i, int parent) {
  DraftNode n;
  n.up = i == 0 ? (parent == -1 ? -1 : -2) : (parent >= 0 && parent < i ? parent : -2);
  for (int k = 0; k < DRAFT_MAX_NODES / 32; k++) n.w[k] = i / 32 == k ? 1u << (i % 32) : 0u;
  return n;
}
__device__ inline void draft_climb(DraftNode& n, const DraftNode& above) {
  n.up = above.up;
  for (int k = 0; k < DRAFT_MAX_NODES / 32; k++) n.w[k] |= above.w[k];
}

// Which of a tree's tiles of DRAFT_TILE nodes hold a value that is not finite, in LDS.  A flag each: a wave may be at the next
// tile's before another has read this one's, and the barriers that follow hang on what is read.
constexpr int DRAFT_TILE = 64;
struct TileFlags {
  int of[DRAFT_MAX_NODES / DRAFT_TILE];
  __device__ void clear() {
    for (int& f : of) f = 0;
  }
  __device__ void mark(int node) { of[node / DRAFT_TILE] = 1; }
  __device__ bool marked(int node) const { return of[node / DRAFT_TILE] != 0; }
};

// x / d for 0 <= x < 2^31 and 1 <= d < 2^31, with the host's m = min(2^32 / d, 2^32 - 1) rounded down: x m / 2^32
// is at most x / d and below it by less than x / 2^32 < 1/2, so its floor is the quotient or one less, which the
// remainder tells.
struct PageDiv {
  uint32_t m;
  int32_t d;
};
// (also for the other divisions by a call's own sizes: a division proper takes some 100 cycles)
inline PageDiv page_div(int32_t d) { return {d == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / (uint32_t)d), d}; }
__device__ inline void page_split(PageDiv v, int x, int& page, int& slot) {
  const uint32_t q = __umulhi((uint32_t)x, v.m), r = (uint32_t)x - q * (uint32_t)v.d;
  const bool more = r >= (uint32_t)v.d;
  page = (int)(q + more);
  slot = (int)(more ? r - v.d : r);
}

// A sequence's row of the table: position x lies in slot x % S of page row[x / S].
struct Pages {
  const int32_t* row;  // M entries
  PageDiv div;
  int32_t P, M;
};
// the table's entry for 0 <= x < M S, as it is: good_page has to pass it before it is used
__device__ inline int page_entry(const Pages& t, int x, int& slot) {
  int k;
  page_split(t.div, x, k, slot);
  return t.row[k];
}
__device__ inline bool good_page(const Pages& t, int id) { return (uint32_t)id < (uint32_t)t.P; }
// for any x: the page, or -1 where the entry is none of the cache's P pages or x is not in the table (which
// is not read then)
__device__ inline int find_page(const Pages& t, int x, int& slot) {
  if (x < 0 || x / t.div.d >= t.M) return -1;
  const int id = page_entry(t, x, slot);
  return good_page(t, id) ? id : -1;
}

}  // namespace gb
