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

// depth of node i (root: 0), -1 when it is absent.  par: the tree's parents (N of them, LDS).
// Every step goes to a smaller index, so the walk ends within i steps.
__device__ inline int draft_depth(const int* par, int i) {
  int d = 0;
  while (i > 0) {
    const int p = par[i];
    if (p < 0 || p >= i) return -1;
    i = p;
    d++;
  }
  return par[0] == -1 ? d : -1;
}

// x / d for 0 <= x < 2^31 and 1 <= d < 2^31, with the host's m = floor(2^32 / d) + 1: x m / 2^32 is
// at least x / d and above it by less than x / 2^32 < 1/2, so its floor is the quotient or one more,
// which the remainder's sign tells.
struct PageDiv {
  uint32_t m;
  int32_t d;
};
inline PageDiv page_div(int32_t d) { return {d == 1 ? 0u : (uint32_t)((1ull << 32) / (uint32_t)d + 1), d}; }
__device__ inline void page_split(PageDiv v, int x, int& page, int& slot) {
  if (v.d == 1) {
    page = x;
    slot = 0;
    return;
  }
  int q = (int)__umulhi((uint32_t)x, v.m);
  int r = (int)((uint32_t)x - (uint32_t)q * (uint32_t)v.d);
  if (r < 0) {
    q--;
    r += v.d;
  }
  page = q;
  slot = r;
}

// where position x of a sequence lies: slot and page, the page -1 where the table's entry is none of
// the cache's P pages or x is past the table's M entries.  Nothing is read outside the table.
struct Pages {
  const int32_t* row;  // the sequence's entries
  PageDiv div;
  int32_t P, M;
};
__device__ inline int find_page(const Pages& t, int x, int& slot) {
  int k;
  page_split(t.div, x, k, slot);
  if (x < 0 || k >= t.M) return -1;
  const int id = t.row[k];
  return id >= 0 && id < t.P ? id : -1;
}

}  // namespace gb
