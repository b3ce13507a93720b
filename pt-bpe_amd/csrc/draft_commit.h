// draft_commit.h -- the accepted path's keys and values into the paged cache, every layer at once:
//
//   cache[layer, table[b, (len_b + t) / S], (len_b + t) % S] = draft[layer, b, path[b, t]],  t < n[b]
//   lens_out[b] = len_b + n[b]
#pragma once

#include "draft.h"

namespace gb {

struct CommitArgs {
  const char *kd, *vd;
  char *kc, *vc;
  const int32_t *table, *lens, *path, *n;
  int32_t* lens_out;
  int64_t kds[4], vds[4], kcs[4], vcs[4];  // byte strides: (layer, seq, node, head) / (layer, page, slot, head)
  int64_t table_stride, path_stride;
  int32_t L, B, N, Hkv, S, P, M;
  int32_t vecs;  // 16-byte pieces of one head's row
  PageDiv div;
};

struct alignas(16) Piece {
  uint32_t v[4];
};

// One workgroup per kept node and layer.  Measured against it: four layers a workgroup (3.1 us became 4.3 for one sequence,
// 64 sequences x 16 layers stayed at 27), four nodes a workgroup with one die for all of a sequence's layer (4.8, 28).
// What bounds the large case is not in here: 17 k rows of 2 KiB go to 4 k different places of 2 MiB each.
__global__ __launch_bounds__(256) void k_commit_nodes(CommitArgs a) {
  const int b = blockIdx.x / a.N, t = blockIdx.x - b * a.N, layer = blockIdx.y;
  const int len = a.lens[b], n = min(a.n[b], a.N);
  // a kept node outside the tree or the cache is not written, and the sequence's length becomes -1
  const Pages pages = {a.table + b * a.table_stride, a.div, a.P, a.M};
  auto place = [&](int k, int& node, int& id, int& slot) {
    node = a.path[b * a.path_stride + k];
    if (node < 0 || node >= a.N || len < 0 || len > INT32_MAX - k) return false;
    id = find_page(pages, len + k, slot);
    return id >= 0;
  };
  int node = 0, id = 0, slot = 0;
  if (t == 0 && layer == 0 && threadIdx.x < 64) {  // (a wave looks at all of them)
    bool ok = len >= 0 && a.n[b] <= a.N;
    for (int k = threadIdx.x; k < n; k += 64) ok &= place(k, node, id, slot);
    ok = __all(ok);
    if (threadIdx.x == 0) a.lens_out[b] = ok ? len + max(n, 0) : -1;
  }
  if (t >= n || !place(t, node, id, slot)) return;
  for (int k = threadIdx.x; k < a.Hkv * a.vecs; k += 256) {
    const int h = k / a.vecs, c = (k - h * a.vecs) * 16;
    const Piece x = *(const Piece*)(a.kd + layer * a.kds[0] + b * a.kds[1] + node * a.kds[2] + h * a.kds[3] + c);
    const Piece y = *(const Piece*)(a.vd + layer * a.vds[0] + b * a.vds[1] + node * a.vds[2] + h * a.vds[3] + c);
    *(Piece*)(a.kc + layer * a.kcs[0] + id * a.kcs[1] + slot * a.kcs[2] + h * a.kcs[3] + c) = x;
    *(Piece*)(a.vc + layer * a.vcs[0] + id * a.vcs[1] + slot * a.vcs[2] + h * a.vcs[3] + c) = y;
  }
}

}  // namespace gb
