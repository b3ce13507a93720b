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

typedef uint32_t Piece __attribute__((ext_vector_type(4)));  // 16 bytes

// One workgroup per kept node and COMMIT_LAYERS layers, half of it for the keys and half for the values; a thread has
// one piece of every one of its layers on its way at a time.  Stores past the caches, for what is written is not read
// before the whole cache is.  64 sequences x 16 layers of 2 KiB rows, 71 MB read and written: with 1 / 2 / 4 / 8 / 16
// layers a workgroup 23 / 16 / 15.5 / 17 / 22 us, a copy's rate would be 14; with stores through the caches 27 at 1
// layer.  One sequence x 6 layers: 6.9 us with any, the call itself.
constexpr int COMMIT_LAYERS = 4;
__global__ __launch_bounds__(256) void k_commit_nodes(CommitArgs a) {
  const int b = blockIdx.x / a.N, t = blockIdx.x - b * a.N, layer = blockIdx.y * COMMIT_LAYERS;
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
  const bool values = threadIdx.x >= 128;
  const int64_t* ds = values ? a.vds : a.kds;
  const int64_t* cs = values ? a.vcs : a.kcs;
  const char* from = (values ? a.vd : a.kd) + layer * ds[0] + b * ds[1] + node * ds[2];
  char* to = (values ? a.vc : a.kc) + layer * cs[0] + id * cs[1] + slot * cs[2];
  const int64_t dl = ds[0], cl = cs[0], dh = ds[3], ch = cs[3];
  const int layers = min(COMMIT_LAYERS, a.L - layer);
  for (int k = threadIdx.x & 127; k < a.Hkv * a.vecs; k += 128) {
    const int h = k / a.vecs, c = (k - h * a.vecs) * 16;
    Piece x[COMMIT_LAYERS];
#pragma unroll
    for (int l = 0; l < COMMIT_LAYERS; l++)
      if (l < layers) x[l] = *(const Piece*)(from + l * dl + h * dh + c);
#pragma unroll
    for (int l = 0; l < COMMIT_LAYERS; l++)
      if (l < layers) __builtin_nontemporal_store(x[l], (Piece*)(to + l * cl + h * ch + c));
  }
}

}  // namespace gb
