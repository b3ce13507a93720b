// draft_attend.h -- attention of a drafted tree over a paged cache.
//
//   o[b,i,h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q[b,i,h] . k_j)
//
// j runs over the cache's positions 0 .. lens[b] - 1 (of kv head h / G) and the nodes on the path
// from the root to i.  An absent node's row is 0.
#pragma once

#include "draft.h"

namespace gb {

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;

struct AttendArgs {
  const void *q, *kc, *vc, *kd, *vd;
  void* out;
  const int32_t *table, *lens, *parents;
  int64_t qs[3], kcs[3], vcs[3], kds[3], vds[3];  // strides: (seq, node, head) / (page, slot, head)
  int64_t table_stride, parents_stride;
  int32_t B, N, Hq, Hkv, D, S, P, M;  // S: page size, P: pages, M: table entries a sequence
  PageDiv div;
  float scale;
};

constexpr int ATT_BLOCK = 256;

__device__ inline float wave_max(float v) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ inline float wave_sum(float v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// One workgroup per (sequence, node, query head): 256 keys at a time, one thread a key for the
// scores, one thread a channel for the sum.
template <typename T>
__global__ __launch_bounds__(ATT_BLOCK) void k_attend_row(AttendArgs a) {
  __shared__ int par[DRAFT_MAX_NODES];
  __shared__ int path[DRAFT_MAX_NODES];
  __shared__ float q[256], w[ATT_BLOCK], red[8];
  __shared__ int64_t row[ATT_BLOCK];
  __shared__ int depth_, bad_;
  const int t = threadIdx.x, h = blockIdx.x % a.Hq, i = blockIdx.x / a.Hq, b = blockIdx.y;
  const int kh = h / (a.Hq / a.Hkv);
  T* out = (T*)a.out + (((int64_t)b * a.N + i) * a.Hq + h) * a.D;
  for (int n = t; n < a.N; n += ATT_BLOCK) par[n] = a.parents[b * a.parents_stride + n];
  for (int d = t; d < a.D; d += ATT_BLOCK)
    q[d] = (float)((const T*)a.q)[b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + d] * a.scale;
  int len = a.lens[b];
  const int64_t cap = (int64_t)a.M * a.S;
  if (t == 0) bad_ = len < 0 || len > cap;
  __syncthreads();
  if (t == 0) {
    const int d = draft_depth(par, i);
    depth_ = d;
    for (int n = i, k = d; k >= 0; k--) {
      path[k] = n;
      n = par[n];
    }
  }
  __syncthreads();
  const int depth = depth_;
  if (depth < 0) {
    for (int d = t; d < a.D; d += ATT_BLOCK) out[d] = (T)0.f;
    return;
  }
  if (len < 0) len = 0;
  if (len > cap) len = (int)cap;
  const int64_t keys = (int64_t)len + depth + 1;
  const Pages pages = {a.table + b * a.table_stride, a.div, a.P, a.M};
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int64_t k0 = 0; k0 < keys; k0 += ATT_BLOCK) {
    const int64_t k = k0 + t;
    float s = -INFINITY;
    int64_t vrow = -1;
    if (k < len) {
      int slot;
      const int id = find_page(pages, (int)k, slot);
      if (id < 0) {
        bad_ = 1;
      } else {
        const T* kp = (const T*)a.kc + id * a.kcs[0] + slot * a.kcs[1] + kh * a.kcs[2];
        vrow = id * a.vcs[0] + slot * a.vcs[1] + kh * a.vcs[2];
        s = 0.f;
        for (int d = 0; d < a.D; d++) s = fmaf(q[d], (float)kp[d], s);
      }
    } else if (k < keys) {
      const int n = path[k - len];
      const T* kp = (const T*)a.kd + b * a.kds[0] + n * a.kds[1] + kh * a.kds[2];
      vrow = b * a.vds[0] + n * a.vds[1] + kh * a.vds[2];
      s = 0.f;
      for (int d = 0; d < a.D; d++) s = fmaf(q[d], (float)kp[d], s);
    }
    float wm = wave_max(s);
    if (t % 64 == 0) red[t / 64] = wm;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float e = s == -INFINITY ? 0.f : expf(s - mn);
    const float ws = wave_sum(e);
    w[t] = e;
    row[t] = vrow;
    if (t % 64 == 0) red[4 + t / 64] = ws;
    __syncthreads();
    const float f = m == -INFINITY ? 0.f : expf(m - mn);
    m = mn;
    l = l * f + (red[4] + red[5] + red[6] + red[7]);
    o *= f;
    if (t < a.D) {
      const int n = (int)(keys - k0 < ATT_BLOCK ? keys - k0 : ATT_BLOCK);
      for (int j = 0; j < n; j++) {
        if (row[j] < 0) continue;
        const T* v = (k0 + j < len ? (const T*)a.vc : (const T*)a.vd) + row[j];
        o = fmaf(w[j], (float)v[t], o);
      }
    }
    __syncthreads();
  }
  if (t < a.D) out[t] = (T)(bad_ ? NAN : o / l);
}

}  // namespace gb
