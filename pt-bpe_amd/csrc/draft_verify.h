// draft_verify.h -- verification of drafted tokens against the target's probabilities.
//
//   c = 0, r = p_0, Z = 1
//   for i = 1 .. N - 1 with parent(i) = c, x = ids[i]:
//     u[i] q_c(x) Z < r(x):  accept: c = i, r = p_i, Z = 1
//     else:                  r <- max(r - Z q_c, 0), Z = sum r
//   next id: the smallest x with sum_{y <= x} r(y) > u[0] sum r;  r without mass: from p_c
//
// Children come after their parents, so one ascending pass visits every context's children.
// Without draft rows q_c is one at the drafted id: r loses that entry.  Probabilities are read
// as they are (finite positive entries, others 0); sums, products and comparisons are in 64 bits,
// so an id near a border of two of them does not hang on the order of the sums.
#pragma once

#include "draft.h"

namespace gb {

struct VerifyArgs {
  const int32_t* parents;
  const void* ids;  // int32 or int64
  const void *target, *draft;
  const float* u;
  const int32_t *ranges, *start;
  int32_t *n, *path, *tokens;
  int64_t parents_stride, ids_stride, u_stride;
  int64_t ts[2], ds[2];  // target / draft strides: (seq, node)
  int32_t B, N, V, C;    // C: rows of ranges (0: none)
  int32_t ids64;
};

constexpr int VER_BLOCK = 1024;
constexpr int VER_TILES = 1024;  // tile sums in LDS

// 16 bytes of a row that is aligned to its elements only
template <typename T>
struct alignas(sizeof(T)) VerVec {
  T v[16 / sizeof(T)];
};

template <typename T>
__device__ inline double prob(T v) {
  const float f = (float)v;
  return f > 0.f && f < INFINITY ? (double)f : 0.0;
}

// sum over the block; every thread gets it.  red: 17 doubles of LDS.
__device__ inline double block_sum(double v, double* red) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = v;
  __syncthreads();
  if (threadIdx.x < 64) {
    double s = threadIdx.x < VER_BLOCK / 64 ? red[threadIdx.x] : 0.0;
    for (int o = 8; o; o >>= 1) s += __shfl_xor(s, o);
    if (threadIdx.x == 0) red[16] = s;
  }
  __syncthreads();
  return red[16];
}

template <typename T>
struct VerRow {
  const T *p, *q;
  int lo, hi;       // entries outside are 0
  int rejected;     // siblings rejected so far
  const double* Z;  // their Z (LDS)
  const int* x;     // their ids (LDS)

  // r at the VEC entries from i on (0 past hi)
  template <bool Q>
  __device__ void load(int i, double* r) const {
    constexpr int VEC = 16 / sizeof(T);
    VerVec<T> vp, vq;
    if (i + VEC <= hi) {
      vp = *(const VerVec<T>*)(p + i);
      if (Q && rejected) vq = *(const VerVec<T>*)(q + i);
    } else {
      for (int k = 0; k < VEC; k++) {
        vp.v[k] = i + k < hi ? p[i + k] : (T)0.f;
        vq.v[k] = Q && rejected && i + k < hi ? q[i + k] : (T)0.f;
      }
    }
    for (int k = 0; k < VEC; k++) {
      double v = prob(vp.v[k]);
      if (Q) {
        if (rejected) {
          const double w = prob(vq.v[k]);
          for (int j = 0; j < rejected; j++) v = fmax(v - Z[j] * w, 0.0);
        }
      } else {
        for (int j = 0; j < rejected; j++)
          if (x[j] == i + k) v = 0.0;
      }
      r[k] = v;
    }
  }
};

// One workgroup per sequence.
template <typename T, bool Q>
__global__ __launch_bounds__(VER_BLOCK) void k_verify(VerifyArgs a) {
  constexpr int VEC = 16 / sizeof(T), TILE = VER_BLOCK * VEC;
  __shared__ int par[DRAFT_MAX_NODES], depth[DRAFT_MAX_NODES], rejx[DRAFT_MAX_NODES], id[DRAFT_MAX_NODES];
  __shared__ float u[DRAFT_MAX_NODES];
  __shared__ double P[DRAFT_MAX_NODES], Qx[DRAFT_MAX_NODES], Z[DRAFT_MAX_NODES + 1], red[17], tile[VER_TILES];
  __shared__ int next_;
  const int t = threadIdx.x, b = blockIdx.x, N = a.N;
  const T* target = (const T*)a.target + b * a.ts[0];
  const T* draft = (const T*)a.draft + b * a.ds[0];
  const int start = a.C ? a.start[b] : 0;
  if (t < N) {
    par[t] = a.parents[b * a.parents_stride + t];
    const int64_t x = a.ids64 ? ((const int64_t*)a.ids)[b * a.ids_stride + t] : ((const int32_t*)a.ids)[b * a.ids_stride + t];
    id[t] = x < 0 || x >= a.V ? -1 : (int)x;
    u[t] = a.u[b * a.u_stride + t];
  }
  __syncthreads();
  auto range = [&](int d, int& lo, int& hi) {
    lo = 0;
    hi = a.V;
    if (!a.C) return;
    int c = (int)(((int64_t)start + d) % a.C);
    if (c < 0) c += a.C;
    lo = max(a.ranges[2 * c], 0);
    hi = min(a.ranges[2 * c + 1], a.V);
  };
  if (t < N) {
    const int d = draft_depth(par, t);
    depth[t] = d;
    double pv = 0, qv = Q ? 0 : 1;
    if (t && d > 0 && id[t] >= 0) {
      int lo, hi;
      range(d - 1, lo, hi);
      if (id[t] >= lo && id[t] < hi) {
        pv = prob(target[par[t] * a.ts[1] + id[t]]);
        if (Q) qv = prob(draft[par[t] * a.ds[1] + id[t]]);
      }
    }
    P[t] = pv;
    Qx[t] = qv;
  }
  __syncthreads();
  int32_t* path = a.path + (int64_t)b * N;
  int32_t* tokens = a.tokens + (int64_t)b * N;
  if (depth[0] < 0) {
    if (t < N) path[t] = tokens[t] = -1;
    if (t == 0) a.n[b] = 0;
    return;
  }
  VerRow<T> row;
  int c = 0, n = 1;
  auto context = [&](int node) {
    c = node;
    row.p = target + node * a.ts[1];
    row.q = draft + node * a.ds[1];
    range(n - 1, row.lo, row.hi);
    row.rejected = 0;
    row.Z = Z;
    row.x = rejx;
  };
  // the tiles' sums of r into tile[], all of it returned
  auto sum_row = [&]() {
    const int tiles = row.hi > row.lo ? (row.hi - row.lo + TILE - 1) / TILE : 0;
    for (int k = 0; k < tiles; k++) {
      double r[VEC], s = 0;
      const int i = row.lo + k * TILE + t * VEC;
      row.template load<Q>(i, r);
      for (int j = 0; j < VEC; j++) s += r[j];
      s = block_sum(s, red);
      if (t == 0) tile[k] = s;
    }
    __syncthreads();
    double s = 0;
    for (int k = 0; k < tiles; k++) s += tile[k];
    return s;
  };
  if (t == 0) {
    path[0] = 0;
    Z[0] = 1.0;
  }
  context(0);
  __syncthreads();
  for (int i = 1; i < N; i++) {
    if (depth[i] < 0 || par[i] != c) continue;
    double r = P[i];
    for (int j = 0; j < row.rejected; j++)
      r = Q ? fmax(r - Z[j] * Qx[i], 0.0) : (rejx[j] == id[i] ? 0.0 : r);
    if ((double)u[i] * Qx[i] * Z[row.rejected] < r) {
      if (t == 0) {
        path[n] = i;
        tokens[n - 1] = id[i];
      }
      n++;
      context(i);
    } else {
      __syncthreads();  // (others may still read the last context's rejected ids)
      if (t == 0) rejx[row.rejected] = id[i];
      row.rejected++;
      __syncthreads();
      const double s = sum_row();
      if (t == 0) Z[row.rejected] = s;
      __syncthreads();
    }
  }
  double s = sum_row();
  if (!(s > 0)) {
    row.rejected = 0;
    s = sum_row();
  }
  // the tile, then the entry
  const double at = (double)u[0] * s;
  const int tiles = row.hi > row.lo ? (row.hi - row.lo + TILE - 1) / TILE : 0;
  if (t == 0) next_ = -1;
  double before = 0;
  int k = 0;
  if (s > 0) {
    int last = 0;
    for (int j = 0; j < tiles; j++)
      if (tile[j] > 0) last = j;
    for (; k < last; k++) {
      if (before + tile[k] > at) break;
      before += tile[k];
    }
    double r[VEC], mine = 0;
    const int i = row.lo + k * TILE + t * VEC;
    row.template load<Q>(i, r);
    for (int j = 0; j < VEC; j++) mine += r[j];
    // inclusive scan over the block: within the waves, then the waves' totals
    double inc = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(inc, o);
      if (t % 64 >= o) inc += y;
    }
    __syncthreads();
    if (t % 64 == 63) red[t / 64] = inc;
    __syncthreads();
    double base = before;
    for (int w = 0; w < t / 64; w++) base += red[w];
    base += inc - mine;
    // the first entry whose sum passes; where rounding lets none pass, the tile's last entry with mass
    int first = INT32_MAX, lastx = -1;
    for (int j = 0; j < VEC; j++) {
      base += r[j];
      if (r[j] > 0) {
        lastx = i + j;
        if (base > at && first == INT32_MAX) first = i + j;
      }
    }
    for (int o = 32; o; o >>= 1) {
      first = min(first, __shfl_xor(first, o));
      lastx = max(lastx, __shfl_xor(lastx, o));
    }
    int* fl = (int*)tile;  // (the tile sums are done with)
    __syncthreads();
    if (t % 64 == 0) {
      fl[t / 64] = first;
      fl[16 + t / 64] = lastx;
    }
    __syncthreads();
    if (t == 0) {
      for (int w = 1; w < 16; w++) {
        first = min(first, fl[w]);
        lastx = max(lastx, fl[16 + w]);
      }
      next_ = first != INT32_MAX ? first : lastx;
    }
  }
  __syncthreads();
  if (t == 0) {
    tokens[n - 1] = next_;
    a.n[b] = n;
  }
  if (t >= n && t < N) path[t] = tokens[t] = -1;
}

}  // namespace gb
