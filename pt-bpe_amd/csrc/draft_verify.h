// draft_verify.h -- verification of drafted tokens against the target's probabilities.
//
//   c = 0, r = p_0, Z = 1
//   for i = 1 .. N - 1 with parent(i) = c, x = ids[i]:
//     u[i] q_c(x) Z < r(x):  accept: c = i, r = p_i, Z = 1
//     else:                  r <- max(r - Z q_c, 0), Z = sum r
//   next id: the smallest x with sum_{y <= x} r(y) > u[0] sum r;  r without mass: from p_c
//
// With ranges a row counts as what it is inside the range of its place, divided by its mass there: p / P, q / Q.  Kept
// times P, r still starts as the row's own entries; then Z = sum r / Q, P / Q at first (without draft rows sum r, P at first).
// A drafted id outside the range says nothing of those inside: it is passed over, as is every one of a draft row without
// mass there.  A P or Q that is 1 but for the type's rounding is taken as 1: rows that were normalised there are used as
// they are, as all are without ranges (so ranges that leave nothing out change nothing).
//
// Children come after their parents, so one ascending pass visits every context's children.
// Without draft rows q_c is one at the drafted id: r loses that entry.  Probabilities are read
// as they are (finite positive entries, others 0); sums, products and comparisons are in 64 bits,
// so an id near a border of two of them does not hang on the order of the sums.
//
// What has to be read: an entry of p and q for every node, and the rows of the contexts that a sum is needed of: the
// last one's for the next id, others' only between a rejected child and its next sibling, and with ranges once for P and Q
// of those with drafted children.  r is worked out anew from the rows and the Z so far whenever it is needed, never stored.
// One workgroup does a sequence: a row of 128 k entries takes it about as long as the rows' share of the card's bandwidth
// once there are 100 sequences: 128 chains of 7 drafts over 131072 fp32 entries take 33 us, 134 MB at 4.0 TB/s.  Small
// calls are dependent loads: one chain over 1091 ids 5.3 us, 48 trees of 40 nodes over 5123 ids held to ranges 18.6 (the
// longest walk: a sum for every context with children, and one per rejected sibling).
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

constexpr int VER_MAX_VOCAB = 1 << 22;
// up to here four waves do a sequence, above 16 (48 trees of 40 nodes over 5123 ids held to ranges: 18.8 us with four, 21.9
// with 16; one chain over 1091: 5.3 and 5.8)
constexpr int VER_SMALL = 8192;
// a sum that falls below this part of itself by subtraction is taken anew: the rest keeps 33 bits and more
constexpr double VER_KEEP = 1.0 / (1 << 20);

// 16 bytes of a row that is aligned to its elements only
template <typename T>
struct alignas(sizeof(T)) VerVec {
  T v[16 / sizeof(T)];
};

template <typename T>
__device__ inline float prob(T v) {
  const float f = (float)v;
  return __builtin_amdgcn_classf(f, 0x180) ? f : 0.f;  // positive, finite
}

// a mass as the rows are divided by it: a row normalised in 32 bits (2^-20 for its sums) and rounded once has 1 to within
// half a step of T
template <typename T>
__device__ inline double mass_of(double m) {
  constexpr double half = sizeof(T) == 4 ? 0x1p-24 : __is_same(T, _Float16) ? 0x1p-11 : 0x1p-8;
  return fabs(m - 1.0) <= half + 0x1p-20 ? 1.0 : m;
}

// a context's row with what its rejected children took
template <typename T, bool Q, bool HELD>
struct VerRow {
  static constexpr int VEC = 16 / sizeof(T);
  const T *p, *q;
  int lo, hi;       // entries outside are 0
  int rejected;     // children rejected so far
  const double* Z;  // their Z (LDS)
  const int* x;     // their ids (LDS)

  struct Raw {
    VerVec<T> p, q;
  };
  __device__ bool two() const { return Q && rejected; }
  // the VEC entries from i on (0 past end)
  __device__ void load(Raw& w, int i, int end) const {
    if (i + VEC <= end) {
      w.p = *(const VerVec<T>*)(p + i);
      if (two()) w.q = *(const VerVec<T>*)(q + i);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; k++) {
        w.p.v[k] = i + k < end ? p[i + k] : (T)0.f;
        if (two()) w.q.v[k] = i + k < end ? q[i + k] : (T)0.f;
      }
    }
  }
  __device__ void values(const Raw& w, int i, double* r) const {
    // entries that are no probabilities are rare: looked for all at once, as the bits above the largest finite value's
    float pv[VEC], qv[VEC];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < VEC; k++) {
      pv[k] = (float)w.p.v[k];
      qv[k] = two() ? (float)w.q.v[k] : 0.f;
      top = max(max(top, __float_as_uint(pv[k])), __float_as_uint(qv[k]));
    }
    if (__any(top > 0x7f7fffffu)) {
#pragma unroll
      for (int k = 0; k < VEC; k++) pv[k] = prob(pv[k]), qv[k] = prob(qv[k]);
    }
#pragma unroll
    for (int k = 0; k < VEC; k++) r[k] = pv[k];
    if (Q) {
      if (!HELD && rejected) {  // (Z of the first is 1)
#pragma unroll
        for (int k = 0; k < VEC; k++) r[k] = fmax(r[k] - (double)qv[k], 0.0);
      }
      for (int j = !HELD; j < rejected; j++) {
        const double z = Z[j];
#pragma unroll
        for (int k = 0; k < VEC; k++) r[k] = fmax(fma(-z, (double)qv[k], r[k]), 0.0);
      }
    } else {
      for (int j = 0; j < rejected; j++)
        if ((uint32_t)(x[j] - i) < (uint32_t)VEC)
#pragma unroll
          for (int k = 0; k < VEC; k++)
            if (x[j] == i + k) r[k] = 0.0;
    }
  }
  __device__ double sum(const Raw& w, int i) const {
    double r[VEC], s = 0;
    values(w, i, r);
#pragma unroll
    for (int k = 0; k < VEC; k++) s += r[k];
    return s;
  }
};

// v of the lane CTRL says (0 where it says none), for the lanes of the rows in MASK
template <int CTRL, int MASK>
__device__ inline double dpp(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, MASK, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, MASK, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// sums over the lanes up to each (rows of 16 lanes first, then the rows before), without LDS
__device__ inline double wave_scan(double v) {
  v += dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ inline double lane_value(double v, int l) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)u, l), hi = __builtin_amdgcn_readlane((int)(u >> 32), l);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double wave_total(double v) { return lane_value(wave_scan(v), 63); }
// a value of one lane (the same for the whole wave)
__device__ inline float lane_value(float v, int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l)); }

// One workgroup of W waves per sequence.  Every wave holds the whole tree (nodes lane and lane + 64) and makes the same
// walk; they part only over the rows.  HELD: with ranges (a kernel of its own, for its sums of P and Q make the others' code
// longer: 5.9 us instead of 5.3 for one chain without ranges).
template <typename T, bool Q, bool HELD, int W>
__global__ __launch_bounds__(64 * W) void k_verify(VerifyArgs a) {
  typedef VerRow<T, Q, HELD> Row;
  constexpr int VEC = Row::VEC, STEP = 64 * VEC, DEEP = (Q && W > 4 ? 16 : 32) / VEC;  // steps in flight (with 16 waves 128 registers have to hold them)
  __shared__ double Z[DRAFT_MAX_NODES], part[W];
  __shared__ int rejx[DRAFT_MAX_NODES];
  __shared__ double rejr[Q ? 1 : DRAFT_MAX_NODES];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, b = blockIdx.x, N = a.N;
  const T* target = (const T*)a.target + b * a.ts[0];
  const T* draft = (const T*)a.draft + b * a.ds[0];
  const int start = HELD ? a.start[b] : 0;

  int par[2], id[2], up[2], depth[2];
  float u[2], P[2] = {0.f, 0.f}, q[2];
  for (int k = 0; k < 2; k++) {
    const int i = lane + 64 * k;
    par[k] = -2, id[k] = -1, u[k] = 0.f, q[k] = Q ? 0.f : 1.f;
    if (i < N) {
      par[k] = a.parents[b * a.parents_stride + i];
      const int64_t x =
          a.ids64 ? ((const int64_t*)a.ids)[b * a.ids_stride + i] : ((const int32_t*)a.ids)[b * a.ids_stride + i];
      id[k] = x < 0 || x >= a.V ? -1 : (int)x;
      u[k] = a.u[b * a.u_stride + i];
    }
    // up: a node on the way to the root, depth steps above; -1: none leads there
    up[k] = i == 0 ? (par[k] == -1 ? 0 : -1) : (par[k] >= 0 && par[k] < i ? par[k] : -1);
    depth[k] = i > 0;
  }
  auto of = [&](const int* v, int i) {  // node i's value, i of each lane's own
    const int x = __shfl(v[0], i & 63), y = N > 64 ? __shfl(v[1], i & 63) : 0;
    return i < 64 ? x : y;
  };
  while (__any(up[0] > 0 || up[1] > 0)) {  // twice the way each time
    int nu[2], nd[2];
    for (int k = 0; k < 2; k++) nu[k] = of(up, max(up[k], 0)), nd[k] = of(depth, max(up[k], 0));
    for (int k = 0; k < 2; k++)
      if (up[k] > 0) {
        depth[k] += nd[k];
        up[k] = nu[k];
      }
  }
  const bool root = __builtin_amdgcn_readfirstlane(up[0]) == 0;
  auto range = [&](int d, int& lo, int& hi) {
    lo = 0;
    hi = a.V;
    if (!HELD) return;
    int c = (int)(((int64_t)start + d) % a.C);
    if (c < 0) c += a.C;
    lo = max(a.ranges[2 * c], 0);
    hi = min(a.ranges[2 * c + 1], a.V);
  };
  bool here[2];
  for (int k = 0; k < 2; k++) {
    here[k] = root && up[k] == 0 && lane + 64 * k < N;
    if (here[k] && lane + 64 * k > 0 && id[k] >= 0) {
      int lo, hi;
      range(depth[k] - 1, lo, hi);
      if (id[k] >= lo && id[k] < hi) {
        P[k] = prob(target[par[k] * a.ts[1] + id[k]]);
        if (Q) q[k] = prob(draft[par[k] * a.ds[1] + id[k]]);
      }
    }
  }
  int32_t* path = a.path + (int64_t)b * N;
  int32_t* tokens = a.tokens + (int64_t)b * N;
  if (!root) {
    if (t < N) path[t] = tokens[t] = -1;
    if (t == 0) a.n[b] = 0;
    return;
  }

  Row row;
  row.Z = Z;
  row.x = rejx;
  // the W parts of [lo, hi) and their sums of r, all of it returned; whole steps of a wave each
  int size = 0;
  auto sums = [&](int lo, int hi) {
    size = hi > lo ? ((hi - lo + W - 1) / W + STEP - 1) / STEP * STEP : STEP;
    const int end = (int)min((int64_t)hi, (int64_t)lo + (int64_t)(wave + 1) * size);
    double s = 0;
    for (int64_t i = (int64_t)lo + (int64_t)wave * size + lane * VEC; i < end; i += DEEP * STEP) {
      typename Row::Raw w[DEEP];
#pragma unroll
      for (int k = 0; k < DEEP; k++)
        if (i + k * STEP < end) row.load(w[k], (int)i + k * STEP, end);
#pragma unroll
      for (int k = 0; k < DEEP; k++)
        if (i + k * STEP < end) s += row.sum(w[k], (int)i + k * STEP);
    }
    s = wave_total(s);
    __syncthreads();
    if (lane == 0) part[wave] = s;
    __syncthreads();
    double all = lane < W ? part[lane] : 0.0;
    return wave_total(all);
  };

  // P, and Qs, the mass of the draft's row, as sums in one order: equal rows have equal ones.  Up to 64 entries every wave
  // sums itself.
  auto masses = [&](int lo, int hi, double& Qs) {
    __shared__ double part_q[W];
    double s = 0, sq = 0;
    if (hi - lo <= 64) {
      if (lo + lane < hi) s = prob(row.p[lo + lane]), sq = prob(row.q[lo + lane]);
      Qs = wave_total(sq);
      return wave_total(s);
    }
#pragma unroll 8
    for (int i = lo + t; i < hi; i += 64 * W) s += prob(row.p[i]), sq += prob(row.q[i]);
    s = wave_total(s), sq = wave_total(sq);
    __syncthreads();
    if (lane == 0) part[wave] = s, part_q[wave] = sq;
    __syncthreads();
    Qs = wave_total(lane < W ? part_q[lane] : 0.0);
    return wave_total(lane < W ? part[lane] : 0.0);
  };

  int c = 0, n = 1, seen = 0;
  double z = 1.0, full = 0;
  row.rejected = 0;
  if (t == 0) path[0] = 0;
  for (;;) {
    row.p = target + c * a.ts[1];
    row.q = draft + c * a.ds[1];
    range(n - 1, row.lo, row.hi);
    // Z of the first child differs from context to context with ranges: no wave may still read the last one's
    if (Q && HELD && row.rejected) __syncthreads();
    row.rejected = 0;
    z = 1.0;    // Z (-1: to be taken)
    full = 0;   // without draft rows the last one that was taken,
    seen = 0;   // and the children rejected by then
    uint64_t kids[2] = {__ballot(here[0] && par[0] == c && lane > 0), __ballot(here[1] && par[1] == c)};
    double Qs = 1.0;
    if constexpr (HELD) {
      for (int k = 0; k < 2; k++) kids[k] &= __ballot(id[k] >= row.lo && id[k] < row.hi);
      z = -1.0;
      if (Q && (kids[0] | kids[1])) {
        z = mass_of<T>(masses(row.lo, row.hi, Qs));
        Qs = mass_of<T>(Qs);
        if (!(Qs > 0)) kids[0] = kids[1] = 0;
        z /= Qs;
      }
    }
    int taken = -1;
    uint64_t gone[2] = {0, 0};
    while (kids[0] | kids[1]) {
      const int k = kids[0] ? 0 : 1, l = __builtin_ctzll(kids[k]);
      kids[k] &= kids[k] - 1;
      const int x = __builtin_amdgcn_readlane(k ? id[1] : id[0], l);
      const double qx = lane_value(k ? q[1] : q[0], l), ux = lane_value(k ? u[1] : u[0], l);
      double r = lane_value(k ? P[1] : P[0], l);
      if ((HELD || row.rejected) && z < 0) {
        full = sums(row.lo, row.hi);
        seen = row.rejected;
        z = !HELD ? full : Q ? full / Qs : row.rejected ? full : mass_of<T>(full);
      }
      if (row.rejected) {
        if (Q) {
          for (int j = 0; j < row.rejected; j++) r = fmax(fma(-Z[j], qx, r), 0.0);
        } else {
          if (__ballot((gone[0] >> lane & 1) && id[0] == x) | __ballot((gone[1] >> lane & 1) && id[1] == x)) r = 0;
        }
      }
      if (ux * qx * z < r) {
        taken = l + 64 * k;
        if (t == 0) {
          path[n] = taken;
          tokens[n - 1] = x;
        }
        break;
      }
      // (every wave writes the same.  The first entry of a context may be written while a slower wave still reads the last
      // context's, which is the same 1, or is kept from it above; before the second there is a sum and its barriers)
      if (Q) {
        Z[row.rejected] = z;
        z = -1.0;
      } else {
        // without draft rows the sum falls by r(x): taken anew only when little is left of it
        gone[k] |= 1ull << l;
        rejx[row.rejected] = x;
        rejr[row.rejected] = r;
        if (HELD && !row.rejected) z = full;
        z = full > 0 && z - r > VER_KEEP * full ? z - r : -1.0;
      }
      row.rejected++;
    }
    if (taken < 0) break;
    c = taken;
    n++;
  }
  double S = -1.0;
  if (!Q && full > 0 && row.rejected > seen) {
    // the parts are known from the last sum, but for the entries that went since: taken off, unless a part loses nearly all
    double mine = lane < W ? part[lane] : 0.0;
    const double before = mine;
    for (int j = seen; j < row.rejected; j++)
      if (lane == (rejx[j] - row.lo) / size) mine -= rejr[j];
    if (!__any(mine < before && !(mine > VER_KEEP * before))) {
      __syncthreads();
      if (wave == 0 && lane < W) part[lane] = mine;
      __syncthreads();
      S = wave_total(mine);
    }
  }
  if (S < 0) S = sums(row.lo, row.hi);
  if (!(S > 0)) {
    row.rejected = 0;
    S = sums(row.lo, row.hi);
  }
  // the part that the number falls into, a part of it, and so on down to a few steps of one wave
  int next = -1;
  if (S > 0) {
    double at = (double)lane_value(u[0], 0) * S;
    int lo = row.lo, hi = row.hi;
    for (;;) {
      const double mine = lane < W ? part[lane] : 0.0, in = wave_scan(mine);
      const uint64_t some = __ballot(mine > 0);
      const uint64_t over = __ballot(lane < W && mine > 0 && in > at);
      const int w = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);  // (rounding let none pass: the last)
      at -= lane_value(in - mine, w);
      lo += w * size;
      hi = (int)min((int64_t)hi, (int64_t)lo + size);
      if (hi - lo <= DEEP * STEP) break;
      sums(lo, hi);
    }
    int last = -1;
    typename Row::Raw w[DEEP];
#pragma unroll
    for (int k = 0; k < DEEP; k++)
      if (lo + k * STEP < hi) row.load(w[k], lo + k * STEP + lane * VEC, hi);
#pragma unroll
    for (int j = 0; j < DEEP; j++) {
      if (lo + j * STEP >= hi || next >= 0) break;
      double r[VEC], mine = 0;
      const int e = lo + j * STEP + lane * VEC;
      row.values(w[j], e, r);
#pragma unroll
      for (int k = 0; k < VEC; k++) mine += r[k];
      const double in = wave_scan(mine);
      double base = in - mine;
      int first = INT32_MAX, back = -1;
#pragma unroll
      for (int k = 0; k < VEC; k++) {
        base += r[k];
        if (r[k] > 0) {
          back = e + k;
          if (base > at && first == INT32_MAX) first = e + k;
        }
      }
      const uint64_t hit = __ballot(first != INT32_MAX), some = __ballot(back >= 0);
      if (hit) next = __builtin_amdgcn_readlane(first, __builtin_ctzll(hit));
      if (some) last = __builtin_amdgcn_readlane(back, 63 - __builtin_clzll(some));
      at -= lane_value(in, 63);
    }
    if (next < 0) next = last;
  }
  if (t == 0) {
    tokens[n - 1] = next;
    a.n[b] = n;
  }
  if (t >= n && t < N) path[t] = tokens[t] = -1;
}

}  // namespace gb
