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
  int32_t splits;  // parts of a sequence's keys
  float* part;     // partial sums: [item][split][row][D], then {max, sum} [item][split][row]
};

constexpr int ATT_BLOCK = 256;
constexpr int ATT_WAVES = ATT_BLOCK / 64;
constexpr int ATT_TILE = 32;  // keys a wave works on at a time
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LOWEST = -3.402823466e38f;  // the running maximum's start: exp2(-inf - LOWEST) is 0, not NaN

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// The inputs' type in the matrix unit.  The weights w are rounded to it before the product with v.  In
// fp16 they are held times 2^12 (the factor leaves with the division by their sum): a weight of 2^-37
// of the largest keeps full precision then, so that many far keys are not lost against a near one.
template <typename T>
struct Half;
template <>
struct Half<bf16_t> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr float bias = 0.f;
  static __device__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};
template <>
struct Half<fp16_t> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr float bias = 12.f;
  static __device__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

template <typename T>
__device__ inline uint32_t pack2(float x, float y) {
  typedef T v2 __attribute__((ext_vector_type(2)));
  const v2 v = {(T)x, (T)y};
  return __builtin_bit_cast(uint32_t, v);
}

// over the four lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ inline float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float quad_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// LDS that only this wave uses: its accesses are done in order, the compiler has to leave them so
__device__ inline void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// exponent all ones in any of the eight halves
template <typename T>
__device__ inline bool not_finite(u32x4 v) {
  const uint32_t e = sizeof(T) == 2 && Half<T>::bias == 0.f ? 0x7f80u : 0x7c00u;
  bool any = false;
  for (int i = 0; i < 4; i++) any |= (v[i] & e) == e || ((v[i] >> 16) & e) == e;
  return any;
}

// The tree of one sequence in LDS: anc[i] the set of nodes on the path from the root to i (i included),
// empty when i is absent.
struct Tree {
  int par[DRAFT_MAX_NODES];
  uint32_t anc[DRAFT_MAX_NODES][4];
};
__device__ inline void tree_paths(Tree& tr, int N, const int32_t* parents) {
  const int t = threadIdx.x;
  if (t < N) tr.par[t] = parents[t];
  __syncthreads();
  if (t < N) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (draft_depth(tr.par, t) >= 0)
      for (int i = t; i >= 0; i = tr.par[i])
        for (int k = 0; k < 4; k++)
          if (i / 32 == k) w[k] |= 1u << (i % 32);
    for (int k = 0; k < 4; k++) tr.anc[t][k] = w[k];
  }
  __syncthreads();
}

// keys of a sequence in tiles: the cache's, then the nodes'
struct Span {
  int len, cache_tiles, tiles;
  bool bad;
};
__device__ inline Span span_of(const AttendArgs& a, int b, int tile) {
  Span s;
  const int cap = a.M * a.S;
  s.len = a.lens[b];
  s.bad = s.len < 0 || s.len > cap;
  s.len = min(max(s.len, 0), cap);
  s.cache_tiles = (int)(((uint32_t)s.len + tile - 1) / tile);
  s.tiles = s.cache_tiles + (a.N + tile - 1) / tile;
  return s;
}

// parts that a sequence of `tiles` tiles is really cut into, at least ATT_MIN tiles each
constexpr int ATT_MIN = 16;
#ifndef ATT_WANT
#define ATT_WANT 1024
#endif
__host__ __device__ inline int parts_of(int tiles, int splits) { 
  const int most = (tiles + ATT_MIN - 1) / ATT_MIN;
  return splits < most ? splits : most;
}

// A workgroup: RB blocks of 16 rows (row m: node m / G, head m % G of one kv head), one part of the keys;
// its waves take the part's tiles of 32 keys in turn and join at the end.
//
// S^T = K Q^T and O^T = V^T P^T in the 16x16x32 matrix instruction: a lane then holds its own row's
// weights (row = lane % 16), running maximum and sums, and the weights of four keys in a row are what the second
// product's operand wants, so nothing is moved between lanes but the maximum.  K goes from memory into the operand
// registers, V through the wave's own LDS, where the transposing read turns it; the rows there are 32 bytes longer
// than the head so that eight of them start in different banks.
template <typename T, int KS, int RB>
__global__ __launch_bounds__(ATT_BLOCK) void k_attend(AttendArgs a) {
  constexpr int DP = 32 * KS, DB = 2 * KS, LROW = DP * 2 + 32;
  constexpr int AREA = ATT_TILE * LROW;  // >= 16 rows of DP + 4 floats
  __shared__ __attribute__((aligned(16))) char lds[ATT_WAVES * AREA];
  __shared__ Tree tr;
  __shared__ float ml[2][ATT_WAVES][RB * 16];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l16 = lane & 15, lq = lane >> 4;
  const int G = a.Hq / a.Hkv, M = a.N * G, RT = (M + RB * 16 - 1) / (RB * 16);
  // blocks go to the 8 dies in turn: the row tiles of one part stay on one die, one after the other
  const int die = blockIdx.x & 7, j8 = blockIdx.x >> 3;
  const int rt = j8 % RT, item = (j8 / RT) * 8 + die;
  if (item >= a.B * a.Hkv * a.splits) return;
  const int split = item % a.splits, bh = item / a.splits, h = bh % a.Hkv, b = bh / a.Hkv;
  const Span sp = span_of(a, b, ATT_TILE);
  const int parts = parts_of(sp.tiles, a.splits);
  if (split >= parts) return;
  const int per = (sp.tiles + parts - 1) / parts;
  const int first = split * per, last = min(first + per, sp.tiles);
  const Pages pages = {a.table + b * a.table_stride, a.div, a.P, a.M};
  const T* kc = (const T*)a.kc + h * a.kcs[2];
  const T* vc = (const T*)a.vc + h * a.vcs[2];
  const T* kd = (const T*)a.kd + b * a.kds[0] + h * a.kds[2];
  const T* vd = (const T*)a.vd + b * a.vds[0] + h * a.vds[2];
  bool bad = sp.bad;

  // a tile's addresses: lane's keys are l16 and 16 + l16 of it, keys past the end are the last key again.  The
  // table's entries are looked at only when they are used, a tile later: nothing waits for them before.
  int id[2], slot[2];
  auto find = [&](int tile) {
    for (int c = 0; c < 2; c++) id[c] = page_entry(pages, min(tile * ATT_TILE + 16 * c + l16, sp.len - 1), slot[c]);
  };
  u32x4 kf[2][KS], vf[2][KS];
  auto load = [&](int c, const T* kp, const T* vp) {
    for (int k = 0; k < KS; k++) {
      const int d = 32 * k + 8 * lq;
      const u32x4 zero = {0, 0, 0, 0};
      kf[c][k] = d < a.D ? *(const u32x4*)(kp + d) : zero;
      vf[c][k] = d < a.D ? *(const u32x4*)(vp + d) : zero;
    }
  };
  auto fetch = [&]() {
    for (int c = 0; c < 2; c++) {
      if (!good_page(pages, id[c])) {  // reads page 0, and the sequence's rows become NaN
        bad = true;
        id[c] = 0;
      }
      load(c, kc + id[c] * a.kcs[0] + slot[c] * a.kcs[1], vc + id[c] * a.vcs[0] + slot[c] * a.vcs[1]);
    }
  };
  auto fetch_nodes = [&](int base) {
    for (int c = 0; c < 2; c++) {
      const int n = min(base + 16 * c + l16, a.N - 1);
      load(c, kd + n * a.kds[1], vd + n * a.vds[1]);
    }
  };
  const int cached = min(last, sp.cache_tiles);
  int tile = first + wave;
  if (tile < cached) {
    find(tile);
    fetch();
    if (tile + ATT_WAVES < cached) find(tile + ATT_WAVES);
  }
  u32x4 qf[RB][KS];
  for (int r = 0; r < RB; r++) {
    const int m = (rt * RB + r) * 16 + l16, n = m / G;
    const T* q = (const T*)a.q + b * a.qs[0] + n * a.qs[1] + (h * G + m - n * G) * a.qs[2];
    for (int k = 0; k < KS; k++) {
      const int d = 32 * k + 8 * lq;
      const u32x4 zero = {0, 0, 0, 0};
      qf[r][k] = m < M && d < a.D ? *(const u32x4*)(q + d) : zero;
    }
  }
  tree_paths(tr, a.N, a.parents + b * a.parents_stride);

  const float scale = a.scale * LOG2E;
  float top[RB], sum[RB];
  f32x4 o[DB][RB];
  for (int r = 0; r < RB; r++) {
    top[r] = LOWEST;
    sum[r] = 0.f;
    for (int d = 0; d < DB; d++) o[d][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  char* area = lds + wave * AREA;
  auto step = [&](auto is_nodes, int base) {
    constexpr bool nodes = decltype(is_nodes)::value;
    bool odd = false;  // a node's value that is not finite
    for (int c = 0; c < 2; c++)
      for (int k = 0; k < KS; k++) {
        if constexpr (nodes) {
          // a node reaches its own descendants only, but 0 times infinity or NaN would reach every row:
          // such values go in as 0 and are added below where they belong
          const bool bad_v = not_finite<T>(vf[c][k]);
          odd |= bad_v;
          for (int i = 0; i < 4; i++) vf[c][k][i] = bad_v ? 0u : vf[c][k][i];
        }
        *(u32x4*)(area + (16 * c + l16) * LROW + (32 * k + 8 * lq) * 2) = vf[c][k];
      }
    wave_order();
    f32x4 s[2][RB];
    for (int c = 0; c < 2; c++)
      for (int r = 0; r < RB; r++) {
        s[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < KS; k++) s[c][r] = Half<T>::mfma(kf[c][k], qf[r][k], s[c][r]);
      }
    const int next = tile + ATT_WAVES;
    if (!nodes && next < cached) {
      fetch();
      if (next + ATT_WAVES < cached) find(next + ATT_WAVES);
    }
    u32x4 p[RB];
    for (int r = 0; r < RB; r++) {
      for (int c = 0; c < 2; c++) s[c][r] *= scale;
      if constexpr (nodes) {
        const int m = (rt * RB + r) * 16 + l16;
        const uint32_t set = m < M ? tr.anc[m / G][base / 32] : 0;
        for (int c = 0; c < 2; c++)
          for (int i = 0; i < 4; i++)
            if (!(set >> (16 * c + 4 * lq + i) & 1)) s[c][r][i] = -INFINITY;
      } else if (base + ATT_TILE > sp.len) {
        for (int c = 0; c < 2; c++)
          for (int i = 0; i < 4; i++)
            if (base + 16 * c + 4 * lq + i >= sp.len) s[c][r][i] = -INFINITY;
      }
      float mx = top[r];
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[c][r][i]);
      mx = quad_max(mx);
      if (__any(mx > top[r])) {
        const float f = __builtin_amdgcn_exp2f(top[r] - mx);
        top[r] = mx;
        sum[r] *= f;
        for (int d = 0; d < DB; d++) o[d][r] *= f;
      }
      const float off = Half<T>::bias - mx;
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 4; i++) s[c][r][i] = __builtin_amdgcn_exp2f(s[c][r][i] + off);
      sum[r] += ((s[0][r][0] + s[0][r][1]) + (s[0][r][2] + s[0][r][3])) +
                ((s[1][r][0] + s[1][r][1]) + (s[1][r][2] + s[1][r][3]));
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 2; i++) p[r][2 * c + i] = pack2<T>(s[c][r][2 * i], s[c][r][2 * i + 1]);
    }
    for (int d = 0; d < DB; d++) {
      u32x4 v;
      for (int c = 0; c < 2; c++) {
        const char* at = area + (16 * c + 4 * lq + (l16 >> 2)) * LROW + (16 * d + 4 * (l16 & 3)) * 2;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 y = __builtin_bit_cast(u32x2, x);
        v[2 * c] = y[0];
        v[2 * c + 1] = y[1];
      }
      for (int r = 0; r < RB; r++) o[d][r] = Half<T>::mfma(v, p[r], o[d][r]);
    }
    wave_order();
    if (!nodes || !__any(odd)) return;
    if constexpr (nodes) {
      // what went in as 0 were pieces of eight values: their finite values come back with their weights
      float* mine = (float*)area + l16 * (DP + 4) + 4 * lq;
#pragma unroll
      for (int r = 0; r < RB; r++) {
        const int m = (rt * RB + r) * 16 + l16;
#pragma unroll 1
        for (int d = 0; d < DB; d++) *(f32x4*)(mine + 16 * d) = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int j = 0; j < ATT_TILE && base + j < a.N; j++) {
          if (m >= M || !(tr.anc[m / G][base / 32] >> j & 1)) continue;
          const T* v = vd + (base + j) * a.vds[1];
          const T* k = kd + (base + j) * a.kds[1];
          const T* q = (const T*)a.q + b * a.qs[0] + (m / G) * a.qs[1] + (h * G + m % G) * a.qs[2];
          float dot = 0.f;
#pragma unroll 1
          for (int e = 0; e < a.D; e++) dot = fmaf((float)q[e], (float)k[e], dot);
          const float w = __builtin_amdgcn_exp2f(dot * scale + Half<T>::bias - top[r]);
#pragma unroll 1
          for (int d = 4 * lq; d < a.D; d += 16) {
            if (!not_finite<T>(*(const u32x4*)(v + d / 8 * 8))) continue;
            for (int i = 0; i < 4; i++) {
              const float y = (float)v[d + i];
              mine[d - 4 * lq + i] += isfinite(y) ? w * y : y;
            }
          }
        }
#pragma unroll
        for (int d = 0; d < DB; d++) o[d][r] += *(const f32x4*)(mine + 16 * d);
      }
      wave_order();
    }
  };
  for (; tile < cached; tile += ATT_WAVES) step(std::false_type(), tile * ATT_TILE);
  for (; tile < last; tile += ATT_WAVES) {
    const int base = (tile - sp.cache_tiles) * ATT_TILE;
    fetch_nodes(base);
    step(std::true_type(), base);
  }

  // the waves' sums joined: maxima first, then 16 rows at a time through LDS
  for (int r = 0; r < RB; r++) {
    sum[r] = quad_sum(sum[r]);
    if (__any(bad)) sum[r] = NAN;
    if (lq == 0) {
      ml[0][wave][r * 16 + l16] = top[r];
      ml[1][wave][r * 16 + l16] = sum[r];
    }
  }
  const int bhr = bh * RT + rt;
  for (int r = 0; r < RB; r++) {
    __syncthreads();
    float* mine = (float*)area + l16 * (DP + 4) + 4 * lq;
    for (int d = 0; d < DB; d++) *(f32x4*)(mine + 16 * d) = o[d][r];
    __syncthreads();
    for (int e = t; e < 16 * DP / 4; e += ATT_BLOCK) {
      const int row = e / (DP / 4), d = e % (DP / 4) * 4, m = (rt * RB + r) * 16 + row;
      if (m >= M || d >= a.D) continue;
      float mx = LOWEST;
      for (int w = 0; w < ATT_WAVES; w++) mx = fmaxf(mx, ml[0][w][r * 16 + row]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float total = 0.f;
      for (int w = 0; w < ATT_WAVES; w++) {
        const float f = __builtin_amdgcn_exp2f(ml[0][w][r * 16 + row] - mx);
        total += f * ml[1][w][r * 16 + row];
        acc += f * *(const f32x4*)((const float*)(lds + w * AREA) + row * (DP + 4) + d);
      }
      if (parts == 1) {
        const int n = m / G;
        T* out = (T*)a.out + (((int64_t)b * a.N + n) * a.Hq + h * G + m - n * G) * a.D + d;
        const bool here = tr.anc[n][n / 32] >> (n % 32) & 1;
        const float f = 1.f / total;
        uint32_t w[2] = {pack2<T>(acc[0] * f, acc[1] * f), pack2<T>(acc[2] * f, acc[3] * f)};
        *(uint64_t*)out = here ? (uint64_t)w[1] << 32 | w[0] : 0;
      } else {
        const int64_t at = ((int64_t)bhr * a.splits + split) * (RB * 16) + r * 16 + row;
        *(f32x4*)(a.part + at * a.D + d) = acc;
        if (d == 0) {
          float* p = a.part + (int64_t)a.B * a.Hkv * RT * a.splits * (RB * 16) * a.D + 2 * at;
          p[0] = mx;
          p[1] = total;
        }
      }
    }
  }
}

// ---- many rows -------------------------------------------------------------------------------
// Above 32 rows a kv head the keys are shared: a workgroup has 128 rows, 32 a wave, and its waves read the same
// tiles of 64 keys from LDS.  The cache's rows go there directly, the next tile's while this one's products run.
// S^T = K Q^T and O^T = V^T P^T in the 32x32x16 instruction, in the same way as above: row = lane % 32, and a
// lane's weights of four keys in a row are the second product's operand.
//
// In LDS a row's 16-byte pieces are permuted so that the operands' reads spread over the banks: K's piece c of
// row r lies at c ^ (r & 7) (eight rows, one piece each), V's at c ^ 4 (r & 3) (four rows, 64 bytes each; rows of
// 128 bytes: c ^ 4 (r / 2 & 1)).
constexpr int WIDE_TILE = 64;
constexpr int WIDE_ROWS = 128;

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c, bf16_t) {
  typedef Half<bf16_t>::v8 v8;
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c, fp16_t) {
  typedef Half<fp16_t>::v8 v8;
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
// over the lanes l, l ^ 32
__device__ inline float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 16 bytes a lane from memory to LDS, the wave's 1024 bytes in a row at `at`.  In assembly because the compiler
// takes every LDS read for one of the bytes in flight and waits for them: here it is the caller who waits (vmcnt)
// and has a barrier before anyone reads.  There is no output register, the address is read at issue, and nothing else
// in these kernels uses m0.
__device__ inline void to_lds(const void* p, uint32_t at) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(p), "s"(__builtin_amdgcn_readfirstlane(at))
               : "memory");
}

__device__ inline void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), as the compiler counts it too
  asm volatile("" ::: "memory");
}

__device__ const u32x4 att_zero = {0, 0, 0, 0};  // what a head's pieces past its end are read from

template <typename T, int DP>
__global__ __launch_bounds__(ATT_BLOCK, DP > 128 ? 1 : 2) void k_attend_wide(AttendArgs a) {
  constexpr int CH = DP / 8, KSTEPS = DP / 16, DB = DP / 32;
  constexpr int TILE_BYTES = WIDE_TILE * DP * 2, PER = WIDE_TILE * CH / ATT_BLOCK;  // pieces a thread moves
  constexpr int RPI = ATT_BLOCK / CH;                                               // rows between them
  __shared__ __attribute__((aligned(16))) char lds[4 * TILE_BYTES];                 // K, V; twice
  __shared__ Tree tr;
  __shared__ int odd_;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l32 = lane & 31, hh = lane >> 5;
  const int G = a.Hq / a.Hkv, M = a.N * G, RT = (M + WIDE_ROWS - 1) / WIDE_ROWS;
  const int die = blockIdx.x & 7, j8 = blockIdx.x >> 3;
  const int rt = j8 % RT, item = (j8 / RT) * 8 + die;
  if (item >= a.B * a.Hkv * a.splits) return;
  const int split = item % a.splits, bh = item / a.splits, h = bh % a.Hkv, b = bh / a.Hkv;
  const Span sp = span_of(a, b, WIDE_TILE);
  const int parts = parts_of(sp.tiles, a.splits);
  if (split >= parts) return;
  const int per = (sp.tiles + parts - 1) / parts;
  const int first = split * per, last = min(first + per, sp.tiles);
  const Pages pages = {a.table + b * a.table_stride, a.div, a.P, a.M};
  const T* kc = (const T*)a.kc + h * a.kcs[2];
  const T* vc = (const T*)a.vc + h * a.vcs[2];
  const T* kd = (const T*)a.kd + b * a.kds[0] + h * a.kds[2];
  const T* vd = (const T*)a.vd + b * a.vds[0] + h * a.vds[2];
  bool bad = sp.bad;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  // thread t moves piece t % CH (as it lies in LDS) of the rows t / CH + RPI i
  const int prow = t / CH, pc = t % CH;
  auto kswz = [](int row) { return row & 7 & (CH - 1); };
  auto vswz = [](int row) { return CH >= 16 ? (row & 3) << 2 : CH == 8 ? (row >> 1 & 1) << 2 : 0; };
  int id[PER], slot[PER];
  auto find = [&](int tile) {
    for (int i = 0; i < PER; i++) id[i] = page_entry(pages, min(tile * WIDE_TILE + prow + RPI * i, sp.len - 1), slot[i]);
  };
  auto stage = [&](int buf) {
    const uint32_t k = lds_at + buf * 2 * TILE_BYTES + wave * 1024;  // the wave's 64 pieces in a row
    for (int i = 0; i < PER; i++) {
      if (!good_page(pages, id[i])) {  // reads page 0, and the sequence's rows become NaN
        bad = true;
        id[i] = 0;
      }
      const int row = prow + RPI * i, ck = (pc ^ kswz(row)) * 8, cv = (pc ^ vswz(row)) * 8;
      const T* kp = kc + id[i] * a.kcs[0] + slot[i] * a.kcs[1] + ck;
      const T* vp = vc + id[i] * a.vcs[0] + slot[i] * a.vcs[1] + cv;
      to_lds(ck < a.D ? (const void*)kp : &att_zero, k + i * ATT_BLOCK * 16);
      to_lds(cv < a.D ? (const void*)vp : &att_zero, k + TILE_BYTES + i * ATT_BLOCK * 16);
    }
  };
  const int cached = min(last, sp.cache_tiles);
  int tile = first;
  if (tile < cached) {
    find(tile);
    wait_loads();
    stage(0);
    if (tile + 1 < cached) find(tile + 1);
  }
  const int m = rt * WIDE_ROWS + wave * 32 + l32, node = m / G;
  const bool rows = rt * WIDE_ROWS + wave * 32 < M;  // (the wave has any)
  u32x4 qf[KSTEPS];
  const T* q = (const T*)a.q + b * a.qs[0] + node * a.qs[1] + (h * G + m - node * G) * a.qs[2];
  for (int k = 0; k < KSTEPS; k++) {
    const int d = 16 * k + 8 * hh;
    qf[k] = m < M && d < a.D ? *(const u32x4*)(q + d) : att_zero;
  }
  if (t == 0) odd_ = 0;
  tree_paths(tr, a.N, a.parents + b * a.parents_stride);

  const float scale = a.scale * LOG2E;
  float top = LOWEST, sum = 0.f;
  f32x16 o[DB];
  for (int d = 0; d < DB; d++)
    for (int i = 0; i < 16; i++) o[d][i] = 0.f;

  auto step = [&](auto is_nodes, int base, int buf) {
    constexpr bool nodes = decltype(is_nodes)::value;
    const char* kt = lds + buf * 2 * TILE_BYTES;
    const char* vt = kt + TILE_BYTES;
    f32x16 s[2];
    for (int c = 0; c < 2; c++) {
      for (int i = 0; i < 16; i++) s[c][i] = 0.f;
      const int row = 32 * c + l32;
      for (int k = 0; k < KSTEPS; k++) {
        const u32x4 kf = *(const u32x4*)(kt + (row * CH + ((2 * k + hh) ^ kswz(row))) * 16);
        s[c] = mfma32(kf, qf[k], s[c], T());
      }
    }
    // key 32 c + 8 (i / 4) + 4 hh + i % 4 of the tile
    for (int c = 0; c < 2; c++) s[c] *= scale;
    if constexpr (nodes) {
      for (int c = 0; c < 2; c++) {
        const uint32_t set = m < M ? tr.anc[node][base / 32 + c] : 0;
        for (int i = 0; i < 16; i++)
          if (!(set >> (8 * (i / 4) + 4 * hh + i % 4) & 1)) s[c][i] = -INFINITY;
      }
    } else if (base + WIDE_TILE > sp.len) {
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 16; i++)
          if (base + 32 * c + 8 * (i / 4) + 4 * hh + i % 4 >= sp.len) s[c][i] = -INFINITY;
    }
    float mx = top;
    for (int c = 0; c < 2; c++)
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[c][i]);
    mx = pair_max(mx);
    if (__any(mx > top)) {
      const float f = __builtin_amdgcn_exp2f(top - mx);
      top = mx;
      sum *= f;
      for (int d = 0; d < DB; d++) o[d] *= f;
    }
    const float off = Half<T>::bias - mx;
    u32x4 p[4];
    float part[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < 2; c++)
      for (int i = 0; i < 16; i += 2) {
        const float x = __builtin_amdgcn_exp2f(s[c][i] + off), y = __builtin_amdgcn_exp2f(s[c][i + 1] + off);
        part[i / 2 % 4] += x + y;
        p[2 * c + i / 8][i / 2 % 4] = pack2<T>(x, y);
      }
    sum += (part[0] + part[1]) + (part[2] + part[3]);
    for (int st = 0; st < 4; st++)  // 16 keys: the lane's are 16 st + 4 hh + {0..3, 8..11}
      for (int d = 0; d < DB; d++) {
        u32x4 v;
        for (int c = 0; c < 2; c++) {
          const int row = 16 * st + 8 * c + 4 * hh + (lane >> 2 & 3), col = 32 * d + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
          const char* at = vt + (row * CH + ((col / 8) ^ vswz(row))) * 16 + (col & 4) * 2;
          const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          const u32x2 y = __builtin_bit_cast(u32x2, x);
          v[2 * c] = y[0];
          v[2 * c + 1] = y[1];
        }
        o[d] = mfma32(v, p[st], o[d], T());
      }
    if constexpr (nodes) {
      if (!odd_) return;
      // the sums of what went in as 0, in the LDS that the tiles do not use now
      float* mine = (float*)(lds + 2 * TILE_BYTES) + ((wave * 32 + l32) * DP / 2);
      for (int half = 0; half < 2; half++) {
        const int d0 = half * (DP / 2);
#pragma unroll 1
        for (int d = 4 * hh; d < DP / 2; d += 8) *(f32x4*)(mine + d) = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int j = 0; j < WIDE_TILE && base + j < a.N; j++) {
          if (m >= M || !(tr.anc[node][(base + j) / 32] >> (j % 32) & 1)) continue;
          const T* v = vd + (base + j) * a.vds[1];
          const T* k = kd + (base + j) * a.kds[1];
          float dot = 0.f;
#pragma unroll 1
          for (int e = 0; e < a.D; e++) dot = fmaf((float)q[e], (float)k[e], dot);
          const float w = __builtin_amdgcn_exp2f(dot * scale + Half<T>::bias - top);
#pragma unroll 1
          for (int d = 4 * hh; d < DP / 2 && d0 + d < a.D; d += 8) {
            if (!not_finite<T>(*(const u32x4*)(v + (d0 + d) / 8 * 8))) continue;
            for (int i = 0; i < 4; i++) {
              const float y = (float)v[d0 + d + i];
              mine[d + i] += isfinite(y) ? w * y : y;
            }
          }
        }
        wave_order();
#pragma unroll
        for (int d = 0; d < DB / 2; d++)
          for (int i = 0; i < 4; i++) {
            const f32x4 x = *(const f32x4*)(mine + 32 * d + 8 * i + 4 * hh);
            for (int e = 0; e < 4; e++) {
              if (half == 0)
                o[d][4 * i + e] += x[e];
              else
                o[DB / 2 + d][4 * i + e] += x[e];
            }
          }
        wave_order();
      }
    }
  };
  for (int buf = 0; tile < cached; tile++, buf ^= 1) {
    wait_loads();     // this wave's pieces of the tile are in LDS
    __syncthreads();  // everyone's are, and the other buffer is free
    if (tile + 1 < cached) {
      stage(buf ^ 1);
      if (tile + 2 < cached) find(tile + 2);
    }
    if (rows) step(std::false_type(), tile * WIDE_TILE, buf);
  }
  for (; tile < last; tile++) {
    // nodes go through registers: a value that is not finite goes in as 0 and is added on its own path
    const int base = (tile - sp.cache_tiles) * WIDE_TILE;
    __syncthreads();
    for (int i = 0; i < PER; i++) {
      const int row = prow + RPI * i, n = min(base + row, a.N - 1);
      const int ck = (pc ^ kswz(row)) * 8, cv = (pc ^ vswz(row)) * 8;
      const u32x4 k = ck < a.D ? *(const u32x4*)(kd + n * a.kds[1] + ck) : att_zero;
      u32x4 v = cv < a.D ? *(const u32x4*)(vd + n * a.vds[1] + cv) : att_zero;
      if (not_finite<T>(v)) {
        v = att_zero;
        odd_ = 1;
      }
      *(u32x4*)(lds + (t + ATT_BLOCK * i) * 16) = k;
      *(u32x4*)(lds + TILE_BYTES + (t + ATT_BLOCK * i) * 16) = v;
    }
    __syncthreads();
    if (rows) step(std::true_type(), base, 0);
  }

  sum += __shfl_xor(sum, 32);
  const bool any_bad = __syncthreads_or(bad);
  if (m >= M) return;
  if (any_bad) sum = NAN;
  const int64_t at = ((int64_t)(bh * RT + rt) * a.splits + split) * WIDE_ROWS + wave * 32 + l32;
  const bool here = tr.anc[node][node / 32] >> (node % 32) & 1;
  const float f = 1.f / sum;
  T* out = (T*)a.out + (((int64_t)b * a.N + node) * a.Hq + h * G + m - node * G) * a.D;
  if (parts > 1 && hh == 0) {
    float* ml = a.part + (int64_t)a.B * a.Hkv * RT * a.splits * WIDE_ROWS * a.D + 2 * at;
    ml[0] = top;
    ml[1] = sum;
  }
  for (int d = 0; d < DB; d++)
    for (int i = 0; i < 4; i++) {
      const int x = 32 * d + 8 * i + 4 * hh;
      if (x >= a.D) continue;
      if (parts > 1) {
        *(f32x4*)(a.part + at * a.D + x) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      } else {
        const uint32_t w[2] = {pack2<T>(o[d][4 * i] * f, o[d][4 * i + 1] * f), pack2<T>(o[d][4 * i + 2] * f, o[d][4 * i + 3] * f)};
        *(uint64_t*)(out + x) = here ? (uint64_t)w[1] << 32 | w[0] : 0;
      }
    }
}

// joins the parts of a sequence: one wave a row
template <typename T>
__global__ __launch_bounds__(ATT_BLOCK) void k_attend_join(AttendArgs a, int rows, int tile) {
  const int G = a.Hq / a.Hkv, M = a.N * G, RT = (M + rows - 1) / rows;
  const int64_t x = (int64_t)blockIdx.x * ATT_WAVES + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (x >= (int64_t)a.B * a.Hkv * M) return;
  const int m = (int)(x % M), bh = (int)(x / M), h = bh % a.Hkv, b = bh / a.Hkv, n = m / G;
  const int parts = parts_of(span_of(a, b, tile).tiles, a.splits);
  if (parts == 1) return;  // (written already)
  // present: the walk to the root
  const int32_t* par = a.parents + b * a.parents_stride;
  const bool here = draft_depth(par, n) >= 0;
  const int64_t at = ((int64_t)bh * RT + m / rows) * a.splits * rows + m % rows;
  const float* ml = a.part + (int64_t)a.B * a.Hkv * RT * a.splits * rows * a.D;
  float mx = LOWEST;
  for (int s = 0; s < parts; s++) mx = fmaxf(mx, ml[2 * (at + (int64_t)s * rows)]);
  T* out = (T*)a.out + (((int64_t)b * a.N + n) * a.Hq + h * G + m - n * G) * a.D;
  for (int d = lane * 4; d < a.D; d += 256) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    for (int s = 0; s < parts; s++) {
      const int64_t r = at + (int64_t)s * rows;
      const float f = __builtin_amdgcn_exp2f(ml[2 * r] - mx);
      total += f * ml[2 * r + 1];
      acc += f * *(const f32x4*)(a.part + r * a.D + d);
    }
    const float f = 1.f / total;
    uint32_t w[2] = {pack2<T>(acc[0] * f, acc[1] * f), pack2<T>(acc[2] * f, acc[3] * f)};
    *(uint64_t*)(out + d) = here ? (uint64_t)w[1] << 32 | w[0] : 0;
  }
}

}  // namespace gb
