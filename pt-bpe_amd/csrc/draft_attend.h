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
  int64_t qs[3], kds[3], vds[3];  // strides: (seq, node, head)
  int64_t khead, vhead;           // the cache's: a head, and in pieces of 16 bytes a page and a slot
  uint32_t kpage, kslot, vpage, vslot;
  int64_t table_stride, parents_stride;
  int32_t B, N, Hq, Hkv, D, S, P, M;  // S: page size, P: pages, M: table entries a sequence
  PageDiv div;                          // S
  float scale;
  int32_t per, most, row_tiles;         // tiles a part of a sequence's keys has at most, parts there are room for
  PageDiv by_G, by_Hkv, by_most, by_per, by_RT;
  float* part;        // [row tile][item][part][row][D], then {max, sum} [row tile][item][part][row]
};

constexpr int ATT_BLOCK = 256;
constexpr int ATT_TILE = 32;  // keys a wave works on at a time
// The keys are cut so that about two workgroups of four waves a CU have work: at 512 / 1024 / 2048 workgroups, the join
// included, one tree over up to 105k positions (2 heads of 48 rows) takes 22 / 28 / 28 us, 7 trees of 27 nodes over up to 4099
// 30 / 27 / 27, 2 tokens over 30k to 60k (8 heads) 115 / 97 / 99: none is best for all.  A part may have 16 tiles before there is
// a second one (with 8 one token over 237 positions takes 8.7 us instead of 6.9, 3 chains of 5 nodes over up to 2000 10.7
// instead of 11.8); as a sequence's parts are equal, they can have about half of that.
constexpr int ATT_WANT = 512, ATT_LEAST = 16;
// a part's sum of an absent row: a present one's is 0 when all of its scores are -infinity, and its result is 0 / 0 then
constexpr float PART_ABSENT = -1.f;
constexpr float LOG2E = 1.44269504088896340736f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// The inputs' type in the matrix unit.  The weights w are rounded to it before the product with v.  In
// fp16 they are held times 2^7 (the factor leaves with the division by their sum, and 2^SLACK times as much is
// still in range): a weight of 2^-21 of the largest keeps full precision then, and those that are lost add up to
// less than 2^-15 over 2^16 keys.
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
  static constexpr float bias = 7.f;
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

template <typename T>
__device__ inline uint64_t pack4(f32x4 v) {
  return (uint64_t)pack2<T>(v[2], v[3]) << 32 | pack2<T>(v[0], v[1]);
}

// Scores are compared as q k and scaled inside the exponent's multiply-add, exp2((q k - max) c + bias), c = |scale| log2 e.
// (One subtraction more than q k c - max c, and not slower: where max c is rounded, past 2^30, the largest weight would
// be anything but 1, and infinite at last.)  A negative scale turns the queries' signs.  A scale of 0 leaves float32's
// smallest c, which takes no score to more than 2^-21 (with 1e-30 products of 1e30 and more were scores still): -inf, what
// is not there, stays -inf.
__device__ inline float score_scale(float scale) { return fmaxf(fabsf(scale) * LOG2E, 0x1p-149f); }
__device__ inline u32x4 negative(u32x4 q) { return q ^ u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u}; }
// a row that has seen no key has the maximum -inf: its weights are taken from 0, and are 0
__device__ inline float at_least(float mx) { return mx == -INFINITY ? 0.f : mx; }

// bytes from the cache's start to a slot
__device__ inline uint64_t cache_row(int id, int slot, uint32_t page, uint32_t one) {
  return ((uint64_t)(uint32_t)id * page + (uint64_t)(uint32_t)slot * one) << 4;
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

__device__ inline u32x4 keep_if(bool in, u32x4 y) {
  for (int i = 0; i < 4; i++) y[i] = in ? y[i] : 0u;
  return y;
}

// s where the set's bit is 1, else -infinity
__device__ inline float if_bit(uint32_t set, int bit, float s) {
  const uint32_t in = (int32_t)(set << (31 - bit)) >> 31;
  return __uint_as_float((__float_as_uint(s) & in) | (0xff800000u & ~in));
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
// empty when i is absent.  The first wave works it out.
struct Tree {
  int up[DRAFT_MAX_NODES];
  __attribute__((aligned(16))) uint32_t anc[DRAFT_MAX_NODES][4];
};
// in two halves, so that what the caller loads meanwhile is not waited for in between
struct Parents {
  int of[2];
};
__device__ inline Parents tree_parents(int N, const int32_t* parents) {
  const int t = threadIdx.x;
  return {{t < 64 && t < N ? parents[t] : -2, t < 64 && t + 64 < N ? parents[t + 64] : -2}};
}
__device__ inline void tree_paths(Tree& tr, int N, Parents parents) {
  const int t = threadIdx.x;
  if (t < 64) {
    const int nodes = N > 64 ? 2 : 1;
    DraftNode n[2];
    auto put = [&](int i, const DraftNode& x) {
      tr.up[i] = x.up;
      *(u32x4*)tr.anc[i] = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
    };
    for (int k = 0; k < 2; k++) n[k] = draft_node(t + 64 * k, parents.of[k]);
    for (;;) {
      for (int k = 0; k < 2; k++)
        if (k < nodes) put(t + 64 * k, n[k]);
      wave_order();
      if (!__any(n[0].up >= 0 || n[1].up >= 0)) break;
      DraftNode above[2];
      for (int k = 0; k < 2; k++)
        if (k < nodes && n[k].up >= 0) {
          above[k].up = tr.up[n[k].up];
          const u32x4 w = *(const u32x4*)tr.anc[n[k].up];
          for (int i = 0; i < 4; i++) above[k].w[i] = w[i];
        }
      wave_order();
      for (int k = 0; k < 2; k++)
        if (k < nodes && n[k].up >= 0) draft_climb(n[k], above[k]);
    }
    for (int k = 0; k < 2; k++)
      if (k < nodes && n[k].up != -1) *(u32x4*)tr.anc[t + 64 * k] = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
}

// a sequence's keys in tiles: the cache's, then the nodes'
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

// values that are the same for the whole workgroup, as such
__device__ inline int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A sequence's tiles are cut into equal parts of at most `per`; a second kernel joins them.
struct Share {
  int parts, first, last;
};
__device__ inline Share share_of(const AttendArgs& a, int tiles, int part) {
  Share s;
  int parts, left, size = tiles;
  page_split(a.by_per, tiles + a.per - 1, parts, left);
  s.parts = 1;
  if (parts > 1) {
    size = (tiles + parts - 1) / parts;
    s.parts = (tiles + size - 1) / size;
  }
  s.first = part * size;
  s.last = min(s.first + size, tiles);
  return s;
}
// a row's place among the parts
__device__ inline int64_t part_row(const AttendArgs& a, int rt, int item, int part, int rows, int row) {
  return (((int64_t)rt * a.B * a.Hkv + item) * a.most + part) * rows + row;
}
__device__ inline float* part_sums(const AttendArgs& a, int RT, int rows) {
  return a.part + (int64_t)RT * a.B * a.Hkv * a.most * rows * a.D;
}

// A workgroup: RB blocks of 16 rows (row m: node m / G, head m % G of one kv head), one part of the keys; its
// waves take the part's tiles of 32 keys in turn and join at the end.
//
// S^T = K Q^T and O^T = V^T P^T in the 16x16x32 matrix instruction: a lane then holds its own row's
// weights (row = lane % 16), running maximum and sums, and the weights of four keys in a row are what the second
// product's operand wants, so nothing is moved between lanes but the maximum.  K and then V go through the wave's own
// LDS: K to be read in the operand's order, V for the transposing read; the rows there are 32 bytes longer than the head
// so that eight of them start in different banks.
//
// What bounds it is memory, or in small calls the way from one load to the next (lengths, table, keys, the join of the
// waves: 6 us without a prefix).  64 chains of 5 nodes, 16 / 4 heads of 64, over 157 to 2237 positions: 24 us, 80 MB at
// 3.3 TB/s, the longest chain's nine turns of its waves after another; one round of workgroups, so nothing evens that out
// (cut finer 28 to 37 with the join).
template <typename T, int KS, int RB, int W>
__global__ __launch_bounds__(64 * W, KS <= 4 ? 2 : 1) void k_attend(AttendArgs a) {
  constexpr int DP = 32 * KS, DB = 2 * KS, LROW = DP * 2 + 32;
  constexpr int DMIN = KS <= 4 ? DP - 24 : DP - 56;  // the heads this is for: DMIN .. DP
  constexpr int AREA = ATT_TILE * LROW;  // >= 16 rows of DP + 4 floats
  __shared__ __attribute__((aligned(16))) char lds[W * AREA];
  __shared__ Tree tr;
  __shared__ float ml[2][W][RB * 16];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l16 = lane & 15, lq = lane >> 4;
  const int G = a.by_G.d, M = a.N * G;
  // blocks go to the 8 dies in turn: the row tiles of one part stay on one die, one after the other
  const int die = blockIdx.x & 7, j8 = blockIdx.x >> 3;
  int rt, work, part, item, h, b;
  page_split(a.by_RT, j8, work, rt);
  work = work * 8 + die;
  if (work >= a.B * a.Hkv * a.most) return;
  page_split(a.by_most, work, item, part);
  page_split(a.by_Hkv, item, b, h);
  const Span sp = span_of(a, b, ATT_TILE);
  const Share sh = share_of(a, sp.tiles, part);
  if (part >= sh.parts) return;
  const int first = sh.first, last = sh.last;
  char* area = lds + wave * AREA;
  const float scale = score_scale(a.scale);
  const Pages pages = {a.table + b * a.table_stride, a.div, a.P, a.M};
  const char* kc = (const char*)((const T*)a.kc + h * a.khead);
  const char* vc = (const char*)((const T*)a.vc + h * a.vhead);
  const T* kd = (const T*)a.kd + b * a.kds[0] + h * a.kds[2];
  const T* vd = (const T*)a.vd + b * a.vds[0] + h * a.vds[2];
  bool bad = sp.bad;

  // what does not hang on the length is loaded first
  const Parents parents = tree_parents(a.N, a.parents + b * a.parents_stride);
  u32x4 qf[RB][KS];
  int node[RB];  // of the lane's rows (0 past the last row)
  for (int r = 0; r < RB; r++) {
    const int m = (rt * RB + r) * 16 + l16;
    int g;
    page_split(a.by_G, m < M ? m : 0, node[r], g);
    const T* q = (const T*)a.q + b * a.qs[0] + node[r] * a.qs[1] + (h * G + g) * a.qs[2];
    for (int k = 0; k < KS; k++) {
      const int d = 32 * k + 8 * lq;
      const u32x4 zero = {0, 0, 0, 0};
      if (m < M && d < a.D)
        qf[r][k] = *(const u32x4*)(q + d);
      else
        qf[r][k] = zero;
    }
  }
  // A tile as the lane loads it: keys l4 and 16 + l4 (past the end the last key again), pieces 4 k + p4 of them, so that
  // four lanes in a row read 64 bytes in a row (in the operands' own order, a key a lane, the L1 took three times as
  // many accesses and the kernel 1.4 times as long).  The table's entries are looked at only when they are used, a turn
  // later: nothing waits for them before.
  const int l4 = lane >> 2, p4 = lane & 3;
  struct Tile {
    u32x4 k[2][KS], v[2][KS];
    int id[2], slot[2];
  } x;
  auto find = [&](int tile) {
    for (int c = 0; c < 2; c++)
      x.id[c] = page_entry(pages, min(tile * ATT_TILE + 16 * c + l4, sp.len - 1), x.slot[c]);
  };
  auto load = [&](int c, const T* kp, const T* vp) {
    for (int k = 0; k < KS; k++) {
      const int d = 32 * k + 8 * p4;
      if (32 * k + 32 <= DMIN) {
        x.k[c][k] = *(const u32x4*)(kp + d);
        x.v[c][k] = *(const u32x4*)(vp + d);
      } else {  // (past the head: K is 0 there, as the query is; V's channels there go nowhere)
        const bool in = d < a.D;
        x.k[c][k] = keep_if(in, *(const u32x4*)(kp + (in ? d : 0)));
        x.v[c][k] = *(const u32x4*)(vp + (in ? d : 0));
      }
    }
  };
  auto fetch = [&]() {
    for (int c = 0; c < 2; c++) {
      if (!good_page(pages, x.id[c])) {  // reads page 0, and the sequence's rows become NaN
        bad = true;
        x.id[c] = 0;
      }
      load(c, (const T*)(kc + cache_row(x.id[c], x.slot[c], a.kpage, a.kslot)),
           (const T*)(vc + cache_row(x.id[c], x.slot[c], a.vpage, a.vslot)));
    }
  };
  auto fetch_nodes = [&](int tile) {
    for (int c = 0; c < 2; c++) {
      const int n = min((tile - sp.cache_tiles) * ATT_TILE + 16 * c + l4, a.N - 1);
      load(c, kd + n * a.kds[1], vd + n * a.vds[1]);
    }
  };
  // one tile of a wave is on its way while another is worked on (with two on their way nothing got faster: 25.5 us
  // against 24.7, and 40 against 27 where the registers then hold one workgroup a CU)
  const int cached = min(last, sp.cache_tiles);
  int tile = first + wave;
  if (tile < cached) {
    find(tile);
    fetch();
    find(tile + W);
  }
  tree_paths(tr, a.N, parents);
  if (a.scale < 0.f)  // (here, where the queries have to be there: nothing above waits for them)
    for (int r = 0; r < RB; r++)
      for (int k = 0; k < KS; k++) qf[r][k] = negative(qf[r][k]);

  float top[RB], sum[RB];
  f32x4 o[DB][RB];
  for (int r = 0; r < RB; r++) {
    top[r] = -INFINITY;
    sum[r] = 0.f;
    for (int d = 0; d < DB; d++) o[d][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto step = [&](auto is_nodes, int base) {
    constexpr bool nodes = decltype(is_nodes)::value;
    // K into the operands' order through the wave's LDS, then V there for the transposing read
    char* mine = area + l4 * LROW + p4 * 16;
    for (int c = 0; c < 2; c++)
      for (int k = 0; k < KS; k++) *(u32x4*)(mine + c * 16 * LROW + k * 64) = x.k[c][k];
    wave_order();
    u32x4 kf[2][KS];
    for (int c = 0; c < 2; c++)
      for (int k = 0; k < KS; k++) kf[c][k] = *(const u32x4*)(area + (16 * c + l16) * LROW + k * 64 + lq * 16);
    wave_order();
    if constexpr (!nodes) {
      if (base + ATT_TILE > sp.len)  // (behind the last position it is loaded again: its value there has to be 0)
        for (int c = 0; c < 2; c++)
          for (int k = 0; k < KS; k++) x.v[c][k] = keep_if(base + 16 * c + l4 < sp.len, x.v[c][k]);
    }
    bool odd = false;  // a node's value that is not finite
    for (int c = 0; c < 2; c++)
      for (int k = 0; k < KS; k++) {
        if constexpr (nodes) {
          // a node reaches its own descendants only, but 0 times infinity or NaN would reach every row:
          // such values go in as 0 and are added below where they belong
          const bool bad_v = not_finite<T>(x.v[c][k]);
          odd |= bad_v;
          x.v[c][k] = keep_if(!bad_v, x.v[c][k]);
        }
        *(u32x4*)(mine + c * 16 * LROW + k * 64) = x.v[c][k];
      }
    wave_order();
    f32x4 s[2][RB];
    for (int c = 0; c < 2; c++)
      for (int r = 0; r < RB; r++) {
        s[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < KS; k++) s[c][r] = Half<T>::mfma(kf[c][k], qf[r][k], s[c][r]);
      }
    if (!nodes && tile + W < cached) {
      fetch();
      find(tile + 2 * W);
    } else if (!nodes && tile + W < last) {
      fetch_nodes(tile + W);
    }
    u32x4 p[RB];
    for (int r = 0; r < RB; r++) {
      if constexpr (nodes) {
        const int m = (rt * RB + r) * 16 + l16;
        const uint32_t set = m < M ? tr.anc[node[r]][base / 32] >> (4 * lq) : 0;
        for (int c = 0; c < 2; c++)
          for (int i = 0; i < 4; i++) s[c][r][i] = if_bit(set, 16 * c + i, s[c][r][i]);
      } else if (base + ATT_TILE > sp.len) {
        for (int c = 0; c < 2; c++)
          for (int i = 0; i < 4; i++)
            if (base + 16 * c + 4 * lq + i >= sp.len) s[c][r][i] = -INFINITY;
      }
      float mx = top[r];
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[c][r][i]);
      mx = quad_max(mx);
      const float from = at_least(mx);
      if (__any(mx > top[r])) {
        const float f = __builtin_amdgcn_exp2f((top[r] - from) * scale);
        top[r] = mx;
        sum[r] *= f;
        for (int d = 0; d < DB; d++) o[d][r] *= f;
      }
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 4; i++) s[c][r][i] = __builtin_amdgcn_exp2f(fmaf(s[c][r][i] - from, scale, Half<T>::bias));
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
          if (m >= M || !(tr.anc[node[r]][base / 32] >> j & 1)) continue;
          const T* v = vd + (base + j) * a.vds[1];
          const T* k = kd + (base + j) * a.kds[1];
          const T* q = (const T*)a.q + b * a.qs[0] + node[r] * a.qs[1] + (h * G + m - node[r] * G) * a.qs[2];
          float dot = 0.f;
#pragma unroll 1
          for (int e = 0; e < a.D; e++) dot = fmaf((float)q[e], (float)k[e], dot);
          const float w = __builtin_amdgcn_exp2f(fmaf((a.scale < 0.f ? -dot : dot) - at_least(top[r]), scale, Half<T>::bias));
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
  for (; tile < cached; tile += W) step(std::false_type(), tile * ATT_TILE);
  if (tile < last) {  // the nodes (at most 32, as there are no more rows): one tile, of one wave
    if (tile < first + W) fetch_nodes(tile);  // (else loaded in its last step)
    step(std::true_type(), (tile - sp.cache_tiles) * ATT_TILE);
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
  for (int r = 0; r < RB; r++) {
    __syncthreads();
    float* mine = (float*)area + l16 * (DP + 4) + 4 * lq;
    for (int d = 0; d < DB; d++) *(f32x4*)(mine + 16 * d) = o[d][r];
    __syncthreads();
    for (int e = t; e < 16 * DP / 4; e += 64 * W) {
      const int row = e / (DP / 4), d = e % (DP / 4) * 4, m = (rt * RB + r) * 16 + row;
      if (m >= M || d >= a.D) continue;
      float mx = -INFINITY;
      for (int w = 0; w < W; w++) mx = fmaxf(mx, ml[0][w][r * 16 + row]);
      const float from = at_least(mx);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float total = 0.f;
      for (int w = 0; w < W; w++) {
        const float f = __builtin_amdgcn_exp2f((ml[0][w][r * 16 + row] - from) * scale);
        total += f * ml[1][w][r * 16 + row];
        acc += f * *(const f32x4*)((const float*)(lds + w * AREA) + row * (DP + 4) + d);
      }
      int n, g;
      page_split(a.by_G, m, n, g);
      const bool here = tr.anc[n][n / 32] >> (n % 32) & 1;
      if (sh.parts == 1) {
        T* out = (T*)a.out + (((int64_t)b * a.N + n) * a.Hq + h * G + g) * a.D + d;
        *(uint64_t*)out = here ? pack4<T>(acc * (1.f / total)) : 0;
      } else {
        const int64_t at = part_row(a, rt, item, part, RB * 16, r * 16 + row);
        const f32x4 none = {0.f, 0.f, 0.f, 0.f};
        *(f32x4*)(a.part + at * a.D + d) = here ? acc : none;
        if (d == 0) {
          float* p = part_sums(a, a.row_tiles, RB * 16) + 2 * at;
          p[0] = here ? mx : -INFINITY;
          p[1] = here ? total : PART_ABSENT;
        }
      }
    }
  }
}

// ---- many rows -------------------------------------------------------------------------------
// Above 32 rows a kv head the keys are shared: a workgroup has 64 to 256 rows, 32 a wave, and its waves read the same
// tiles of 64 keys from LDS.  Rows go there directly, the next tile's while this one's products run.
// S^T = K Q^T and O^T = V^T P^T in the 32x32x16 instruction, in the same way as above: row = lane % 32, and a
// lane's weights of four keys in a row are the second product's operand.
//
// Up to about 100 rows the cache's bytes bound it: 64 rows of heads of 128 over 131071 positions take 111 us and the
// join 7, 537 MB at 4.8 TB/s.  Above it is the matrix units: 256 rows, 32 sequences over 8k to 16k: 500 to 550 us, 414
// GFLOP at 750 to 830 TFLOP/s.  There is one workgroup a CU, so the longest sequence, 1.3 times the mean, sets the time, and over
// all of it the matrix units are busy for 44 % (58 % while a CU has work): the rest is what does not overlap of the
// exponentials, waits and bank conflicts, and the clock, which the card lowers (the first launches take 480; no order of
// the instructions, depth of the loads or priority of the waves made the later ones faster).  Small calls are the way from one
// load to the next again: 432 rows without a prefix 9.6 us.
//
// In LDS a row's 16-byte pieces are permuted so that the operands' reads spread over the banks: eight rows' piece of K in
// different ones (piece c of row r lies at c ^ (r & 7), in rows of 64 bytes at c ^ (r / 4 & 1), in those of 192, whose
// starts are in four places already, at (c + (r / 4 & 1)) % 12), four rows' 64 bytes of V too (c ^ 4 (r & 3); rows of 128
// bytes: c ^ 4 (r / 2 & 1); rows of 64 and 192 as they are).
template <int CH>
__device__ inline int key_slot(int row, int c) {  // where piece c of a row of CH lies
  if constexpr (CH == 12) {
    const int x = c + (row >> 2 & 1);
    return x < 12 ? x : x - 12;
  }
  return c ^ (CH == 4 ? row >> 2 & 1 : row & 7);
}
template <int CH>
__device__ inline int key_piece(int row, int at) {  // the piece that lies there
  if constexpr (CH == 12) {
    const int x = at - (row >> 2 & 1);
    return x < 0 ? x + 12 : x;
  }
  return key_slot<CH>(row, at);
}
template <int CH>
__device__ inline int value_slot(int row, int c) {  // (its own inverse)
  return c ^ (CH >= 16 ? (row & 3) << 2 : CH == 8 ? (row >> 1 & 1) << 2 : 0);
}
// A part may have 4 tiles before there is a second one (2 heads of 432 rows over 960 positions, with 8 / 4 / 2: 23.4 / 18.4 /
// 16.6 us; with 2 those over 64 take 15.9 instead of 11.6 for the join), and equal parts about half of that.  `Many` tiles:
// eight for every CU.
constexpr int WIDE_TILE = DRAFT_TILE, WIDE_LEAST = 4, WIDE_MANY = 2048;
constexpr float SLACK = 8.f;

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

// LDS by its byte address; `plus` goes into the instruction
template <typename V>
__device__ inline V lds_read(uint32_t at, int plus) {
  return *(const __attribute__((address_space(3))) V*)(uintptr_t)(at + plus);
}
__device__ inline u32x2 lds_read_tr(uint32_t at, int plus) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)(uintptr_t)(at + plus)));
}
__device__ inline void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), as the compiler counts it too
  asm volatile("" ::: "memory");
}

// what a head's pieces past its end and the values behind the last position are read from
__device__ const u32x4 att_zero[32] = {};

template <typename T, int DP, bool FULL, int W>
__global__ __launch_bounds__(64 * W, DP > 128 ? 1 : DP > 32 ? 2 : 3) void k_attend_wide(AttendArgs a) {
  constexpr int BLOCK = 64 * W, ROWS = 32 * W;
  constexpr int CH = DP / 8, KSTEPS = DP / 16, DB = DP / 32;
  constexpr int TILE_BYTES = WIDE_TILE * DP * 2, PER = WIDE_TILE * CH / BLOCK;  // pieces a thread moves
  static_assert(WIDE_TILE * CH % BLOCK == 0, "");
  constexpr uint32_t VBUF = 2 * TILE_BYTES;
  constexpr int TURN = W < 4 ? W : 4;  // waves that take turns at working out places
  __shared__ __attribute__((aligned(16))) char lds[4 * TILE_BYTES];  // K of two tiles, V of two
  __shared__ uint64_t offs[4][2][WIDE_TILE];                         // the rows' places in the cache: tile % 4, K or V
  __shared__ Tree tr;
  __shared__ TileFlags odd_;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l32 = lane & 31, hh = lane >> 5;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const float scale = score_scale(a.scale);
  const int G = a.by_G.d, M = a.N * G;
  const int die = blockIdx.x & 7, j8 = blockIdx.x >> 3;
  int rt, work, part, item, h, b;
  page_split(a.by_RT, j8, work, rt);
  work = work * 8 + die;
  if (work >= a.B * a.Hkv * a.most) return;
  page_split(a.by_most, work, item, part);
  page_split(a.by_Hkv, item, b, h);
  const Span sp = span_of(a, b, WIDE_TILE);
  const Share sh = share_of(a, sp.tiles, part);
  if (part >= sh.parts) return;
  const int m = rt * ROWS + wave * 32 + l32;
  int node, head;  // (of row 0 past the last row)
  page_split(a.by_G, m < M ? m : 0, node, head);
  const bool rows = rt * ROWS + uni(wave) * 32 < M;  // (the wave has any)

  // where this lane's operands lie in a tile: K's piece 2 k + hh of row l32, V's four keys of 16 channels
  uint32_t koff[KSTEPS], voff[DB];
  for (int k = 0; k < KSTEPS; k++) koff[k] = lds_at + (l32 * CH + key_slot<CH>(l32, 2 * k + hh)) * 16;
  for (int d = 0; d < DB; d++) {
    const int row = 4 * hh + (lane >> 2 & 3), col = 32 * d + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
    voff[d] = lds_at + VBUF + (row * CH + value_slot<CH>(row, col / 8)) * 16 + (col & 4) * 2;
  }
  // A wave's 32 rows of the queries and of the result lie in the tiles' place, as K's rows do, before and after them; the
  // lanes move pieces that lie in a row (in the operands' own order, 32 bytes of a row at a time, the queries took 2 us
  // longer and the result 2.5).
  const uint32_t own = wave * 32 * CH * 16;
  auto walk = [&](const T* p, int64_t by_node, int64_t by_head, auto&& piece) {
    const int x = rt * ROWS + wave * 32;
    int n, g;
    if constexpr (CH == 12) {
      for (int i = 0; i < CH / 2; i++) {
        const int row = (lane + 64 * i) / CH;
        page_split(a.by_G, x + row, n, g);
        piece(i, row, lane + 64 * i - row * CH, p + (n * by_node + (h * G + g) * by_head), x + row < M);
      }
    } else {  // a row's place from the last one's: 64-bit products are the dearest instructions here
      const int step = 64 / CH, row = lane / CH;
      int dn, dg;
      page_split(a.by_G, x + row, n, g);
      page_split(a.by_G, step, dn, dg);
      p += n * by_node + (h * G + g) * by_head;
      for (int i = 0; i < CH / 2; i++) {
        piece(i, row + step * i, lane % CH, p, x + row + step * i < M);
        p += dn * by_node + dg * by_head;
        g += dg;
        if (g >= G) {
          g -= G;
          p += by_node - G * by_head;
        }
      }
    }
  };
  // the pieces of a tile that thread t moves: at pc(i), as it lies in LDS, of row prow(i)
  auto prow = [&](int i) { return CH == 12 ? (t + BLOCK * i) / CH : t / CH + BLOCK / CH * i; };
  auto pc = [&](int i) { return CH == 12 ? (t + BLOCK * i) % CH : t % CH; };

  {
    const int first = uni(sh.first), last = uni(sh.last), cached = min(last, uni(sp.cache_tiles));
    int tile = first;
    bool bad = sp.bad;
    float top = -INFINITY, sum = 0.f;  // the row's reference and its sum of weights
    f32x16 o[DB];
    for (int d = 0; d < DB; d++)
      for (int i = 0; i < 16; i++) o[d][i] = 0.f;
    u32x4 qf[KSTEPS];
    // the nodes' keys and values, in the same way as the cache's
    int nkb = 0, nvb = 0;  // the buffers they are in
    const T* kd = (const T*)a.kd + b * a.kds[0] + h * a.kds[2];
    const T* vd = (const T*)a.vd + b * a.vds[0] + h * a.vds[2];
    auto stage_nodes = [&](int tile) {
      for (int i = 0; i < PER; i++) {
        const int row = prow(i), n = min((tile - uni(sp.cache_tiles)) * WIDE_TILE + row, a.N - 1);
        const int ck = key_piece<CH>(row, pc(i)) * 8, cv = value_slot<CH>(row, pc(i)) * 8;
        const uint32_t to = lds_at + wave * 1024 + i * BLOCK * 16;
        to_lds(FULL || ck < a.D ? (const void*)(kd + n * a.kds[1] + ck) : att_zero, to + nkb * TILE_BYTES);
        to_lds(FULL || cv < a.D ? (const void*)(vd + n * a.vds[1] + cv) : att_zero, to + VBUF + nvb * TILE_BYTES);
      }
    };

    auto scores = [&](f32x16* s, uint32_t buf) {
      for (int c = 0; c < 2; c++) {
        for (int i = 0; i < 16; i++) s[c][i] = 0.f;
        for (int k = 0; k < KSTEPS; k++)
          s[c] = mfma32(lds_read<u32x4>(koff[k] + buf, c * 32 * CH * 16), qf[k], s[c], T());
      }
    };
    // The weights are taken from a reference that follows the maximum: it moves when a score is over it by 2^8 in the
    // weights, so that the sums are seldom scaled anew.
    auto follow = [&](const f32x16* s) {
      float mx = top;
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[c][i]);
      mx = pair_max(mx);
      if (__any((mx - top) * scale > SLACK)) {
        const float f = __builtin_amdgcn_exp2f((top - at_least(mx)) * scale);
        top = mx;
        sum *= f;
        for (int d = 0; d < DB; d++) o[d] *= f;
      }
    };
    auto weigh = [&](const f32x16* s, u32x4* p) {
      const float from = at_least(top);
      float part[4] = {0.f, 0.f, 0.f, 0.f};
      for (int c = 0; c < 2; c++)
        for (int i = 0; i < 16; i += 2) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[c][i] - from, scale, Half<T>::bias));
          const float y = __builtin_amdgcn_exp2f(fmaf(s[c][i + 1] - from, scale, Half<T>::bias));
          part[i / 2 % 4] += x + y;
          p[2 * c + i / 8][i / 2 % 4] = pack2<T>(x, y);
        }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
    };
    auto product = [&](const u32x4* p, uint32_t buf) {
      for (int st = 0; st < 4; st++)  // 16 keys: the lane's are 16 st + 4 hh + {0..3, 8..11}
        for (int d = 0; d < DB; d++) {
          const u32x2 x = lds_read_tr(voff[d] + buf, 16 * st * CH * 16), y = lds_read_tr(voff[d] + buf, (16 * st + 8) * CH * 16);
          o[d] = mfma32(u32x4{x[0], x[1], y[0], y[1]}, p[st], o[d], T());
        }
    };

    {
      const int len = uni(sp.len);
      if (t == 0) odd_.clear();
      const Parents parents = tree_parents(a.N, a.parents + b * a.parents_stride);
      const Pages pages = {a.table + b * a.table_stride, a.div, a.P, a.M};
      const char* kc = (const char*)((const T*)a.kc + h * a.khead);
      const char* vc = (const char*)((const T*)a.vc + h * a.vhead);
      // A row's place is worked out once, by the lanes of one wave (the waves take turns), and goes to the others through
      // LDS; its table entry is loaded TURN tiles before that, and looked at only then: nothing waits for it.
      int entry = 0, slot = 0;
      auto find = [&](int tile) { entry = page_entry(pages, min(tile * WIDE_TILE + lane, len - 1), slot); };
      auto locate = [&](int tile) {
        if (!good_page(pages, entry)) {  // reads page 0, and the sequence's rows become NaN
          bad = true;
          entry = 0;
        }
        offs[tile & 3][0][lane] = cache_row(entry, slot, a.kpage, a.kslot);
        offs[tile & 3][1][lane] = (first + tile) * WIDE_TILE + lane < len ? cache_row(entry, slot, a.vpage, a.vslot)
                                                                          : (uint64_t)((const char*)att_zero - vc);
      };
      // tiles t of the part are counted from its first: what is in LDS where goes by t & 1 and t & 3
      auto stage = [&](int t, int kv, int buf) {
        const uint32_t to = lds_at + kv * VBUF + buf * TILE_BYTES + wave * 1024;  // the wave's 64 pieces in a row
        for (int i = 0; i < PER; i++) {
          const int row = prow(i), c = (kv ? value_slot<CH>(row, pc(i)) : key_piece<CH>(row, pc(i))) * 8;
          const char* p = (kv ? vc : kc) + offs[t & 3][kv][row] + c * 2;
          to_lds(FULL || c < a.D ? (const void*)p : att_zero, to + i * BLOCK * 16);
        }
      };
      if (rows)
        walk((const T*)a.q + b * a.qs[0], a.qs[1], a.qs[2], [&](int i, int row, int at, const T* p, bool in) {
          const int c = key_piece<CH>(row, at) * 8;
          to_lds(in && (FULL || c < a.D) ? (const void*)(p + c) : att_zero, lds_at + own + i * 1024);
        });
      const int n_cached = cached - tile;  // (of this part; at most 0 when it has the nodes alone)
      if (n_cached > 0) {
        find(first + wave);
        for (int k = wave; k < 3; k += TURN) {
          locate(k);
          find(first + k + TURN);
        }
      }
      wait_loads();
      if (rows) {
        for (int k = 0; k < KSTEPS; k++) qf[k] = lds_read<u32x4>(koff[k] + own, 0);
        if (a.scale < 0.f)
          for (int k = 0; k < KSTEPS; k++) qf[k] = negative(qf[k]);
      }
      __syncthreads();
      if (n_cached <= 0) {
        stage_nodes(tile);
      } else {
        stage(0, 0, 0);
        stage(0, 1, 0);
        if (n_cached > 1) stage(1, 0, 1);
      }
      tree_paths(tr, a.N, parents);

      // The cache's tiles: a tile's scores are worked out while the weights of the one before it are, in the matrix
      // unit and beside it.  So K comes two tiles ahead and V one.
      f32x16 s[2], n[2];
      auto hide = [&](f32x16* s, int t) {  // key 32 c + 8 (i / 4) + 4 hh + i % 4 of the tile
        const int base = (first + t) * WIDE_TILE;
        if (base + WIDE_TILE <= len) return;
        for (int c = 0; c < 2; c++)
          for (int i = 0; i < 16; i++)
            if (base + 32 * c + 8 * (i / 4) + 4 * hh + i % 4 >= len) s[c][i] = -INFINITY;
      };
      auto arrive = [&](int t, int buf) {
        wait_loads();     // this wave's pieces are in LDS
        __syncthreads();  // everyone's are; what the last tile was read from is free
        if (wave == ((t + 3) & (TURN - 1))) {
          locate(t + 3);
          find(first + t + 3 + TURN);
        }
        if (t + 2 < n_cached) stage(t + 2, 0, buf);
        if (t + 1 < n_cached) stage(t + 1, 1, buf ^ 1);
      };
      // tile t, whose scores are s, and the scores n of the next; in eight steps, each with products beside the
      // exponentials of another step's weights
      auto turn = [&](const f32x16* s, f32x16* n, int t, int buf) {
        const uint32_t vb = buf * TILE_BYTES, kb = vb ^ TILE_BYTES;
        const float from = at_least(top);
        float part[2] = {0.f, 0.f};
        u32x4 p[4];
        auto keys = [&](int i) {
          for (int k = i * KSTEPS / 4; k < (i + 1) * KSTEPS / 4; k++)
            for (int c = 0; c < 2; c++) {
              const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
              n[c] = mfma32(lds_read<u32x4>(koff[k], kb + c * 32 * CH * 16), qf[k], k ? n[c] : zero, T());
            }
        };
        auto values = [&](int st) {
          for (int d = 0; d < DB; d++) {
            const u32x2 x = lds_read_tr(voff[d], vb + 16 * st * CH * 16), y = lds_read_tr(voff[d], vb + (16 * st + 8) * CH * 16);
            o[d] = mfma32(u32x4{x[0], x[1], y[0], y[1]}, p[st], o[d], T());
          }
        };
        auto expo = [&](int st, int half) {
          for (int e = 0; e < 4; e += 2) {
            const int i = 8 * (st & 1) + 4 * half + e;
            const float x = __builtin_amdgcn_exp2f(fmaf(s[st / 2][i] - from, scale, Half<T>::bias));
            const float y = __builtin_amdgcn_exp2f(fmaf(s[st / 2][i + 1] - from, scale, Half<T>::bias));
            part[half] += x + y;
            p[st][2 * half + e / 2] = pack2<T>(x, y);
          }
        };
        auto then = []() { __builtin_amdgcn_sched_barrier(0); };
        expo(0, 0), keys(0);
        then();
        expo(0, 1), keys(1);
        then();
        expo(1, 0), values(0);
        then();
        expo(1, 1), keys(2);
        then();
        expo(2, 0), values(1);
        then();
        expo(2, 1), keys(3);
        then();
        expo(3, 0), expo(3, 1), values(2);
        then();
        values(3);
        sum += part[0] + part[1];
        hide(n, t + 1);
        follow(n);
      };
      if (n_cached > 0) {
        wait_loads();
        __syncthreads();
        if (rows) {
          scores(s, 0);
          hide(s, 0);
          follow(s);
        }
        int t = 0;
        for (; t + 2 < n_cached; t += 2) {
          arrive(t, 0);
          if (rows) turn(s, n, t, 0);
          arrive(t + 1, 1);
          if (rows) turn(n, s, t + 1, 1);
        }
        if (t + 1 < n_cached) {
          arrive(t, 0);
          if (rows) turn(s, n, t, 0);
          t++;
          s[0] = n[0];
          s[1] = n[1];
        }
        arrive(t, t & 1);
        if (cached < last) {
          nvb = (t & 1) ^ 1;
          stage_nodes(cached);
        }
        if (rows) {
          u32x4 p[4];
          weigh(s, p);
          product(p, (t & 1) * TILE_BYTES);
        }
        tile = cached;
      }
    }

    // the tree's own keys, one tile after the other
    while (tile < last) {
      const int base = (tile - uni(sp.cache_tiles)) * WIDE_TILE;
      wait_loads();
      // a value that is not finite would reach every row as 0 times itself: it becomes 0 and is added on its own path
      for (int i = 0; i < PER; i++) {
        u32x4* at = (u32x4*)(lds + VBUF + nvb * TILE_BYTES + (t + BLOCK * i) * 16);
        if (not_finite<T>(*at)) {
          *at = u32x4{0, 0, 0, 0};
          odd_.mark(base);
        }
      }
      __syncthreads();
      const int kb = nkb, vb = nvb;
      const bool more = ++tile < last, odd = odd_.marked(base);
      if (more && !odd) {  // (else the other buffers are needed below)
        nkb ^= 1;
        nvb ^= 1;
        stage_nodes(tile);
      }
      f32x16 s[2];
      u32x4 p[4];
      if (rows) {
        scores(s, kb * TILE_BYTES);
        for (int c = 0; c < 2; c++) {
          const uint32_t set = m < M ? tr.anc[node][base / 32 + c] >> (4 * hh) : 0;
          for (int i = 0; i < 16; i++) s[c][i] = if_bit(set, 8 * (i / 4) + i % 4, s[c][i]);
        }
        follow(s);
        weigh(s, p);
        product(p, vb * TILE_BYTES);
      }
      if (!odd) continue;
      // the sums of what went in as 0 (the finite values of its pieces with their weights), two waves at a time, in the LDS
      // that the tile does not use
#pragma unroll 1
      for (int turn = 0; turn < W; turn += 2) {
        if (turn) __syncthreads();
        if (!rows || uni(wave) / 2 * 2 != turn) continue;
        float* mine = (float*)(lds + (wave & 1 ? VBUF + (vb ^ 1) * TILE_BYTES : (kb ^ 1) * TILE_BYTES)) + l32 * DP;
#pragma unroll 1
        for (int d = 4 * hh; d < DP; d += 8) *(f32x4*)(mine + d) = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int j = 0; j < WIDE_TILE && base + j < a.N; j++) {
          if (m >= M || !(tr.anc[node][(base + j) / 32] >> (j % 32) & 1)) continue;
          const T* v = vd + (base + j) * a.vds[1];
          const T* k = kd + (base + j) * a.kds[1];
          const T* q = (const T*)a.q + b * a.qs[0] + node * a.qs[1] + (h * G + head) * a.qs[2];
          float dot = 0.f;
#pragma unroll 1
          for (int e = 0; e < a.D; e++) dot = fmaf((float)q[e], (float)k[e], dot);
          const float w = __builtin_amdgcn_exp2f(fmaf((a.scale < 0.f ? -dot : dot) - at_least(top), scale, Half<T>::bias));
#pragma unroll 1
          for (int d = 4 * hh; d < a.D; d += 8) {
            if (!not_finite<T>(*(const u32x4*)(v + d / 8 * 8))) continue;
            for (int i = 0; i < 4; i++) {
              const float y = (float)v[d + i];
              mine[d + i] += isfinite(y) ? w * y : y;
            }
          }
        }
        wave_order();
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const f32x4 x = *(const f32x4*)(mine + 32 * d + 8 * i + 4 * hh);
#pragma unroll
            for (int e = 0; e < 4; e++) o[d][4 * i + e] += x[e];
          }
      }
      __syncthreads();
      if (more) stage_nodes(tile);
    }

    sum += __shfl_xor(sum, 32);
    if (__syncthreads_or(bad)) sum = NAN;
    if (m < M) {
      const int64_t at = part_row(a, rt, item, part, ROWS, wave * 32 + l32);
      const bool here = tr.anc[node][node / 32] >> (node % 32) & 1;
      const float f = 1.f / sum;
      if (sh.parts > 1 && hh == 0) {
        float* ml = part_sums(a, a.row_tiles, ROWS) + 2 * at;
        ml[0] = here ? top : -INFINITY;
        ml[1] = here ? sum : PART_ABSENT;
      }
      for (int d = 0; d < DB; d++)
        for (int i = 0; i < 4; i++) {
          const int x = 32 * d + 8 * i + 4 * hh;
          if (x >= a.D) continue;
          const f32x4 y = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]}, none = {0.f, 0.f, 0.f, 0.f};
          if (sh.parts > 1)
            *(f32x4*)(a.part + at * a.D + x) = here ? y : none;
          else
            *(uint64_t*)(lds + own + (l32 * CH + key_slot<CH>(l32, 4 * d + i)) * 16 + 8 * hh) = here ? pack4<T>(y * f) : 0;
        }
    }
    if (sh.parts == 1 && rows) {
      wave_order();
      const int64_t line = (int64_t)a.Hq * a.D;
      walk((const T*)a.out + (int64_t)b * a.N * line, line, a.D, [&](int, int row, int c, const T* p, bool in) {
        if (in && (FULL || c * 8 < a.D))
          *(u32x4*)(const_cast<T*>(p) + c * 8) = *(const u32x4*)(lds + own + (row * CH + key_slot<CH>(row, c)) * 16);
      });
    }
  }
}

// Joins the parts: D / 4 threads a row, BY of them over its parts, J parts in flight each.  Rows of sequences with
// one part were written already.  4 us for few parts, of which 3 are the launch and its first loads; 512 rows of 128 of 63
// parts 7.4 us (18 MB).
template <typename T, int BY, int J>
__global__ __launch_bounds__(ATT_BLOCK) void k_attend_join(AttendArgs a, int rows, int tile) {
  __shared__ f32x4 acc_[BY > 1 ? ATT_BLOCK : 1];
  __shared__ float ml_[2][BY > 1 ? ATT_BLOCK : 1];
  const int G = a.by_G.d, M = a.N * G, t = threadIdx.x;
  const int q = a.D / 4, each = ATT_BLOCK / (q * BY);  // rows a workgroup
  const int r = t / (q * BY), by = t / q % BY, d = t % q * 4;
  const uint32_t x = blockIdx.x * each + r;  // (the host keeps the rows below 2^31)
  const bool on = r < each && x < (uint32_t)(a.B * a.Hkv * M);
  const int bh = on ? (int)(x / (uint32_t)M) : 0, m = on ? (int)(x - bh * M) : 0, b = bh / a.Hkv, h = bh - b * a.Hkv, n = m / G;
  const int parts = on ? share_of(a, span_of(a, b, tile).tiles, 0).parts : 1;
  const float scale = score_scale(a.scale);
  const int64_t base = part_row(a, m / rows, bh, 0, rows, m % rows);
  const float* ml = part_sums(a, a.row_tiles, rows);
  float mx = -INFINITY, total = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float m2, float l2, f32x4 v) {
    const float up = fmaxf(mx, m2), from = at_least(up);
    const float f = __builtin_amdgcn_exp2f((mx - from) * scale), g = __builtin_amdgcn_exp2f((m2 - from) * scale);
    total = total * f + l2 * g;
    acc = acc * f + v * g;
    mx = up;
  };
  if (parts > 1)
    for (int k = by; k < parts; k += J * BY) {
      float m2[J], l2[J];
      f32x4 v[J];
#pragma unroll
      for (int j = 0; j < J; j++) {
        const int64_t at = base + (int64_t)min(k + j * BY, parts - 1) * rows;
        m2[j] = ml[2 * at];
        l2[j] = ml[2 * at + 1];
        v[j] = *(const f32x4*)(a.part + at * a.D + d);
      }
#pragma unroll
      for (int j = 0; j < J; j++)
        if (k + j * BY < parts) add(m2[j], l2[j], v[j]);
    }
  if constexpr (BY > 1) {
    acc_[t] = acc;
    ml_[0][t] = mx;
    ml_[1][t] = total;
    __syncthreads();
    if (by || r >= each) return;
    for (int k = 1; k < BY; k++) add(ml_[0][t + k * q], ml_[1][t + k * q], acc_[t + k * q]);
  }
  if (parts == 1) return;
  const bool absent = ml[2 * base + 1] == PART_ABSENT;
  T* out = (T*)a.out + (((int64_t)b * a.N + n) * a.Hq + h * G + m - n * G) * a.D + d;
  *(uint64_t*)out = absent ? 0 : pack4<T>(acc * (1.f / total));
}

}  // namespace gb
