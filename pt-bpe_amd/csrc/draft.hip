// draft.hip -- C entries of the decoding operators (include/geobpe.h, "decoding"): device pointers,
// the caller's stream, no allocation and no synchronisation, so every call can be captured.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <type_traits>

#include "../../include/geobpe.h"
#include "draft_attend.h"
#include "draft_commit.h"
#include "draft_verify.h"

using namespace gb;

namespace {
thread_local char g_draft_error[256];

int fail(int rc, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_draft_error, sizeof(g_draft_error), fmt, ap);
  va_end(ap);
  return rc;
}

// the caller's device, put back at the end
struct OnDevice {
  int old = -1;
  bool ok;
  explicit OnDevice(int device) {
    ok = hipGetDevice(&old) == hipSuccess && (old == device || hipSetDevice(device) == hipSuccess);
    if (old == device) old = -1;
  }
  ~OnDevice() {
    if (old >= 0) (void)hipSetDevice(old);
  }
};

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? GEOBPE_OK : fail(GEOBPE_EHIP, "%s: %s", what, hipGetErrorString(e));
}

bool aligned(const void* p, const int64_t* strides, int n, int64_t unit) {
  if ((uintptr_t)p % 16) return false;
  for (int i = 0; i < n; i++)
    if (strides[i] % unit) return false;
  return true;
}

// How a call is cut: rows a workgroup works on, tiles of keys a part has at most.  The host does not know the lengths, so the
// cut is made for the table's positions: short sequences under a long table make few parts (4 x 8 heads over 8191 of 131072
// positions 228 + 5 us, over 8191 of 8191 30 + 7; the figures below are of tables that fit the longest sequence).
struct AttendPlan {
  bool wide;
  int rb, waves, rows, tile, per, most;
  int64_t row_tiles, blocks, bytes;
};
AttendPlan attend_plan(const geobpe_attend_args& x) {
  AttendPlan p;
  const int64_t M = x.nodes * (x.heads / x.kv_heads);
  p.wide = M > (x.head_dim > 128 ? 16 : 32);
  p.rb = M <= 16 ? 1 : 2;
  p.tile = p.wide ? WIDE_TILE : ATT_TILE;
  const int64_t tiles = (x.max_pages * x.page_size + p.tile - 1) / p.tile + (x.nodes + p.tile - 1) / p.tile;
  const int64_t items = x.seqs * x.kv_heads;
  // Where the tiles are many: 256 rows share one where there are more than 128 and heads of 128 (32 sequences x 8 heads of
  // 256 rows over 16k: 508 us instead of 548), 64 where there are no more and the heads are narrow, so that no wave is
  // idle (40 x 8 heads of 48 rows over 9k: 102 us instead of 115; with heads of 64, which wait for memory, 122 instead of
  // 114).  Where they are few 128 make more workgroups (2 heads of 432 rows over 960: 18 us instead of 22; 16 heads of 40
  // rows over 3k: 14.1 instead of 16.0).
  const bool many = items * ((M + 255) / 256) * tiles >= WIDE_MANY;
  p.rows = !p.wide ? 16 * p.rb
           : many && M > 128 && x.head_dim > 96 && x.head_dim <= 128 ? 256
           : many && M <= 64 && x.head_dim <= 32 ? 64 : 128;
  p.row_tiles = (M + p.rows - 1) / p.rows;
  // With few rows eight waves where sequences need not be cut then: 128 to 256 workgroups (64 sequences x 4 heads: 26 us
  // instead of 25 + 10 for the join; 160 x 1000 positions 16 instead of 24), or 17 to 32 tiles (600 positions 10.0 instead of
  // 12.0; at 33 tiles of heads of 128 17.4 instead of 16.1); else four, and finer parts (7 x 12 heads: 27 us instead of 40).
  const int64_t uncut = items * p.row_tiles;
  const bool eight = x.head_dim <= 128 && uncut <= 256 && (uncut >= 128 || (tiles > ATT_LEAST && tiles <= 32));
  p.waves = p.wide ? p.rows / 32 : eight ? 8 : 4;
  const int64_t want = ATT_WANT * 4 / p.waves;
  int64_t even = (uncut * tiles + want - 1) / want;
  // where whole parts are more than that after all, and a second round of workgroups would be a small one, they are half
  // as long (86 x 4 heads over 4k to 8k positions, 688 workgroups: 193 us instead of 241; 12 x 2 over 33k to 66k, 528: 125
  // instead of 160.  With 512 in the first place it takes longer: 16 x 2 heads over up to 12k 53 instead of 42)
  if (even < tiles && uncut * ((tiles + even - 1) / even) > want) even = (even + 1) / 2;
  // The least tiles of a part.  Sequences stay whole up to 256 tiles with eight waves and few rows (160 sequences of 2000 or
  // 8000 positions: 23 us instead of 34, 64 instead of 72), and up to 96 where they make a round of workgroups without a
  // cut: few rows, 320 over up to 3000 positions 84 us instead of 103 (but 400 over up to 4000 74 instead of 66); many,
  // 480 over 2000 64 instead of 83, 320 over 3k to 6k 201 instead of 227 (but 344 over 4k to 8k 219 instead of 194).
  const int least = !p.wide && p.waves == 8 ? 256 : uncut >= 256 && tiles <= 96 ? 96 : p.wide ? WIDE_LEAST : ATT_LEAST;
  p.per = (int)(even > tiles ? tiles : even > least ? even : least);
  p.most = (int)((tiles + p.per - 1) / p.per);
  p.blocks = (items * p.most + 7) / 8 * 8 * p.row_tiles;
  p.bytes = p.most > 1 ? uncut * p.most * p.rows * (x.head_dim + 2) * 4 : 0;
  return p;
}
int attend_sizes(const geobpe_attend_args& x, AttendPlan& plan) {
  if (x.seqs < 0 || x.nodes < 1 || x.nodes > DRAFT_MAX_NODES || x.kv_heads < 1 || x.heads < x.kv_heads ||
      x.heads % x.kv_heads || x.head_dim < 8 || x.head_dim > 256 || x.head_dim % 8 || x.page_size < 1 || x.pages < 1 ||
      x.max_pages < 0 || x.dtype < 0 || x.dtype > 1 || x.seqs > 65535 || x.heads > 65535 || x.pages > INT32_MAX ||
      x.page_size > DRAFT_MAX_POSITIONS || x.max_pages > DRAFT_MAX_POSITIONS / x.page_size)
    return fail(GEOBPE_EARG, "tree attention: sizes out of range");
  if (x.seqs == 0) return GEOBPE_OK;
  if (x.seqs * x.nodes * x.heads > INT32_MAX / ATT_BLOCK || (plan = attend_plan(x)).blocks > INT32_MAX / ATT_BLOCK)
    return fail(GEOBPE_EARG, "tree attention: %lld sequences of %lld rows are too many for one call", (long long)x.seqs,
                (long long)(x.nodes * x.heads));
  return GEOBPE_OK;
}

template <typename T, int KS>
void attend_narrow(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)p.blocks), block(64 * p.waves);
  if constexpr (KS > 4) {
    hipLaunchKernelGGL((k_attend<T, KS, 1, 4>), grid, block, 0, s, a);
  } else if (p.waves == 8) {
    if (p.rb == 1)
      hipLaunchKernelGGL((k_attend<T, KS, 1, 8>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((k_attend<T, KS, 2, 8>), grid, block, 0, s, a);
  } else {
    if (p.rb == 1)
      hipLaunchKernelGGL((k_attend<T, KS, 1, 4>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((k_attend<T, KS, 2, 4>), grid, block, 0, s, a);
  }
}
template <typename T>
void attend_launch(const AttendArgs& a, const AttendPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)p.blocks), block(64 * p.waves);
  if (p.wide) {
    if (p.waves == 2)
      hipLaunchKernelGGL((k_attend_wide<T, 32, false, 2>), grid, block, 0, s, a);
    else if (a.D <= 32)
      hipLaunchKernelGGL((k_attend_wide<T, 32, false, 4>), grid, block, 0, s, a);
    else if (a.D > 64 && a.D <= 96)
      hipLaunchKernelGGL((k_attend_wide<T, 96, false, 4>), grid, block, 0, s, a);
    else if (a.D == 64)
      hipLaunchKernelGGL((k_attend_wide<T, 64, true, 4>), grid, block, 0, s, a);
    else if (a.D < 64)
      hipLaunchKernelGGL((k_attend_wide<T, 64, false, 4>), grid, block, 0, s, a);
    else if (a.D == 128 && p.waves == 8)
      hipLaunchKernelGGL((k_attend_wide<T, 128, true, 8>), grid, block, 0, s, a);
    else if (a.D == 128)
      hipLaunchKernelGGL((k_attend_wide<T, 128, true, 4>), grid, block, 0, s, a);
    else if (a.D < 128 && p.waves == 8)
      hipLaunchKernelGGL((k_attend_wide<T, 128, false, 8>), grid, block, 0, s, a);
    else if (a.D < 128)
      hipLaunchKernelGGL((k_attend_wide<T, 128, false, 4>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((k_attend_wide<T, 256, false, 4>), grid, block, 0, s, a);
  } else {
    switch ((a.D + 31) / 32) {
      case 1: attend_narrow<T, 1>(a, p, s); break;
      case 2: attend_narrow<T, 2>(a, p, s); break;
      case 3: attend_narrow<T, 3>(a, p, s); break;
      case 4: attend_narrow<T, 4>(a, p, s); break;
      case 5:
      case 6: attend_narrow<T, 6>(a, p, s); break;
      default: attend_narrow<T, 8>(a, p, s);
    }
  }
  if (p.most > 1) {
    // eight threads over a row's parts where they are many and the rows too few to fill the card
    const int64_t rows = (int64_t)a.B * a.N * a.Hq;
    const int by = p.most > 16 && rows * (a.D / 4) < 512 * ATT_BLOCK && a.D <= 128 ? 8 : 1, each = ATT_BLOCK / (a.D / 4 * by);
    const dim3 joins((unsigned)((rows + each - 1) / each));
    if (by == 8)
      hipLaunchKernelGGL((k_attend_join<T, 8, 8>), joins, dim3(ATT_BLOCK), 0, s, a, p.rows, p.tile);
    else if (p.most > 2)
      hipLaunchKernelGGL((k_attend_join<T, 1, 8>), joins, dim3(ATT_BLOCK), 0, s, a, p.rows, p.tile);
    else
      hipLaunchKernelGGL((k_attend_join<T, 1, 2>), joins, dim3(ATT_BLOCK), 0, s, a, p.rows, p.tile);
  }
}

template <typename T, bool HELD, int W>
void verify_waves(const VerifyArgs& a, hipStream_t s) {
  if (a.draft)
    hipLaunchKernelGGL((k_verify<T, true, HELD, W>), dim3((unsigned)a.B), dim3(64 * W), 0, s, a);
  else
    hipLaunchKernelGGL((k_verify<T, false, HELD, W>), dim3((unsigned)a.B), dim3(64 * W), 0, s, a);
}
template <typename T>
void verify_launch(const VerifyArgs& a, hipStream_t s) {
  if (a.V <= VER_SMALL)
    a.C ? verify_waves<T, true, 4>(a, s) : verify_waves<T, false, 4>(a, s);
  else
    a.C ? verify_waves<T, true, 16>(a, s) : verify_waves<T, false, 16>(a, s);
}
}  // namespace

extern "C" {

const char* geobpe_draft_error(void) { return g_draft_error; }

int64_t geobpe_tree_attention_work(const geobpe_attend_args* p) {
  AttendPlan plan;
  if (!p || attend_sizes(*p, plan) != GEOBPE_OK) return -1;
  return p->seqs ? plan.bytes : 0;
}

int geobpe_tree_attention(int device, void* stream, const geobpe_attend_args* p, void* d_work, int64_t work_bytes) {
  if (!p) return fail(GEOBPE_EARG, "no arguments");
  const geobpe_attend_args& x = *p;
  AttendPlan plan;
  const int rc = attend_sizes(x, plan);
  if (rc != GEOBPE_OK) return rc;
  if (!(fabs(x.scale) <= 2e38)) return fail(GEOBPE_EARG, "tree attention: scale %g is not finite in 32 bits", x.scale);
  if (x.seqs == 0) return GEOBPE_OK;
  if (!x.d_q || !x.d_k_cache || !x.d_v_cache || !x.d_k || !x.d_v || !x.d_lens || !x.d_parents || !x.d_out ||
      (x.max_pages && !x.d_table) || (plan.bytes && !d_work))
    return fail(GEOBPE_EARG, "tree attention: null pointer");
  if (work_bytes < plan.bytes)
    return fail(GEOBPE_EARG, "tree attention: %lld bytes of work space, %lld are needed", (long long)work_bytes,
                (long long)plan.bytes);
  if (!aligned(x.d_q, x.q_stride, 3, 8) || !aligned(x.d_k_cache, x.kc_stride, 3, 8) ||
      !aligned(x.d_v_cache, x.vc_stride, 3, 8) || !aligned(x.d_k, x.k_stride, 3, 8) ||
      !aligned(x.d_v, x.v_stride, 3, 8) || (uintptr_t)x.d_out % 16 || (uintptr_t)d_work % 16)
    return fail(GEOBPE_EARG, "tree attention: rows are not 16-byte aligned");
  for (int i = 0; i < 2; i++)
    if (x.kc_stride[i] < 0 || x.vc_stride[i] < 0 || x.kc_stride[i] / 8 > UINT32_MAX || x.vc_stride[i] / 8 > UINT32_MAX)
      return fail(GEOBPE_EARG, "tree attention: a page or slot of the cache spans more than 64 GiB");
  AttendArgs a;
  a.q = x.d_q, a.kc = x.d_k_cache, a.vc = x.d_v_cache, a.kd = x.d_k, a.vd = x.d_v, a.out = x.d_out;
  a.table = (const int32_t*)x.d_table, a.lens = (const int32_t*)x.d_lens, a.parents = (const int32_t*)x.d_parents;
  for (int i = 0; i < 3; i++) a.qs[i] = x.q_stride[i], a.kds[i] = x.k_stride[i], a.vds[i] = x.v_stride[i];
  a.khead = x.kc_stride[2], a.vhead = x.vc_stride[2];
  a.kpage = (uint32_t)(x.kc_stride[0] / 8), a.kslot = (uint32_t)(x.kc_stride[1] / 8);
  a.vpage = (uint32_t)(x.vc_stride[0] / 8), a.vslot = (uint32_t)(x.vc_stride[1] / 8);
  a.table_stride = x.table_stride, a.parents_stride = x.parents_stride;
  a.B = (int)x.seqs, a.N = (int)x.nodes, a.Hq = (int)x.heads, a.Hkv = (int)x.kv_heads, a.D = (int)x.head_dim;
  a.S = (int)x.page_size, a.P = (int)x.pages, a.M = (int)x.max_pages;
  a.div = page_div(a.S);
  a.scale = (float)x.scale;
  a.per = plan.per;
  a.most = plan.most;
  a.row_tiles = (int)plan.row_tiles;
  a.by_G = page_div(a.Hq / a.Hkv), a.by_Hkv = page_div(a.Hkv), a.by_most = page_div(a.most), a.by_per = page_div(a.per),
  a.by_RT = page_div(a.row_tiles);
  a.part = (float*)d_work;
  OnDevice on(device);
  if (!on.ok) return fail(GEOBPE_EHIP, "tree attention: device %d", device);
  if (x.dtype == 0)
    attend_launch<bf16_t>(a, plan, (hipStream_t)stream);
  else
    attend_launch<fp16_t>(a, plan, (hipStream_t)stream);
  return launched("tree attention");
}

int geobpe_verify_draft(int device, void* stream, const geobpe_verify_args* p) {
  if (!p) return fail(GEOBPE_EARG, "no arguments");
  const geobpe_verify_args& x = *p;
  if (x.seqs < 0 || x.seqs > INT32_MAX / 1024 || x.nodes < 1 || x.nodes > DRAFT_MAX_NODES || x.vocab < 1 ||
      x.vocab > VER_MAX_VOCAB || x.classes < 0 || x.classes > INT32_MAX || x.dtype < 0 || x.dtype > 2)
    return fail(GEOBPE_EARG, "verify: sizes out of range");
  if (x.seqs == 0) return GEOBPE_OK;
  if (!x.d_parents || !x.d_ids || !x.d_target || !x.d_u || !x.d_n || !x.d_path || !x.d_tokens ||
      (x.classes && (!x.d_ranges || !x.d_start)))
    return fail(GEOBPE_EARG, "verify: null pointer");
  VerifyArgs a;
  a.parents = (const int32_t*)x.d_parents, a.ids = x.d_ids, a.target = x.d_target, a.draft = x.d_draft;
  a.u = (const float*)x.d_u, a.ranges = (const int32_t*)x.d_ranges, a.start = (const int32_t*)x.d_start;
  a.n = (int32_t*)x.d_n, a.path = (int32_t*)x.d_path, a.tokens = (int32_t*)x.d_tokens;
  a.parents_stride = x.parents_stride, a.ids_stride = x.ids_stride, a.u_stride = x.u_stride;
  for (int i = 0; i < 2; i++) a.ts[i] = x.target_stride[i], a.ds[i] = x.draft_stride[i];
  a.B = (int)x.seqs, a.N = (int)x.nodes, a.V = (int)x.vocab, a.C = (int)x.classes, a.ids64 = x.ids_int64 != 0;
  OnDevice on(device);
  if (!on.ok) return fail(GEOBPE_EHIP, "verify: device %d", device);
  const hipStream_t s = (hipStream_t)stream;
  if (x.dtype == 0)
    verify_launch<bf16_t>(a, s);
  else if (x.dtype == 1)
    verify_launch<fp16_t>(a, s);
  else
    verify_launch<float>(a, s);
  return launched("verify");
}

int geobpe_commit_draft(int device, void* stream, const geobpe_commit_args* p) {
  if (!p) return fail(GEOBPE_EARG, "no arguments");
  const geobpe_commit_args& x = *p;
  if (x.layers < 1 || x.layers > 65535 || x.seqs < 0 || x.nodes < 1 || x.nodes > DRAFT_MAX_NODES || x.kv_heads < 1 ||
      x.kv_heads > 65535 || x.head_bytes < 16 || x.head_bytes > 65536 || x.head_bytes % 16 || x.page_size < 1 ||
      x.pages < 1 || x.max_pages < 0 || x.pages > INT32_MAX || x.page_size > DRAFT_MAX_POSITIONS ||
      x.max_pages > DRAFT_MAX_POSITIONS / x.page_size || x.seqs > INT32_MAX / 256 / x.nodes)
    return fail(GEOBPE_EARG, "commit: sizes out of range");
  if (x.seqs == 0) return GEOBPE_OK;
  if (!x.d_k || !x.d_v || !x.d_k_cache || !x.d_v_cache || !x.d_lens || !x.d_path || !x.d_n || !x.d_lens_out ||
      (x.max_pages && !x.d_table))
    return fail(GEOBPE_EARG, "commit: null pointer");
  if (x.d_lens_out == x.d_lens) return fail(GEOBPE_EARG, "commit: the new lengths would replace those that are still read");
  if (!aligned(x.d_k, x.k_stride, 4, 16) || !aligned(x.d_v, x.v_stride, 4, 16) ||
      !aligned(x.d_k_cache, x.kc_stride, 4, 16) || !aligned(x.d_v_cache, x.vc_stride, 4, 16))
    return fail(GEOBPE_EARG, "commit: rows are not 16-byte aligned");
  CommitArgs a;
  a.kd = (const char*)x.d_k, a.vd = (const char*)x.d_v, a.kc = (char*)x.d_k_cache, a.vc = (char*)x.d_v_cache;
  a.table = (const int32_t*)x.d_table, a.lens = (const int32_t*)x.d_lens, a.path = (const int32_t*)x.d_path;
  a.n = (const int32_t*)x.d_n, a.lens_out = (int32_t*)x.d_lens_out;
  for (int i = 0; i < 4; i++)
    a.kds[i] = x.k_stride[i], a.vds[i] = x.v_stride[i], a.kcs[i] = x.kc_stride[i], a.vcs[i] = x.vc_stride[i];
  a.table_stride = x.table_stride, a.path_stride = x.path_stride;
  a.L = (int)x.layers, a.B = (int)x.seqs, a.N = (int)x.nodes, a.Hkv = (int)x.kv_heads;
  a.S = (int)x.page_size, a.P = (int)x.pages, a.M = (int)x.max_pages, a.vecs = (int)(x.head_bytes / 16);
  a.div = page_div(a.S);
  OnDevice on(device);
  if (!on.ok) return fail(GEOBPE_EHIP, "commit: device %d", device);
  hipLaunchKernelGGL(k_commit_nodes, dim3((unsigned)(a.B * a.N), (unsigned)((a.L + COMMIT_LAYERS - 1) / COMMIT_LAYERS)),
                     dim3(256), 0, (hipStream_t)stream, a);
  return launched("commit");
}

}  // extern "C"
