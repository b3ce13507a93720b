// draft.hip -- C entries of the decoding operators (include/geobpe.h, "decoding"): device pointers,
// the caller's stream, no allocation and no synchronisation, so every call can be captured.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>

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
}  // namespace

extern "C" {

const char* geobpe_draft_error(void) { return g_draft_error; }

int geobpe_tree_attention(int device, void* stream, const geobpe_attend_args* p) {
  if (!p) return fail(GEOBPE_EARG, "no arguments");
  const geobpe_attend_args& x = *p;
  if (x.seqs < 0 || x.nodes < 1 || x.nodes > DRAFT_MAX_NODES || x.kv_heads < 1 || x.heads < x.kv_heads ||
      x.heads % x.kv_heads || x.head_dim < 8 || x.head_dim > 256 || x.head_dim % 8 || x.page_size < 1 || x.pages < 1 ||
      x.max_pages < 0 || x.dtype < 0 || x.dtype > 1 || x.seqs > 65535 || x.heads > 65535 || x.pages > INT32_MAX ||
      x.page_size > INT32_MAX || x.max_pages > INT32_MAX / x.page_size)
    return fail(GEOBPE_EARG, "tree attention: sizes out of range");
  if (x.seqs == 0) return GEOBPE_OK;
  if (!x.d_q || !x.d_k_cache || !x.d_v_cache || !x.d_k || !x.d_v || !x.d_lens || !x.d_parents || !x.d_out ||
      (x.max_pages && !x.d_table))
    return fail(GEOBPE_EARG, "tree attention: null pointer");
  if (!aligned(x.d_q, x.q_stride, 3, 8) || !aligned(x.d_k_cache, x.kc_stride, 3, 8) ||
      !aligned(x.d_v_cache, x.vc_stride, 3, 8) || !aligned(x.d_k, x.k_stride, 3, 8) ||
      !aligned(x.d_v, x.v_stride, 3, 8) || (uintptr_t)x.d_out % 16)
    return fail(GEOBPE_EARG, "tree attention: rows are not 16-byte aligned");
  AttendArgs a;
  a.q = x.d_q, a.kc = x.d_k_cache, a.vc = x.d_v_cache, a.kd = x.d_k, a.vd = x.d_v, a.out = x.d_out;
  a.table = (const int32_t*)x.d_table, a.lens = (const int32_t*)x.d_lens, a.parents = (const int32_t*)x.d_parents;
  for (int i = 0; i < 3; i++) {
    a.qs[i] = x.q_stride[i], a.kcs[i] = x.kc_stride[i], a.vcs[i] = x.vc_stride[i];
    a.kds[i] = x.k_stride[i], a.vds[i] = x.v_stride[i];
  }
  a.table_stride = x.table_stride, a.parents_stride = x.parents_stride;
  a.B = (int)x.seqs, a.N = (int)x.nodes, a.Hq = (int)x.heads, a.Hkv = (int)x.kv_heads, a.D = (int)x.head_dim;
  a.S = (int)x.page_size, a.P = (int)x.pages, a.M = (int)x.max_pages;
  a.div = page_div(a.S);
  a.scale = (float)x.scale;
  OnDevice on(device);
  if (!on.ok) return fail(GEOBPE_EHIP, "tree attention: device %d", device);
  const dim3 grid((unsigned)(a.N * a.Hq), (unsigned)a.B);
  if (x.dtype == 0)
    hipLaunchKernelGGL(k_attend_row<bf16_t>, grid, dim3(ATT_BLOCK), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(k_attend_row<fp16_t>, grid, dim3(ATT_BLOCK), 0, (hipStream_t)stream, a);
  return launched("tree attention");
}

int geobpe_verify_draft(int device, void* stream, const geobpe_verify_args* p) {
  if (!p) return fail(GEOBPE_EARG, "no arguments");
  const geobpe_verify_args& x = *p;
  if (x.seqs < 0 || x.seqs > INT32_MAX || x.nodes < 1 || x.nodes > DRAFT_MAX_NODES || x.vocab < 1 ||
      x.vocab > (int64_t)VER_TILES * VER_BLOCK * 4 || x.classes < 0 || x.classes > INT32_MAX || x.dtype < 0 || x.dtype > 2)
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
  const dim3 grid((unsigned)a.B), block(VER_BLOCK);
  const hipStream_t s = (hipStream_t)stream;
#define VERIFY(T)                                                        \
  do {                                                                   \
    if (a.draft)                                                         \
      hipLaunchKernelGGL((k_verify<T, true>), grid, block, 0, s, a);     \
    else                                                                 \
      hipLaunchKernelGGL((k_verify<T, false>), grid, block, 0, s, a);    \
  } while (0)
  if (x.dtype == 0)
    VERIFY(bf16_t);
  else if (x.dtype == 1)
    VERIFY(fp16_t);
  else
    VERIFY(float);
#undef VERIFY
  return launched("verify");
}

int geobpe_commit_draft(int device, void* stream, const geobpe_commit_args* p) {
  if (!p) return fail(GEOBPE_EARG, "no arguments");
  const geobpe_commit_args& x = *p;
  if (x.layers < 1 || x.layers > 65535 || x.seqs < 0 || x.nodes < 1 || x.nodes > DRAFT_MAX_NODES || x.kv_heads < 1 ||
      x.kv_heads > 65535 || x.head_bytes < 16 || x.head_bytes > 65536 || x.head_bytes % 16 || x.page_size < 1 ||
      x.pages < 1 || x.max_pages < 0 || x.pages > INT32_MAX || x.page_size > INT32_MAX ||
      x.max_pages > INT32_MAX / x.page_size || x.seqs > INT32_MAX / x.nodes)
    return fail(GEOBPE_EARG, "commit: sizes out of range");
  if (x.seqs == 0) return GEOBPE_OK;
  if (!x.d_k || !x.d_v || !x.d_k_cache || !x.d_v_cache || !x.d_lens || !x.d_path || !x.d_n || !x.d_lens_out ||
      (x.max_pages && !x.d_table))
    return fail(GEOBPE_EARG, "commit: null pointer");
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
  hipLaunchKernelGGL(k_commit, dim3((unsigned)(a.B * a.N), (unsigned)a.L), dim3(256), 0, (hipStream_t)stream, a);
  return launched("commit");
}

}  // extern "C"
