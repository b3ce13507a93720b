"""The decoding operators (geobpe.draft) against plain 64-bit implementations written here.

Attention's tolerance, from the number of bits: the 16-bit inputs are exact in 64 bits.  The kernel rounds the
weights w to the inputs' type before the product with v (half a step: eps / 2 relative each), the result once (eps / 2),
and computes scores and sums in 32 bits: a score of D products has an error of at most D 2^-24 sum |q k| scale, which
exp turns into a relative error of w; the tests' scores stay below |s| = 64 in sum |q k| scale <= 64 terms of it, so that
is below 2^-24 (D + 8) 64 < 2^-9.5 at D = 256, and below 2^-10 up to 128.  All of them are relative errors of the
weights, so |error| <= (eps / 2 + 2^-9.5) sum w |v| / sum w + eps / 2 |o|, twice over for the weights' sum:
bound = (eps + 2^-8) (sum w |v| / sum w) + eps / 2 |o|.  Verification and commit are exact."""
import ctypes
import os
import shutil
import struct
import subprocess

import numpy as np
import pytest
import torch

from conftest import REPO
from geobpe import draft

BF, FP = torch.bfloat16, torch.float16


# ---------------------------------------------------------------- plain implementations (64 bits, python loops)
def tree_paths(parents):
    """Per node the nodes from the root to it, None when it is absent."""
    out = []
    for i, p in enumerate(parents):
        if i == 0:
            out.append([0] if p == -1 else None)
        else:
            out.append(out[p] + [i] if 0 <= p < i and out[p] is not None else None)
    return out


def ref_attention(q, k_cache, v_cache, block_table, lens, k, v, parents, scale=None):
    """float64 result and the tolerance's sum w |v| / sum w."""
    q, kc, vc, k, v = (x.double().cpu().numpy() for x in (q, k_cache, v_cache, k, v))
    table, lens, parents = block_table.cpu().numpy(), lens.cpu().numpy(), parents.cpu().numpy()
    B, N, Hq, D = q.shape
    P, S, Hkv, _ = kc.shape
    M = table.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        paths = tree_paths((parents if parents.ndim == 1 else parents[b]).tolist())
        pos = np.arange(max(0, min(int(lens[b]), M * S)))
        ids = table[b][pos // S]
        bad = not 0 <= lens[b] <= M * S or (ids < 0).any() or (ids >= P).any()
        for i, path in enumerate(paths):
            if path is None:
                continue
            if bad:
                out[b, i] = np.nan
                continue
            for h in range(Hq):
                g = h // (Hq // Hkv)
                K = np.concatenate([kc[ids, pos % S, g], k[b, path, g]])
                V = np.concatenate([vc[ids, pos % S, g], v[b, path, g]])
                s = K @ q[b, i, h] * scale
                with np.errstate(invalid="ignore"):
                    w = np.exp(s - s.max())
                    out[b, i, h] = w @ V / w.sum()
                    mag[b, i, h] = w @ np.abs(V) / w.sum()
    return out, mag


def check_attention(got, ref, dtype):
    out, mag = ref
    eps = torch.finfo(dtype).eps
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(out))
    with np.errstate(invalid="ignore"):
        err = np.abs(got - out)
    tol = (eps + 2.0 ** -8) * mag + eps / 2 * np.abs(out) + 2.0 ** -24
    bad = ~(err <= tol) & ~np.isnan(out) & ~(np.isinf(out) & (out == got))
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), got[bad][:5], out[bad][:5])


def ref_verify(parents, ids, target, draft_, u, ranges=None, start=None):
    ids, u, parents = ids.cpu().numpy(), u.double().cpu().numpy(), parents.cpu().numpy()
    B, N, V = target.shape
    clean = lambda x: np.where(np.isfinite(x) & (x > 0), x, 0.0)  # noqa: E731
    target = clean(target.double().cpu().numpy())
    draft_ = None if draft_ is None else clean(draft_.double().cpu().numpy())
    n, paths, tokens = np.zeros(B, int), np.full((B, N), -1), np.full((B, N), -1)
    for b in range(B):
        present = tree_paths((parents if parents.ndim == 1 else parents[b]).tolist())
        par = (parents if parents.ndim == 1 else parents[b]).tolist()
        if present[0] is None:
            continue

        def row(rows, c, depth):
            keep = np.ones(V, bool)
            if ranges is not None:
                lo, hi = ranges[(int(start[b]) + depth) % len(ranges)].tolist()
                keep = (np.arange(V) >= lo) & (np.arange(V) < hi)
            return np.where(keep, rows[b, c], 0.0)

        path, toks = [0], []
        while True:
            c, d = path[-1], len(path) - 1
            r, Z, kept = row(target, c, d), 1.0, None
            for i in range(c + 1, N):
                if present[i] is None or par[i] != c:
                    continue
                x = int(ids[b, i])
                inside = 0 <= x < V
                if draft_ is None:
                    q = np.zeros(V)
                    qx = 1.0
                    if inside:
                        q[x] = 1.0
                else:
                    q = row(draft_, c, d)
                    qx = q[x] if inside else 0.0
                if u[b, i] * qx * Z < (r[x] if inside else 0.0):
                    kept = i
                    break
                r = np.maximum(r - Z * q, 0.0)
                Z = r.sum()
            if kept is None:
                break
            path.append(kept)
            toks.append(int(ids[b, kept]))
        if not r.sum() > 0:
            r = row(target, c, d)
        cum = np.cumsum(r)
        if cum[-1] > 0:
            hit = np.flatnonzero(cum > u[b, 0] * cum[-1])
            toks.append(int(hit[0]) if len(hit) else int(np.flatnonzero(r)[-1]))
        else:
            toks.append(-1)
        n[b] = len(path)
        paths[b, :len(path)] = path
        tokens[b, :len(toks)] = toks
    return n, paths, tokens


def check_verify(got, ref):
    for g, r, name in zip(got, ref, ("n", "path", "tokens")):
        assert np.array_equal(g.cpu().numpy(), r), (name, g.cpu().numpy().tolist(), r.tolist())


def make_parents(g, B, N, kind):
    if kind == "chain":
        p = np.tile(np.arange(-1, N - 1), (B, 1))
    elif kind == "flat":
        p = np.zeros((B, N), int)
    else:
        p = np.stack([[0] + [int(g.integers(0, i)) for i in range(1, N)] for _ in range(B)])
    p[:, 0] = -1
    return torch.tensor(p, dtype=torch.int32)


def make_attention(seed, B, N, lens, Hq, Hkv, D, S, dtype, kind="random", device="cpu", spare=0):
    """A case whose unused slots, spare pages and absent nodes hold NaN."""
    g = np.random.default_rng(seed)
    M = max(1, max(-(-max(x, 0) // S) for x in lens) + spare)
    P = B * M + 2
    t = lambda *s: torch.tensor(g.standard_normal(s), dtype=torch.float32).to(dtype)  # noqa: E731
    kc, vc = torch.full((P, S, Hkv, D), float("nan"), dtype=dtype), torch.full((P, S, Hkv, D), float("nan"), dtype=dtype)
    table = torch.tensor(g.permutation(P)[:B * M].reshape(B, M), dtype=torch.int32)
    for b, n in enumerate(lens):
        pos = torch.arange(max(n, 0))
        page = table[b].long()[pos // S]
        kc[page, pos % S], vc[page, pos % S] = t(len(pos), Hkv, D), t(len(pos), Hkv, D)
    case = dict(q=t(B, N, Hq, D), k_cache=kc, v_cache=vc, block_table=table,
                lens=torch.tensor(lens, dtype=torch.int32), k=t(B, N, Hkv, D), v=t(B, N, Hkv, D),
                parents=make_parents(g, B, N, kind))
    return {k: v.to(device) for k, v in case.items()}


def make_verify(seed, B, N, V, dtype, kind, drafted=True, sharp=2.0, ranges=None, device="cpu"):
    g = np.random.default_rng(seed)
    parents = make_parents(g, B, N, kind)
    start = torch.tensor(g.integers(0, 50, B), dtype=torch.int32) if ranges is not None else None
    a = g.standard_normal((B, N, V)) * sharp
    near = a + g.standard_normal((B, N, V)) * 0.7
    if ranges is not None:
        for b in range(B):
            for i, path in enumerate(tree_paths(parents[b].tolist())):
                lo, hi = ranges[(int(start[b]) + len(path) - 1) % len(ranges)].tolist()
                out = np.ones(V, bool)
                out[lo:hi] = False
                a[b, i, out] = near[b, i, out] = -np.inf
    soft = lambda x: torch.softmax(torch.tensor(x, dtype=torch.float32), -1).to(dtype)  # noqa: E731
    p, q = soft(a), soft(near)
    ids = torch.zeros(B, N, dtype=torch.int64)
    for b in range(B):
        for i in range(1, N):
            w = q[b, parents[b, i]].double().numpy()
            ids[b, i] = int(g.choice(V, p=w / w.sum()))
    out = dict(parents=parents, ids=ids, target=p, draft=q if drafted else None,
               u=torch.tensor(g.random((B, N)), dtype=torch.float32), ranges=ranges, start=start)
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in out.items()}


def on(case, device="cuda"):
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in case.items()}


def make_commit(seed, L, B, N, lens, Hkv, D, S, dtype):
    g = np.random.default_rng(seed)
    M = max(-(-(x + N) // S) for x in lens)
    P = B * M + 1
    r = lambda *s: torch.tensor(g.standard_normal(s), dtype=torch.float32).to(dtype)  # noqa: E731
    n = g.integers(0, N + 1, B)
    path = np.full((B, N), -1)
    for b in range(B):
        path[b, :n[b]] = np.sort(g.choice(N, n[b], replace=False))
    return dict(k_cache=r(L, P, S, Hkv, D), v_cache=r(L, P, S, Hkv, D),
                block_table=torch.tensor(g.permutation(P)[:B * M].reshape(B, M), dtype=torch.int32),
                lens=torch.tensor(lens, dtype=torch.int32), k=r(L, B, N, Hkv, D), v=r(L, B, N, Hkv, D),
                path=torch.tensor(path, dtype=torch.int32), n=torch.tensor(n, dtype=torch.int32))


def ref_commit(c):
    kc, vc = c["k_cache"].clone(), c["v_cache"].clone()
    P, S = kc.shape[1:3]
    B, M = c["block_table"].shape
    N = c["path"].shape[1]
    lens = c["lens"].tolist()
    for b in range(B):
        m, n, ok = lens[b], int(c["n"][b]), lens[b] >= 0 and int(c["n"][b]) <= N
        for t in range(min(n, N)):
            node, at = int(c["path"][b, t]), m + t
            id_ = int(c["block_table"][b, at // S]) if 0 <= at < M * S else -1
            if m < 0 or not 0 <= node < N or not 0 <= id_ < P:
                ok = False
                continue
            kc[:, id_, at % S], vc[:, id_, at % S] = c["k"][:, b, node], c["v"][:, b, node]
        lens[b] = m + max(n, 0) if ok else -1
    return kc, vc, torch.tensor(lens, dtype=torch.int32)


# ---------------------------------------------------------------- CPU: refusals, addresses
def attend(c):
    return draft.tree_attention(c["q"], c["k_cache"], c["v_cache"], c["block_table"], c["lens"], c["k"], c["v"],
                                c["parents"], c.get("scale"))


def refuse(f, c, exc, match, **change):
    with pytest.raises(exc, match=match):
        f({**c, **change})


def test_attention_refusals():
    c = make_attention(0, 2, 3, [5, 9], 4, 2, 16, 4, BF)
    refuse(attend, c, ValueError, "HIP device only")
    refuse(attend, c, TypeError, "torch tensor", q=None)
    refuse(attend, c, TypeError, "torch tensor", k_cache=1)
    refuse(attend, c, TypeError, "q is of type Float", q=c["q"].float())
    refuse(attend, c, TypeError, "k is of type Half", k=c["k"].half())
    refuse(attend, c, TypeError, "v_cache", v_cache=c["v_cache"].half())
    refuse(attend, c, TypeError, "lens", lens=c["lens"].long())
    refuse(attend, c, TypeError, "block_table", block_table=c["block_table"].long())
    refuse(attend, c, TypeError, "parents", parents=c["parents"].long())
    refuse(attend, c, ValueError, "parents", parents=c["parents"][:, :2])
    refuse(attend, c, ValueError, "parents", parents=c["parents"].t().contiguous().t())
    refuse(attend, c, ValueError, "block_table", block_table=c["block_table"][:1])
    refuse(attend, c, ValueError, "v_cache", v_cache=c["v_cache"][:3])
    refuse(attend, c, ValueError, "sequences", lens=c["lens"][:1], block_table=c["block_table"][:1])
    refuse(attend, c, ValueError, "key heads", q=c["q"][:, :, :3])
    refuse(attend, c, ValueError, "key heads", q=c["q"][:, :, :0])
    refuse(attend, c, ValueError, "k:", k=c["k"][:, :2])
    refuse(attend, c, ValueError, "16-byte aligned", q=c["q"].transpose(2, 3).contiguous().transpose(2, 3))
    odd = torch.zeros(c["q"].numel() + 1, dtype=BF)[1:].view(c["q"].shape)
    refuse(attend, c, ValueError, "16-byte aligned", q=odd)
    wide = torch.zeros(2, 3, 4, 20, dtype=BF)[..., :16]
    refuse(attend, c, ValueError, "16-byte aligned", q=wide)
    refuse(attend, c, ValueError, "no backward", q=c["q"].clone().requires_grad_())
    with torch.no_grad():
        refuse(attend, c, ValueError, "HIP device only", q=c["q"].clone().requires_grad_())
    big = make_attention(0, 1, 129, [5], 2, 2, 16, 4, BF)
    refuse(attend, big, ValueError, "1 to 128 nodes")
    d12 = make_attention(0, 1, 1, [5], 2, 2, 12, 4, BF)
    refuse(attend, d12, ValueError, "multiple of 8")
    d264 = make_attention(0, 1, 1, [5], 2, 2, 264, 4, BF)
    refuse(attend, d264, ValueError, "multiple of 8")
    refuse(attend, c, ValueError, "more than",
           block_table=torch.zeros(2, 1, dtype=torch.int32).expand(2, 1 << 30))


def verify(c):
    return draft.verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"], c["ranges"], c["start"])


def test_verify_refusals():
    c = make_verify(0, 2, 4, 20, torch.float32, "random")
    refuse(verify, c, ValueError, "HIP device only")
    refuse(verify, c, TypeError, "torch tensor", target=[1])
    refuse(verify, c, TypeError, "Double", target=c["target"].double())
    refuse(verify, c, TypeError, "draft", draft=c["draft"].half())
    refuse(verify, c, ValueError, "draft", draft=c["draft"][:, :3])
    refuse(verify, c, TypeError, "ids", ids=c["ids"].float())
    refuse(verify, c, ValueError, "ids", ids=c["ids"][:, :3])
    refuse(verify, c, TypeError, "u is", u=c["u"].double())
    refuse(verify, c, ValueError, "belong together", ranges=torch.zeros(1, 2, dtype=torch.int32))
    refuse(verify, c, ValueError, "not empty", ranges=torch.zeros(0, 2, dtype=torch.int32),
           start=torch.zeros(2, dtype=torch.int32))
    refuse(verify, c, ValueError, "last dimension", target=c["target"].transpose(1, 2).contiguous().transpose(1, 2))
    refuse(verify, c, ValueError, "last dimension", u=c["u"].t().contiguous().t())
    refuse(verify, c, ValueError, "no backward", target=c["target"].clone().requires_grad_())
    wide = torch.zeros(1, 1, 1).expand(1, 1, (1 << 22) + 1)
    one = torch.zeros(1, 1, dtype=torch.int32)
    refuse(verify, c, ValueError, "vocabulary", target=wide, draft=wide, ids=one, parents=one, u=one.float())


def commit(c):
    return draft.commit(c["k_cache"], c["v_cache"], c["block_table"], c["lens"], c["k"], c["v"], c["path"], c["n"])


def test_commit_refusals():
    c = make_commit(0, 2, 3, 4, [0, 5, 7], 2, 16, 4, BF)
    refuse(commit, c, ValueError, "HIP device only")
    refuse(commit, c, TypeError, "torch tensor", k_cache=None)
    refuse(commit, c, ValueError, "v_cache", v_cache=c["v_cache"][:1])
    refuse(commit, c, TypeError, "k is", k=c["k"].half())
    refuse(commit, c, ValueError, "k:", k=c["k"][0])
    refuse(commit, c, ValueError, "k_cache", k_cache=c["k_cache"][0, 0])
    refuse(commit, c, TypeError, "path", path=c["path"].long())
    refuse(commit, c, ValueError, "n:", n=c["n"][:2])
    refuse(commit, c, ValueError, "expanded", k_cache=c["k_cache"][:1].expand(2, -1, -1, -1, -1))
    both = torch.zeros(2, 20, 4, 2, 16, dtype=BF)
    P = c["k_cache"].shape[1]
    refuse(commit, c, ValueError, "cache's own memory", k_cache=both[:, :P], k=both[:, P - 1:P + 2])
    refuse(commit, c, ValueError, "cache's own memory", v_cache=both[:, :P], v=both[:, :3])
    refuse(commit, c, ValueError, "v_cache is k_cache", v_cache=c["k_cache"])
    refuse(commit, c, ValueError, "conjugates", **{x: c[x].to(torch.complex64).conj() if x == "k" else c[x].to(torch.complex64)
                                                   for x in ("k", "v", "k_cache", "v_cache")})
    refuse(commit, c, ValueError, "multiple of 16", **{k: c[k][..., :4].contiguous() for k in ("k", "v", "k_cache", "v_cache")})


_ATTEND = struct.Struct("35qd")  # include/geobpe.h geobpe_attend_args
_VERIFY = struct.Struct("23q")   # geobpe_verify_args
_COMMIT = struct.Struct("35q")   # geobpe_commit_args


def test_c_entries_refuse_without_a_device():
    """The C entries check sizes, pointers and alignment before they touch a device."""
    from geobpe import _native
    L = _native.lib()
    assert L.geobpe_tree_attention(0, None, None, None, 0) == _native.E_ARG
    ok = dict(ptr=[256] * 9, st=[64, 64, 64] * 5, rest=[1, 0], sizes=[1, 2, 4, 2, 64, 16, 3, 2, 0])
    pack = lambda d: _ATTEND.pack(*d["ptr"], *d["st"], *d["rest"], *d["sizes"], 1.0)  # noqa: E731
    for i, bad in ((0, -1), (1, 0), (1, 129), (2, 3), (3, 0), (4, 60), (4, 264), (5, 0), (6, 0), (7, 1 << 31), (8, 2)):
        d = {**ok, "sizes": [bad if j == i else x for j, x in enumerate(ok["sizes"])]}
        assert L.geobpe_tree_attention(0, None, pack(d), 256, 1 << 40) == _native.E_ARG, (i, bad)
        assert b"sizes" in L.geobpe_draft_error()
        assert L.geobpe_tree_attention_work(pack(d)) == -1
    long = {**ok, "sizes": [1, 2, 4, 2, 64, 16, 3, 1000, 0]}
    need = L.geobpe_tree_attention_work(pack(long))
    assert need > 0 and L.geobpe_tree_attention_work(pack({**ok, "sizes": [0, *ok["sizes"][1:]]})) == 0
    assert L.geobpe_tree_attention(0, None, pack(long), 256, need - 1) == _native.E_ARG
    assert b"work space" in L.geobpe_draft_error()
    assert L.geobpe_tree_attention(0, None, pack(long), None, need) == _native.E_ARG
    assert L.geobpe_tree_attention(0, None, pack(long), 264, need) == _native.E_ARG
    for i in range(9):
        d = {**ok, "ptr": [0 if j == i else x for j, x in enumerate(ok["ptr"])]}
        assert L.geobpe_tree_attention(0, None, pack(d), 256, 1 << 40) == _native.E_ARG and b"null" in L.geobpe_draft_error()
    d = {**ok, "ptr": [256 + 2, *ok["ptr"][1:]]}
    assert L.geobpe_tree_attention(0, None, pack(d), 256, 1 << 40) == _native.E_ARG and b"aligned" in L.geobpe_draft_error()
    d = {**ok, "st": [65, *ok["st"][1:]]}
    assert L.geobpe_tree_attention(0, None, pack(d), 256, 1 << 40) == _native.E_ARG and b"aligned" in L.geobpe_draft_error()
    d = {**ok, "sizes": [0, *ok["sizes"][1:]]}
    assert L.geobpe_tree_attention(0, None, pack(d), 256, 1 << 40) == 0  # no sequences: nothing to do
    assert L.geobpe_verify_draft(0, None, None) == _native.E_ARG
    v = [256] * 10 + [8, 8, 8, 8, 0, 4, 4]
    for i, bad in ((0, -1), (1, 0), (1, 129), (2, 0), (2, (1 << 22) + 1), (3, -1), (5, 3)):
        sizes = [bad if j == i else x for j, x in enumerate([2, 4, 20, 0, 0, 2])]
        assert L.geobpe_verify_draft(0, None, _VERIFY.pack(*v, *sizes)) == _native.E_ARG, (i, bad)
    assert L.geobpe_verify_draft(0, None, _VERIFY.pack(*[0, *v[1:]], 2, 4, 20, 0, 0, 2)) == _native.E_ARG
    assert L.geobpe_commit_draft(0, None, None) == _native.E_ARG
    k = [256] * 9 + [64] * 16 + [2, 4]
    for i, bad in ((0, 0), (1, -1), (2, 0), (3, 0), (4, 24), (5, 0), (6, 0), (7, -1)):
        sizes = [bad if j == i else x for j, x in enumerate([1, 2, 4, 2, 128, 16, 3, 2])]
        assert L.geobpe_commit_draft(0, None, _COMMIT.pack(*k, *sizes)) == _native.E_ARG, (i, bad)
    assert L.geobpe_commit_draft(0, None, _COMMIT.pack(*k[:8], 512, 8, *k[10:], 1, 2, 4, 2, 128, 16, 3, 2)) == _native.E_ARG
    assert b"aligned" in L.geobpe_draft_error()
    assert L.geobpe_commit_draft(0, None, _COMMIT.pack(*k, 1, 2, 4, 2, 128, 16, 3, 2)) == _native.E_ARG
    assert b"new lengths" in L.geobpe_draft_error()  # (they are the old ones' memory here)


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """csrc/draft.h built for the CPU: the kernels' own tree walk and page addresses."""
    d = tmp_path_factory.mktemp("draft_host")
    src = d / "h.cpp"
    src.write_text("""
#include <stdint.h>
#define __device__
static inline uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a * b) >> 32); }
#include "draft.h"
using namespace gb;
extern "C" int page(const int32_t* row, int M, int P, int S, int x, int* slot) {
  Pages t = {row, page_div(S), P, M};
  return find_page(t, x, *slot);
}
extern "C" int split_ok(int d, int x) {
  int k, s;
  page_split(page_div(d), x, k, s);
  return k == x / d && s == x % d;
}
extern "C" int paths(const int* par, int N, uint32_t* w, int* here) {  // all nodes at once, as the kernels do it
  DraftNode now[DRAFT_MAX_NODES], next[DRAFT_MAX_NODES];
  for (int i = 0; i < N; i++) now[i] = draft_node(i, par[i]);
  int turns = 0;
  for (bool more = true; more;) {
    more = false;
    for (int i = 0; i < N; i++) {
      next[i] = now[i];
      if (now[i].up >= 0) {
        draft_climb(next[i], now[now[i].up]);
        more = true;
      }
    }
    for (int i = 0; i < N; i++) now[i] = next[i];
    turns += more;
  }
  for (int i = 0; i < N; i++) {
    here[i] = now[i].up == -1;
    for (int k = 0; k < 4; k++) w[4 * i + k] = now[i].w[k];
  }
  return turns;
}
""")
    so = d / "h.so"
    subprocess.run([shutil.which("g++"), "-O1", "-shared", "-fPIC", "-Wno-unknown-pragmas", "-fsanitize=undefined",
                    "-fno-sanitize-recover", f"-I{os.path.join(REPO, 'pt-bpe_amd', 'csrc')}", str(src), "-o", str(so)],
                   check=True)
    return ctypes.CDLL(str(so))


def test_page_addresses(host):
    g = np.random.default_rng(0)
    big = 2 ** 31 - 1
    for d in [1, 2, 3, 5, 7, 16, 24, 48, 1000, 65537, 2 ** 30, 2 ** 30 + 1, big - 1, big]:
        xs = [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, big // d * d - 1, big // d * d, big - 1, big]
        for x in [v for v in xs if 0 <= v <= big] + g.integers(0, big, 200, endpoint=True).tolist():
            assert host.split_ok(d, int(x)), (d, x)


def test_bad_pages_are_found(host):
    slot = ctypes.c_int()
    row = np.array([3, -1, 7, 8, 2 ** 31 - 1, -2 ** 31], dtype=np.int32)
    p = row.ctypes.data_as(ctypes.c_void_p)
    got = [host.page(p, 6, 8, 4, x, ctypes.byref(slot)) for x in range(0, 24, 4)]
    assert got == [3, -1, 7, -1, -1, -1]
    assert host.page(p, 6, 8, 4, 2 * 4 + 3, ctypes.byref(slot)) == 7 and slot.value == 3
    assert host.page(p, 2, 8, 4, 8, ctypes.byref(slot)) == -1  # past the table: not read
    assert host.page(None, 0, 8, 4, 0, ctypes.byref(slot)) == -1
    assert host.page(p, 6, 8, 4, -1, ctypes.byref(slot)) == -1


def test_tree_walk(host):
    g = np.random.default_rng(1)
    for trial in range(50):
        N = int(g.integers(1, 129))
        par = g.integers(-3, N + 2, N).astype(np.int32)
        if trial % 3:
            par = np.array([-1] + [int(g.integers(0, i)) for i in range(1, N)], dtype=np.int32)
        if trial % 4 == 0:
            par[0] = -1
        if trial == 0:
            par = np.arange(-1, 127, dtype=np.int32)
            N = 128
        w, here = (ctypes.c_uint32 * (4 * N))(), (ctypes.c_int * N)()
        assert host.paths(par.ctypes.data_as(ctypes.c_void_p), N, w, here) <= 7
        for i, want in enumerate(tree_paths(par.tolist())):
            got = [j for j in range(128) if w[4 * i + j // 32] >> j % 32 & 1]
            assert bool(here[i]) == (want is not None) and (want is None or got == want)


# ---------------------------------------------------------------- GPU
ATTEND = [
    # B, N, lens, Hq, Hkv, D, S, tree
    (1, 1, [0], 1, 1, 8, 1, "chain"),
    (1, 1, [1], 2, 1, 16, 16, "chain"),
    (2, 1, [31, 33], 8, 8, 64, 16, "chain"),
    (3, 5, [0, 1, 300], 4, 4, 80, 24, "chain"),
    (2, 3, [64, 128], 16, 2, 128, 32, "random"),
    (2, 17, [255, 257], 6, 2, 96, 7, "random"),
    (1, 64, [1000], 8, 2, 128, 64, "random"),
    (1, 128, [129], 4, 1, 64, 16, "random"),
    (2, 127, [63, 500], 7, 1, 32, 3, "flat"),
    (1, 33, [2049], 2, 2, 256, 128, "random"),
    (4, 9, [5, 0, 77, 641], 14, 2, 120, 48, "chain"),
    (1, 2, [5000], 4, 1, 136, 16, "chain"),
    (70, 4, [i * 3 for i in range(70)], 4, 2, 64, 16, "random"),
    (5, 3, [10, 900, 33, 0, 2000], 12, 1, 200, 16, "chain"),
    (40, 5, [(i * 37) % 300 for i in range(40)], 16, 4, 64, 16, "chain"),
    (30, 40, [(i * 97) % 2500 for i in range(30)], 16, 8, 64, 32, "random"),
    # rows for 256-row workgroups: whole and cut heads, several row tiles, the head's last pieces missing
    (2, 96, [70, 1500], 8, 2, 96, 16, "random"),
    (1, 128, [3001], 6, 3, 72, 5, "random"),
    (3, 128, [0, 1, 64], 16, 4, 128, 16, "random"),
    (1, 37, [257], 32, 2, 128, 128, "chain"),
    (2, 128, [40, 700], 2, 1, 256, 32, "random"),
    (1, 50, [65], 8, 1, 8, 1, "flat"),
    # eight waves over one part: 17 to 32 tiles
    (1, 3, [700], 4, 4, 64, 16, "chain"),
    (2, 7, [601, 540], 8, 2, 128, 16, "random"),
    (3, 2, [960, 0, 33], 4, 2, 40, 24, "chain"),
    # many tiles: 256 rows of 104, 64 rows of heads up to 32
    (20, 70, [(i * 211) % 1100 + 300 for i in range(20)], 20, 5, 104, 64, "random"),
    (26, 40, [(i * 211) % 1100 + 300 for i in range(26)], 7, 7, 24, 64, "random"),
    # 8 waves over few rows, and heads past 128 with one and more row tiles
    (33, 2, [(i * 71) % 1200 for i in range(33)], 8, 4, 104, 16, "chain"),
    (2, 16, [511, 513], 1, 1, 248, 64, "random"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape", ATTEND, ids=lambda s: "x".join(map(str, (s[0], s[1], max(s[2]), *s[3:]))))
def test_attention(shape, dtype):
    B, N, lens, Hq, Hkv, D, S, kind = shape
    c = make_attention(1, B, N, lens, Hq, Hkv, D, S, dtype, kind)
    check_attention(attend(on(c)), ref_attention(**c), dtype)


@pytest.mark.gpu
def test_attention_long_context():
    """One sequence of 70 000 positions: the work is split and joined."""
    c = make_attention(2, 1, 6, [70001], 4, 1, 64, 64, BF)
    check_attention(attend(on(c)), ref_attention(**c), BF)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 40])
def test_attention_absent_nodes_and_sequences(N):
    c = make_attention(3, 4, N, [40, 0, 7, 100], 8, 2, 64, 16, BF)
    c["parents"][0, 2] = -1           # absent, and what hangs on it
    c["parents"][1, 0] = -2           # the whole sequence
    c["parents"][2, 3] = 3            # not before itself
    c["parents"][3, 1:] = -5          # the root alone
    paths = [tree_paths(p) for p in c["parents"].tolist()]
    for b, ps in enumerate(paths):    # what absent nodes hold must not matter
        for i, x in enumerate(ps):
            if x is None:
                c["k"][b, i] = float("nan")
                c["v"][b, i] = float("inf")
                c["q"][b, i] = float("nan")
    got = attend(on(c))
    check_attention(got, ref_attention(**c), BF)
    for b, ps in enumerate(paths):
        for i, x in enumerate(ps):
            if x is None:
                assert not got[b, i].any()


@pytest.mark.gpu
@pytest.mark.parametrize("N,lens", [(6, [70, 3]), (40, [70, 600])])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_one_nodes_values_stay_on_its_path(N, lens, value):
    """A present node whose value is not finite reaches the rows below it and no other."""
    c = make_attention(4, 2, N, lens, 4, 2, 64, 16, FP)
    c["v"][0, 3, 1, 5] = value
    c["v"][1, N - 1, 0, :] = value
    check_attention(attend(on(c)), ref_attention(**c), FP)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [4, 40])
def test_attention_bad_pages_and_lengths(N):
    c = make_attention(5, 6, N, [40, 40, 40, 40, 40, 40], 4, 2, 64, 16, BF)
    c["block_table"][1, 2] = -1
    c["block_table"][2, 0] = c["k_cache"].shape[0]
    c["lens"][3] = -1
    c["lens"][4] = 49                 # three pages of 16
    c["lens"][5] = 2 ** 31 - 1
    c["parents"][4, 2] = -1           # (still 0, not NaN)
    check_attention(attend(on(c)), ref_attention(**c), BF)
    c["lens"][1] = 32                 # the bad page is not needed
    got = attend(on(c))
    assert torch.isfinite(got[1]).all() and not torch.isfinite(got[2]).any()


@pytest.mark.gpu
def test_attention_extreme_scores():
    """Scores of +-1e4 and more: the running maximum carries the sums; a whole prefix far below the tree."""
    c = make_attention(6, 3, 5, [200, 200, 200], 4, 2, 64, 16, BF)
    c["q"][0] *= 100
    c["k_cache"][c["block_table"][1].long()] = torch.where(
        torch.isnan(c["k_cache"][c["block_table"][1].long()]), float("nan"), -1.0).to(BF)
    c["q"][1] = c["q"][1].abs() * 30
    c["k"][2] = 0
    ref = ref_attention(**c)
    got = attend(on(c))
    assert torch.isfinite(got).all()
    check_attention(got[1:], (ref[0][1:], ref[1][1:]), BF)
    # sequence 0's scores reach 1e3: 32-bit sums are off by up to 2^-24 (D + 8) 1e3 there, 4e-3 of a weight
    err = (got[0].double().cpu().numpy() - ref[0][0])
    assert (np.abs(err) <= (2 ** -6) * ref[1][0] + 2 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 70])
def test_attention_strides_and_shared_tree(N):
    """Heads before slots, a fused qkv tensor, one tree for the batch, a table wider than needed."""
    c = make_attention(7, 3, N, [50, 90, 10], 4, 2, 64, 16, BF, spare=2)
    ref = make_attention(7, 3, N, [50, 90, 10], 4, 2, 64, 16, BF, spare=2)
    ref["parents"] = ref["parents"][1].contiguous()
    want = ref_attention(**ref)
    d = on(c)
    qkv = torch.zeros(3, N, 8 + 2 + 2, 64, dtype=BF, device="cuda")
    qkv[:, :, :4], qkv[:, :, 8:10], qkv[:, :, 10:] = d["q"], d["k"], d["v"]
    d["q"], d["k"], d["v"] = qkv[:, :, :4], qkv[:, :, 8:10], qkv[:, :, 10:]
    d["k_cache"] = d["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack([d["v_cache"], d["v_cache"]], 1)
    d["v_cache"] = both[:, 1]
    d["parents"] = d["parents"][1].contiguous()
    wide = torch.full((3, d["block_table"].shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, :d["block_table"].shape[1]] = d["block_table"]
    d["block_table"] = wide
    check_attention(attend(d), want, BF)
    d["scale"] = 0.3
    check_attention(attend(d), ref_attention(**ref, scale=0.3), BF)
    # queries shared by the batch (stride 0)
    d["q"] = qkv[:1, :, :4].expand(3, -1, -1, -1)
    ref["q"] = ref["q"][:1].expand(3, -1, -1, -1)
    check_attention(attend(d), ref_attention(**ref, scale=0.3), BF)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 40])
def test_attention_far_offsets(N):
    """Pages past 2^31 elements of the cache."""
    S, Hkv, D = 64, 8, 128
    P = (1 << 31) // (S * Hkv * D) + 3
    kc = torch.zeros(P, S, Hkv, D, dtype=BF, device="cuda")
    c = make_attention(8, 1, N, [130], 8, 8, D, S, BF)
    far = torch.tensor([[P - 1, 0, P - 2]], dtype=torch.int32)
    for b in range(3):
        kc[far[0, b].item()] = c["k_cache"][c["block_table"][0, b].item()].cuda()
    vc = torch.zeros_like(kc)
    for b in range(3):
        vc[far[0, b].item()] = c["v_cache"][c["block_table"][0, b].item()].cuda()
    want = ref_attention(**c)
    d = on({**c, "block_table": far})
    d["k_cache"], d["v_cache"] = kc, vc
    check_attention(attend(d), want, BF)


@pytest.mark.gpu
def test_attention_no_sequences():
    c = make_attention(0, 2, 3, [5, 9], 4, 2, 16, 4, BF, device="cuda")
    e = {k: v[:0] if k not in ("k_cache", "v_cache") else v for k, v in c.items()}
    assert attend(e).shape == (0, 3, 4, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("N,Hq,D", [(30, 12, 128), (70, 4, 136), (12, 3, 256), (2, 4, 96), (70, 4, 96), (40, 2, 32), (33, 1, 32)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_values_not_finite_by_shape(N, Hq, D, value):
    """The same where a workgroup has 256 rows, where heads are cut, and where there are few rows."""
    c = make_attention(9, 3, N, [200, 0, 33], Hq, 1, D, 16, BF)
    c["v"][0, N // 2, 0, D - 1] = value
    c["v"][1, 0, 0, 0] = value            # the root: every row
    c["v"][2, N - 1, 0, :] = value
    check_attention(attend(on(c)), ref_attention(**c), BF)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,Hq,Hkv,D", [(20, 70, 20, 5, 104), (26, 40, 7, 7, 24)])
def test_attention_values_not_finite_among_many_tiles(B, N, Hq, Hkv, D):
    c = make_attention(18, B, N, [(i * 211) % 1100 + 300 for i in range(B)], Hq, Hkv, D, 64, FP)
    c["v"][0, N // 2, Hkv - 1, D - 1] = float("nan")
    c["v"][1, 0, 0, 0] = -float("inf")
    c["v"][B - 1, N - 1, :, :] = float("inf")
    check_attention(attend(on(c)), ref_attention(**c), FP)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [4, 40])
def test_attention_committed_values_not_finite(N):
    """Infinity at the last committed position stays infinity: what fills its tile up does not make it NaN."""
    c = make_attention(10, 4, N, [1, 31, 65, 640], 4, 2, 64, 16, BF)
    for b, n in enumerate(c["lens"].tolist()):
        page = c["block_table"][b, (n - 1) // 16].item()
        c["v_cache"][page, (n - 1) % 16, 1, 3] = float("inf") if b % 2 else -float("inf")
    check_attention(attend(on(c)), ref_attention(**c), BF)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 40])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_keys_not_finite(N, value):
    """A key that is not finite: scores of +-infinity and NaN, in the cache and in the tree, for its rows alone."""
    c = make_attention(11, 3, N, [100, 50, 0], 2, 2, 64, 16, BF)
    c["k_cache"][c["block_table"][0, 2].item(), 5, 0, 7] = value
    c["k"][1, 2, 1, 0] = value
    c["k"][2, :, 0, 1] = value            # no other key: the row has no weights
    ref = ref_attention(**c)
    got = attend(on(c))
    assert np.isnan(ref[0]).any() and np.isfinite(ref[0]).any()
    check_attention(got, ref, BF)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 40])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-3])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_scales(N, scale, dtype):
    """Zero (the mean of the values) and negative ones, with a value that is not finite among them."""
    c = make_attention(12, 2, N, [90, 600], 4, 2, 64, 16, dtype)
    c["v"][1, N - 1, 0, 3] = float("inf")
    c["scale"] = scale
    check_attention(attend(on(c)), ref_attention(**c), dtype)


@pytest.mark.gpu
def test_attention_without_pages():
    """A table without entries, a cache of one slot: the tree alone, and a length that cannot be."""
    c = make_attention(13, 3, 4, [0, 0, 0], 2, 1, 64, 1, BF)
    c["block_table"] = torch.zeros(3, 0, dtype=torch.int32)
    c["lens"][2] = 1
    check_attention(attend(on(c)), ref_attention(**c), BF)


@pytest.mark.gpu
@pytest.mark.parametrize("N,Hq,D", [(2, 4, 64), (24, 8, 128), (70, 8, 128)])
def test_attention_graphs_and_streams(N, Hq, D):
    """Sequences that are cut (work space): two captured graphs replayed in turn with eager calls between, lengths that
    change between replays, and two streams at once."""
    cases = [make_attention(14 + i, 2, N, [5000, 3], Hq, 2, D, 64, BF) for i in range(2)]
    dev = [on(c) for c in cases]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for d in dev:
            attend(d)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for d in dev:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(attend(d))
        graphs.append(g)
    for lens in ([5000, 3], [513, 0], [1, 3]):
        for c, d in zip(cases, dev):
            c["lens"] = torch.tensor(lens, dtype=torch.int32)
            d["lens"].copy_(c["lens"])
        want = [ref_attention(**c) for c in cases]
        for i in (0, 1, 0):
            outs[i].fill_(7)
            graphs[i].replay()
            check_attention(outs[i], want[i], BF)
            check_attention(attend(dev[1 - i]), want[1 - i], BF)
        streams = [torch.cuda.Stream() for _ in range(2)]
        both = []
        for st, d in zip(streams, dev):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                both.append([attend(d) for _ in range(3)])
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for got, w in zip(both, want):
            for x in got:
                check_attention(x, w, BF)
                assert torch.equal(x, got[0])  # (the joins have one order)


VERIFY = [
    # B, N, V, tree, drafted
    (1, 1, 1, "chain", True),
    (2, 1, 7, "chain", False),
    (3, 2, 5, "chain", True),
    (16, 5, 91, "chain", True),
    (16, 5, 1091, "chain", False),
    (12, 12, 33, "flat", True),
    (12, 12, 33, "flat", False),
    (9, 40, 300, "random", True),
    (9, 40, 300, "random", False),
    (3, 128, 40, "random", True),
    (2, 128, 40, "flat", False),
    (4, 6, 4097, "random", True),
    (3, 5, 20001, "random", True),
    (2, 4, 65537, "flat", False),
    (2, 4, 65537, "flat", True),
    (1, 3, 8192, "chain", True),
    (1, 3, 8193, "flat", False),
    (1, 3, 700001, "flat", True),
    (1, 3, 700001, "flat", False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, FP])
@pytest.mark.parametrize("shape", VERIFY, ids=lambda s: "x".join(map(str, s)))
def test_verify(shape, dtype):
    B, N, V, kind, drafted = shape
    c = make_verify(11, B, N, V, dtype, kind, drafted)
    check_verify(verify(on(c)), ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"]))


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("classes", [1, 3, 4])
def test_verify_ranges(classes, drafted):
    V = 300
    ranges = torch.tensor([[0, 285], [290, 295], [295, 300], [285, 290]][:classes], dtype=torch.int32)
    c = make_verify(12, 24, 20, V, torch.float32, "random", drafted, ranges=ranges)
    want = ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"], ranges, c["start"])
    check_verify(verify(on(c)), want)
    d = on(c)  # what lies outside a range is not read
    d["target"] = torch.where(d["target"] > 0, d["target"], float("nan"))
    check_verify(verify(d), want)
    for bad in ([-5, 10 ** 6], [200, 100], [400, 500]):  # past the row, empty, behind it
        r = torch.tensor([bad] * classes, dtype=torch.int32)
        check_verify(verify(on({**c, "ranges": r})),
                     ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"], r, c["start"]))


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
def test_verify_edges(drafted):
    """Numbers at both ends, rows without mass, entries that are no probabilities, ids outside the vocabulary,
    the same id twice, equal rows, absent nodes."""
    c = make_verify(13, 12, 10, 50, torch.float32, "random", drafted)
    c["u"][0] = 0
    c["u"][1] = float(np.nextafter(np.float32(1), np.float32(0)))
    c["target"][2] = 0
    c["target"][3, :, ::2] = float("nan")
    c["target"][3, :, 1] = float("inf")
    c["target"][3, :, 3] = -1
    c["ids"][4, 1:6] = torch.tensor([-1, 50, 2 ** 40, -2 ** 40, 49])
    c["parents"][5] = torch.tensor([-1] + [0] * 9)
    c["ids"][5] = 7
    c["parents"][7, 0] = 0
    c["parents"][8, 1] = -1
    c["parents"][9, 4] = 4
    if drafted:
        c["draft"][6] = c["target"][6]
        c["draft"][10] = 0
        c["draft"][11] = 1e30
    want = ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"])
    check_verify(verify(on(c)), want)
    assert want[0][7] == 0 and (want[1][7] == -1).all()
    d = on(c)  # int32 ids, strided rows, a shared tree
    d["ids"] = c["ids"].clamp(-1, 50).int().cuda()
    check_verify(verify(d), want)
    wide = torch.full((12, 10, 61), 0.5, device="cuda")
    wide[..., 3:53] = d["target"]
    d["target"] = wide[..., 3:53]
    check_verify(verify(d), want)
    d["parents"] = c["parents"][0].contiguous().cuda()
    check_verify(verify(d), ref_verify(c["parents"][0], c["ids"], c["target"], c["draft"], c["u"]))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 300, 20000])
def test_verify_drafts_that_take_nearly_all(V):
    """Drafts without probabilities that hold nearly the whole row: what is left after them, parts of a sum among it, is
    summed anew."""
    B, N = 8, 20
    c = make_verify(15, B, N, V, torch.float32, "flat", False)
    g = np.random.default_rng(15)
    rest = g.random((B, N, V)).astype(np.float32) * np.float32(2 ** -40)
    c["target"] = torch.tensor(rest)
    for b in range(B):
        x = g.choice(V, N - 1, replace=False)
        c["ids"][b, 1:] = torch.tensor(x)
        c["target"][b, :, x] = torch.tensor(g.random(N - 1).astype(np.float32))
        c["u"][b, 1:] = 1.0 if b % 2 else float(0.99)
        c["u"][b, 0] = float(g.random())
    want = ref_verify(c["parents"], c["ids"], c["target"], None, c["u"])
    assert (want[0] == 1).any()
    check_verify(verify(on(c)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
def test_verify_numbers_outside(drafted):
    """u that is NaN, negative or not below 1: no child is kept for NaN, the next id is the first or the last with mass."""
    c = make_verify(16, 8, 6, 3000, BF, "chain", drafted)
    c["target"][..., -100:] = 0
    for b, x in enumerate((float("nan"), -1.0, 1.0, 2.0, float("inf"), -float("inf"))):
        c["u"][b] = x
    check_verify(verify(on(c)), ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"]))


@pytest.mark.gpu
def test_verify_outputs_are_tensors_of_their_own():
    """The three results share an allocation and nothing else: contiguous, written to alone, in inference mode too, kept
    after the others are gone; none for no sequences."""
    c = make_verify(19, 5, 7, 40, torch.float32, "random")
    d, want = on(c), ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"])
    for inference in (False, True):
        with torch.inference_mode(inference):
            got = verify(d)
            assert [x.shape for x in got] == [(5,), (5, 7), (5, 7)] and all(x.is_contiguous() and x.dtype == torch.int32 for x in got)
            assert got.n.is_inference() == inference and not got.path.requires_grad
            got.path.fill_(-9)
            assert np.array_equal(got.n.cpu(), want[0]) and np.array_equal(got.tokens.cpu(), want[2])
            tokens = got.tokens
            del got
            torch.empty(5 * 15, dtype=torch.int32, device="cuda").fill_(3)
            assert np.array_equal(tokens.cpu(), want[2]) and torch.equal((tokens + 1).cpu(), torch.tensor(want[2] + 1, dtype=torch.int32))
    e = {k: v[:0] for k, v in d.items() if isinstance(v, torch.Tensor)}
    assert [x.shape for x in verify({**d, **e})] == [(0,), (0, 7), (0, 7)]


@pytest.mark.gpu
def test_verify_captured():
    """Replays over new numbers, with eager calls between; shared rows (stride 0)."""
    c = make_verify(17, 4, 8, 9000, torch.float32, "random")
    d = on(c)
    verify(d)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = verify(d)
    gen = torch.Generator().manual_seed(1)
    for _ in range(4):
        c["u"] = torch.rand(4, 8, generator=gen)
        d["u"].copy_(c["u"])
        g.replay()
        want = ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"])
        check_verify(out, want)
        check_verify(verify(d), want)
    one = {**c, "target": c["target"][:1, :1].expand(4, 8, -1), "draft": c["draft"][:1, :1].expand(4, 8, -1)}
    e = {**d, "target": d["target"][:1, :1].expand(4, 8, -1), "draft": d["draft"][:1, :1].expand(4, 8, -1)}
    check_verify(verify(e), ref_verify(one["parents"], one["ids"], one["target"], one["draft"], one["u"]))


@pytest.mark.gpu
def test_verify_follows_the_target():
    """The next token is distributed as the target's row, whatever the draft: 4096 sequences of three drafts of
    the root (the same rows, own numbers), every id's share within 5 standard deviations."""
    V, B, N = 12, 4096, 4
    g = torch.Generator().manual_seed(5)
    p = torch.softmax(torch.randn(V, generator=g) * 1.5, -1)
    q = torch.softmax(torch.randn(V, generator=g) * 1.5, -1)
    ids = torch.multinomial(q.expand(B, V), N, replacement=True, generator=g)
    u = torch.rand(B, N, generator=g)
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
    r = draft.verify(parents.cuda(), ids.cuda(), p.cuda().expand(B, N, V), q.cuda().expand(B, N, V), u.cuda())
    first = r.tokens[:, 0].cpu()
    share = torch.bincount(first, minlength=V).double() / B
    sd = (p.double() * (1 - p.double()) / B).sqrt()
    assert ((share - p.double()).abs() <= 5 * sd).all()
    assert int((r.n == 2).sum()) > B // 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32, torch.uint8])
@pytest.mark.parametrize("layers,lens,S", [(1, [0], 1), (3, [0, 15, 16, 17], 16), (2, [5, 100, 63], 7)])
def test_commit(layers, lens, S, dtype):
    c = make_commit(21, layers, len(lens), 6, lens, 2, 48, S, dtype)
    kc, vc, want = ref_commit(c)
    d = on(c)
    got = commit(d)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(d["k_cache"].cpu(), kc) and torch.equal(d["v_cache"].cpu(), vc)
    assert torch.equal(d["lens"].cpu(), c["lens"])
    # one layer at a time, slots behind heads
    for l in range(layers):
        e = on({**c, "k": c["k"][l], "v": c["v"][l], "k_cache": c["k_cache"][l], "v_cache": c["v_cache"][l]})
        e["k_cache"] = e["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(commit(e).cpu(), want)
        assert torch.equal(e["k_cache"].cpu(), kc[l]) and torch.equal(e["v_cache"].cpu(), vc[l])


@pytest.mark.gpu
def test_commit_what_does_not_fit_is_left():
    c = make_commit(22, 2, 7, 6, [10, 10, 10, 10, 10, 10, 10], 2, 64, 8, BF)
    c["n"][:] = 4
    c["path"][:] = torch.tensor([0, 1, 3, 5, -1, -1])
    c["lens"][0] = c["block_table"].shape[1] * 8 - 2   # two fit
    c["lens"][1] = -3
    c["lens"][2] = 2 ** 31 - 2
    c["block_table"][3, 1] = 10 ** 6
    c["path"][4, 2] = 6
    c["n"][5] = 7
    c["n"][6] = -4
    kc, vc, want = ref_commit(c)
    d = on(c)
    assert torch.equal(commit(d).cpu(), want)
    assert want.tolist() == [-1, -1, -1, -1, -1, -1, 10]
    assert torch.equal(d["k_cache"].cpu(), kc) and torch.equal(d["v_cache"].cpu(), vc)


@pytest.mark.gpu
def test_commit_edges():
    """The same node twice, no pages at all, no nodes kept, many layers."""
    c = make_commit(23, 9, 3, 5, [0, 30, 7], 1, 8, 4, BF)
    c["n"][:] = torch.tensor([5, 0, 3])
    c["path"][0] = torch.tensor([1, 1, 0, 4, 4])
    kc, vc, want = ref_commit(c)
    d = on(c)
    assert torch.equal(commit(d).cpu(), want)
    assert torch.equal(d["k_cache"].cpu(), kc) and torch.equal(d["v_cache"].cpu(), vc)
    d = on({**c, "block_table": torch.zeros(3, 0, dtype=torch.int32)})
    assert commit(d).tolist() == [-1, 30, -1]
    assert torch.equal(d["k_cache"].cpu(), c["k_cache"]) and torch.equal(d["v_cache"].cpu(), c["v_cache"])
    e = {k: v[:, :0] if k in ("k", "v") else v if k in ("k_cache", "v_cache") else v[:0] for k, v in on(c).items()}
    assert commit(e).shape == (0,)


# ---------------------------------------------------------------- the tokenizer's own path
class _Vocabulary:
    """What BPE.id_ranges needs, without a device: 20 residue tokens and merges, 3 bins an angle."""
    B, res_init, _tokens = 3, True, dict.fromkeys(range(20))

    def __getattr__(self, name):
        from geobpe.bpe import BPE
        f = getattr(BPE, name)
        return f.fget(self) if isinstance(f, property) else f.__get__(self)


def test_id_ranges_follow_the_encoded_order():
    from geobpe.bpe import BPE
    v = _Vocabulary()
    r = v.id_ranges()
    assert r.tolist() == [[0, 20], [23, 26], [26, 29], [20, 23]] and v.vocab_size == 29
    assert v.id_ranges("cpu") is v.id_ranges("cpu") and torch.equal(v.id_ranges("cpu"), torch.tensor(r))
    v._tokens = dict.fromkeys(range(25))
    old = v._id_ranges
    assert v.id_ranges("cpu")[0].tolist() == [0, 25] and len(old) == 2  # (a graph may hold the earlier one)
    with pytest.raises(ValueError, match="29|34"):
        v.verify_draft(None, None, torch.zeros(1, 1, 12), None, None, None)
    v.res_init = False
    with pytest.raises(NotImplementedError):
        v.id_ranges()
    assert BPE.verify_draft and BPE.id_ranges


def test_draft_cache_refusals():
    with pytest.raises(ValueError):
        draft.DraftCache(0, 1, 1, 1, 64, device="cpu")
    with pytest.raises(TypeError):
        draft.DraftCache(1, 1, 1, 1, 64, dtype=torch.float32, device="cpu")
    c = draft.DraftCache(2, 3, 100, 4, 64, device="cpu", page_size=16)
    assert c.k.shape == (2, 21, 16, 4, 64) and c.block_table.tolist()[1][0] == 7 and c.lens.tolist() == [0] * 3


def _golden_bpe():
    from conftest import load_golden
    from geobpe.bpe import BPE
    meta, corpus, _ = load_golden("g40x50_b5")
    bpe = BPE(corpus, bins={1: 5}, res_init=True, rmsd_partition_min_size=float("inf"), seed=0)
    bpe.initialize()
    bpe.bin()
    bpe.run(30)
    return bpe


@pytest.mark.gpu
def test_encoded_chains_lie_in_the_ranges():
    bpe = _golden_bpe()
    r = bpe.id_ranges()
    ids, off = bpe.encode_all()
    for a, b in zip(off[:-1], off[1:]):
        place = np.arange(b - a) % 4
        assert (ids[a:b] >= r[place, 0]).all() and (ids[a:b] < r[place, 1]).all()
    bpe.close()


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_decoding_run(graph):
    """A two-layer attention model over the trained vocabulary, drafts from its own first layer's logits: steps of
    attend / verify_draft / keep, compared step by step with the plain implementations, then recovered.  With
    ``graph`` a step is captured once and replayed with eager work between the replays."""
    bpe = _golden_bpe()
    dev, B, N, H, Hkv, D, L, V = "cuda", 3, 9, 4, 2, 64, 2, bpe.vocab_size + 2
    g = torch.Generator().manual_seed(3)
    w = lambda *s: (torch.randn(*s, generator=g) / s[0] ** 0.5).cuda()  # noqa: E731
    emb, wq, wk, wv, wo = w(V, 64), w(L, 64, H * D), w(L, 64, Hkv * D), w(L, 64, Hkv * D), w(L, H * D, 64)
    emb = emb * V ** 0.5
    wl, wd = w(64, V) * 3, w(64, V) * 3
    parents = torch.tensor([-1, 0, 1, 2, 0, 4, 5, 1, 7], dtype=torch.int32)
    up = parents.clamp(min=0).long().cuda()
    ranges = bpe.id_ranges(dev)
    depth = torch.tensor([len(p) - 1 for p in tree_paths(parents.tolist())], device=dev)
    cache = draft.DraftCache(L, B, 200, Hkv, D, BF, dev, page_size=16)
    par = parents.cuda()

    from geobpe.bpe import num_bonds
    bonds = np.array([num_bonds(t) for t in bpe._tokens.values()])
    ends = torch.tensor(np.pad(bonds % 3 != 0, (0, V - len(bonds))), device=dev)  # motifs that end a chain
    inner = np.flatnonzero(bonds % 3 == 0)

    def mask(x, start):  # each place's own ids, no end of a chain among them
        lo, hi = ranges[((start[:, None] + depth) % 4).long()].unbind(-1)
        y = torch.arange(V, device=dev)
        return torch.softmax(x.masked_fill((y < lo[..., None]) | (y >= hi[..., None]) | ends, -torch.inf), -1)

    def step(root, start, w_ids, u):
        """-> the kept ids, and everything a plain implementation needs to check the step"""
        q_rows = mask((emb[root] @ wd)[:, None].expand(B, N, V), start)
        cum = q_rows[:, up].cumsum(-1)
        ids = (cum <= w_ids[..., None] * cum[..., -1:]).sum(-1).clamp(max=V - 1)
        ids[:, 0] = root
        x = emb[ids]
        seen, ks, vs = [], [], []
        for l in range(L):
            q, k, v = ((x @ m[l]).to(BF).view(B, N, -1, D) for m in (wq, wk, wv))
            o = cache.attend(l, q, k, v, par)
            seen.append((q, o))
            ks.append(k)
            vs.append(v)
            x = x + o.float().reshape(B, N, -1) @ wo[l]
        p_rows = mask(x @ wl, start)
        got = bpe.verify_draft(par, ids, p_rows, q_rows, u, start)
        ks, vs = torch.stack(ks), torch.stack(vs)
        cache.keep(ks, vs, got)
        return got, ids, p_rows, q_rows, seen, ks, vs

    gen = torch.Generator().manual_seed(9)
    root = torch.tensor(inner[:3], device=dev)
    start = torch.ones(B, dtype=torch.int32, device=dev)
    w_ids, u = torch.rand(B, N, generator=gen).cuda(), torch.rand(B, N, generator=gen).cuda()
    if graph:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(root, start, w_ids, u)
        torch.cuda.current_stream().wait_stream(s)
        cache.lens.zero_()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            out = step(root, start, w_ids, u)
    chains = [[int(r)] for r in root.cpu()]
    keys = [[[] for _ in range(B)] for _ in range(L)]
    for t in range(6):
        w_ids.copy_(torch.rand(B, N, generator=gen))
        u.copy_(torch.rand(B, N, generator=gen))
        before = cache.lens.clone()
        if graph:
            captured.replay()
            torch.cuda.synchronize()
        else:
            out = step(root, start, w_ids, u)
        got, ids, p_rows, q_rows, seen, ks, vs = out
        check_verify(got, ref_verify(parents, ids, p_rows, q_rows, u, ranges, start.cpu()))
        for l, (q, o) in enumerate(seen):
            check_attention(o, ref_attention(q, cache.k[l], cache.v[l], cache.block_table, before, ks[l], vs[l], parents), BF)
        n = got.n.tolist()
        for b in range(B):
            chains[b] += got.tokens[b, :n[b]].tolist()
            for l in range(L):
                keys[l][b] += [ks[l, b, i].cpu() for i in got.path[b, :n[b]].tolist()]
                pos = torch.arange(len(keys[l][b]))
                page = cache.block_table[b].cpu().long()[pos // 16]
                assert torch.equal(cache.k[l].cpu()[page, pos % 16], torch.stack(keys[l][b]))
        assert cache.lens.tolist() == [len(c) - 1 for c in chains]
        root.copy_(got.tokens.gather(1, (got.n.long() - 1)[:, None])[:, 0])
        start.add_(got.n)
        torch.zeros(1000, device=dev).normal_().sum().item()  # (eager work between the replays)
    for c in chains:
        c = c[:len(c) // 4 * 4] + [int(np.flatnonzero(bonds == 2)[0])]  # whole tokens and a last residue
        dq = bpe.dequantize(c)
        assert bpe.quantize(dq) == c
        assert 3 * bpe.recover_structure(bpe.recover(dq), dq).n - 1 == bonds[c[::4]].sum()
    bpe.close()
