"""More of the decoding operators (geobpe.draft) against plain 64-bit implementations: rows held to id ranges that have
mass outside them, scales and scores at the ends of float32, long contexts with every tile visible, a prompt in chains, caches
that share memory, what autograd is told.

Attention's tolerance is test_draft.py's, from the same count of roundings."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from conftest import REPO
from geobpe import draft
from test_draft import (_ATTEND, _Vocabulary, attend, check_attention, check_verify, commit, make_attention, make_commit,
                        make_verify, on, ref_attention, ref_verify, refuse, tree_paths, verify)

BF, FP = torch.bfloat16, torch.float16


# ---------------------------------------------------------------- rows held to their place's ids
def ref_held(parents, ids, target, draft_, u, ranges, start):
    """Verification with ranges: every row divided by what it holds inside the range of its place (1 where that is 1 but for
    the type's rounding, half a step and 2^-20 for a 32-bit softmax's sum), drafted ids outside it (or of a draft row without
    mass there) passed over.  64 bits, a loop over the children."""
    near = torch.finfo(target.dtype).eps / 2 + 2.0 ** -20
    mass = lambda x: 1.0 if abs(x.sum() - 1) <= near else x.sum()  # noqa: E731
    ids, u, parents, start = ids.cpu().numpy(), u.double().cpu().numpy(), parents.cpu().numpy(), start.cpu().numpy()
    ranges = ranges.cpu().numpy()
    B, N, V = target.shape
    clean = lambda x: np.where(np.isfinite(x) & (x > 0), x, 0.0)  # noqa: E731
    target = clean(target.double().cpu().numpy())
    draft_ = None if draft_ is None else clean(draft_.double().cpu().numpy())
    n, paths, tokens = np.zeros(B, int), np.full((B, N), -1), np.full((B, N), -1)
    for b in range(B):
        par = (parents if parents.ndim == 1 else parents[b]).tolist()
        present = tree_paths(par)
        if present[0] is None:
            continue
        path, toks = [0], []
        while True:
            c = path[-1]
            lo, hi = ranges[(int(start[b]) + len(toks)) % len(ranges)]
            lo, hi = max(int(lo), 0), min(int(hi), V)
            p = target[b, c, lo:hi] if lo < hi else np.zeros(0)
            r, Z, kept = p.copy(), mass(p), None
            if draft_ is not None:
                q = draft_[b, c, lo:hi] if lo < hi else np.zeros(0)
                Q = mass(q)
            for i in range(c + 1, N):
                x = int(ids[b, i]) - lo
                if present[i] is None or par[i] != c or not 0 <= x < hi - lo:
                    continue
                if draft_ is None:
                    took, most = np.zeros(hi - lo), Z
                    took[x] = np.inf
                elif Q > 0:
                    took, most = q * (Z / Q), q[x] * (Z / Q)
                else:
                    continue
                if u[b, i] * most < r[x]:
                    kept = i
                    break
                r = np.maximum(r - took, 0.0)
                Z = r.sum()
            if kept is None:
                break
            path.append(kept)
            toks.append(int(ids[b, kept]))
        if not r.sum() > 0:
            r = p
        cum = np.cumsum(r)
        if len(cum) and cum[-1] > 0:
            hit = np.flatnonzero(cum > u[b, 0] * cum[-1])
            toks.append(lo + (int(hit[0]) if len(hit) else int(np.flatnonzero(r)[-1])))
        else:
            toks.append(-1)
        n[b] = len(path)
        paths[b, :len(path)] = path
        tokens[b, :len(toks)] = toks
    return n, paths, tokens


def make_held(seed, B, N, V, dtype, kind, ranges, drafted=True, sharp=2.0):
    """Rows over the whole vocabulary, ids drawn from them: some outside their range."""
    c = make_verify(seed, B, N, V, dtype, kind, True, sharp)
    g = np.random.default_rng(seed + 1000)
    c["ranges"] = torch.tensor(ranges, dtype=torch.int32)
    c["start"] = torch.tensor(g.integers(0, 50, B), dtype=torch.int32)
    for b in range(B):  # (a range of a few ids seldom meets an id of the whole vocabulary)
        for i, path in enumerate(tree_paths(c["parents"][b].tolist())):
            lo, hi = c["ranges"][(int(c["start"][b]) + len(path) - 2) % len(ranges)].clamp(0, V).tolist()
            if i and hi > lo and g.random() < 0.7:
                c["ids"][b, i] = int(g.integers(lo, hi))
    if not drafted:
        c["draft"] = None
    return c


FIRST = [  # ids, range, drafted: tokens after a root with three drafts of its own
    (12, (3, 9), True), (12, (3, 9), False), (12, (0, 12), True), (300, (7, 12), True), (300, (7, 12), False),
]


def first_tokens(V, held, drafted, B, seed):
    """One root, three drafts drawn from its draft row, the rows' mass in and outside the range [lo, hi)."""
    g = torch.Generator().manual_seed(seed)
    p = torch.softmax(torch.randn(V, generator=g) * 1.5, -1)
    q = torch.softmax(torch.randn(V, generator=g) * 1.5, -1)
    lo, hi = held
    inside = torch.zeros(V, dtype=torch.bool)
    inside[lo:hi] = True
    if not inside.all():  # (half of the target's mass and a third of the draft's lie outside)
        p, q = (torch.where(inside, a * x / x[inside].sum(), (1 - a) * x / x[~inside].sum()) for x, a in ((p, 1 / 2), (q, 2 / 3)))
    N = 4
    ids = torch.multinomial(q.expand(B, V), N, replacement=True, generator=g)
    if not drafted:  # (the same ids for everyone, the likeliest first: what is kept of them too often shows)
        ids = (lo + p[lo:hi].topk(N).indices).expand(B, N).contiguous()
    c = dict(parents=torch.tensor([-1, 0, 0, 0], dtype=torch.int32), ids=ids, target=p.expand(B, N, V),
             draft=q.expand(B, N, V) if drafted else None, u=torch.rand(B, N, generator=g),
             ranges=torch.tensor([held], dtype=torch.int32), start=torch.zeros(B, dtype=torch.int32))
    want = p.double()[lo:hi] / p.double()[lo:hi].sum()
    return c, want


def share_of_target(tokens, held, want):
    """Every id's share within 5 standard deviations of the target's row held to the range."""
    lo, hi = held
    assert ((tokens >= lo) & (tokens < hi)).all()
    share = torch.bincount(tokens - lo, minlength=hi - lo).double() / len(tokens)
    return bool(((share - want).abs() <= 5 * (want * (1 - want) / len(tokens)).sqrt()).all())


@pytest.mark.parametrize("V,held,drafted", FIRST)
def test_held_rows_follow_the_target_plainly(V, held, drafted):
    """The plain implementation itself: the target's row divided by its mass in the range.  Rows taken as they are
    inside it (their mass as 1) give other shares wherever mass lies outside."""
    c, want = first_tokens(V, held, drafted, 2048, 3)
    args = [c[k] for k in ("parents", "ids", "target", "draft", "u", "ranges", "start")]
    assert share_of_target(torch.tensor(ref_held(*args)[2][:, 0]), held, want)
    as_they_are = torch.tensor(ref_verify(*args)[2][:, 0])
    assert share_of_target(as_they_are, held, want) == (held == (0, V))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("V,held,drafted", FIRST)
def test_verify_held_rows_follow_the_target(V, held, drafted, dtype):
    c, want = first_tokens(V, held, drafted, 8192, 5)
    if dtype == BF:  # (a row in 16 bits is another row: its own shares are the ones to follow)
        c["target"] = c["target"][:1, :1].to(BF).expand_as(c["target"])
        lo, hi = held
        want = c["target"][0, 0, lo:hi].double()
        want = want / want.sum()
        if drafted:
            c["draft"] = c["draft"][:1, :1].to(BF).expand_as(c["draft"])
    r = verify(on(c))
    assert share_of_target(r.tokens[:, 0].cpu().long(), held, want)
    assert int((r.n == 2).sum()) > 500


HELD = [
    # B, N, V, tree, ranges
    (9, 20, 300, "random", [[0, 285], [290, 295], [295, 300], [285, 290]]),
    (6, 30, 60, "flat", [[10, 50]]),
    (6, 30, 60, "flat", [[3, 8], [5, 60]]),
    (12, 7, 1091, "chain", [[0, 1076], [1081, 1086], [1086, 1091], [1076, 1081]]),
    (5, 128, 90, "random", [[0, 17], [17, 34], [34, 90]]),
    (4, 128, 50, "flat", [[1, 49]]),
    (5, 9, 5123, "random", [[0, 5108], [5108, 5123]]),
    (3, 6, 20001, "flat", [[1, 20000], [19000, 30000]]),
    (3, 4, 70001, "random", [[-5, 69999], [5, 70001], [0, 40000]]),
    (2, 1, 40, "chain", [[5, 9]]),
    (4, 6, 40, "random", [[0, 0], [10, 5], [50, 60], [0, 40]]),
    (4, 6, 40, "random", [[7, 8], [0, 40]]),
    (3, 65, 200, "random", [[0, 64], [64, 129], [100, 116], [100, 117]]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, BF, FP])
@pytest.mark.parametrize("shape", HELD, ids=lambda s: "x".join(map(str, s[:4])))
def test_verify_held_rows(shape, dtype, drafted):
    B, N, V, kind, ranges = shape
    c = make_held(31, B, N, V, dtype, kind, ranges, drafted)
    want = ref_held(c["parents"], c["ids"], c["target"], c["draft"], c["u"], c["ranges"], c["start"])
    check_verify(verify(on(c)), want)
    d = on(c)  # int32 ids, rows that begin anywhere
    d["ids"] = d["ids"].int()
    wide = torch.full((B, N, V + 9), float("nan"), dtype=dtype, device="cuda")
    wide[..., 3:V + 3] = d["target"]
    d["target"] = wide[..., 3:V + 3]
    check_verify(verify(d), want)


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("V,ranges", [(40, [[3, 30]]), (40, [[3, 12], [20, 25]]), (9000, [[10, 8999]])])
def test_verify_held_rows_edges(V, ranges, drafted):
    """Rows and drafts without mass in the range, rows of any mass, equal rows, ids outside the range and the vocabulary, the
    same id twice, numbers at both ends, absent nodes."""
    B, N = 14, 10
    c = make_held(32, B, N, V, torch.float32, "random", ranges, drafted)
    lo, hi = ranges[0]
    c["parents"][3:10] = torch.tensor([-1] + [0] * (N - 1), dtype=torch.int32)
    c["target"][0] = 0
    c["target"][1, :, lo:hi:2] = float("nan")
    c["target"][1, :, lo + 1] = float("inf")
    c["target"][2] *= 1e-30
    c["target"][4] *= 7
    c["ids"][5, 1:6] = torch.tensor([-1, V, 2 ** 40, lo - 1, hi])
    c["ids"][6] = lo + 2
    c["u"][7] = 0
    c["u"][8] = float(np.nextafter(np.float32(1), np.float32(0)))
    c["u"][9] = float("nan")
    c["parents"][10, 0] = 0
    c["parents"][11, 1] = -1
    c["start"][12] = -7
    c["start"][13] = 2 ** 31 - 1
    if drafted:
        c["draft"][3, :, lo:hi] = 0
        c["draft"][4] = c["target"][4] / 2
        c["draft"][7] *= 1e30
        c["draft"][8, :, lo + 1:hi:3] = 0
    want = ref_held(c["parents"], c["ids"], c["target"], c["draft"], c["u"], c["ranges"], c["start"])
    assert want[0][10] == 0 and want[2][0, 0] == -1
    check_verify(verify(on(c)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, BF, FP])
@pytest.mark.parametrize("V", [40, 1091, 20001])
def test_verify_ranges_that_leave_nothing_out(V, dtype, drafted):
    """Rows that sum to 1 but for their rounding inside the range are used as they are: a range of everything, or of all that
    is not 0, changes no id."""
    c = make_verify(34, 64, 9, V, dtype, "random", drafted)
    want = ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"])
    d = on(c)
    check_verify(verify(d), want)
    d["ranges"], d["start"] = torch.tensor([[0, V], [-1, V + 3]], dtype=torch.int32).cuda(), torch.arange(64, dtype=torch.int32).cuda()
    check_verify(verify(d), want)
    ranges = torch.tensor([[0, V - 15], [V - 10, V - 5], [V - 5, V], [V - 15, V - 10]], dtype=torch.int32)
    c = make_verify(35, 64, 9, V, dtype, "random", drafted, ranges=ranges)
    check_verify(verify(on(c)), ref_verify(c["parents"], c["ids"], c["target"], c["draft"], c["u"], ranges, c["start"]))


@pytest.mark.gpu
def test_verify_held_rows_captured():
    """A captured call with ranges, replayed over new rows and numbers with eager calls between."""
    ranges = [[0, 285], [290, 295], [295, 300], [285, 290]]
    c = make_held(33, 6, 20, 300, torch.float32, "random", ranges)
    d = on(c)
    verify(d)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = verify(d)
    for seed in range(4):
        c = make_held(40 + seed, 6, 20, 300, torch.float32, "random", ranges)
        for k in d:
            d[k].copy_(c[k])
        g.replay()
        want = ref_held(c["parents"], c["ids"], c["target"], c["draft"], c["u"], c["ranges"], c["start"])
        check_verify(out, want)
        check_verify(verify(d), want)


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
def test_vocabulary_holds_plain_rows_to_their_place(drafted):
    """BPE.verify_draft over a model's plain softmax, wider than the vocabulary: the first token after the root is
    distributed as the target's row among the ids of its place."""
    v = _Vocabulary()
    V, B, N = v.vocab_size + 3, 8192, 4
    g = torch.Generator().manual_seed(8)
    for place in range(4):
        p = torch.softmax(torch.randn(V, generator=g), -1)
        q = torch.softmax(torch.randn(V, generator=g), -1)
        ids = torch.multinomial(q.expand(B, V), N, replacement=True, generator=g)
        u = torch.rand(B, N, generator=g)
        lo, hi = v.id_ranges()[place].tolist()
        if not drafted:
            ids = (lo + p[lo:hi].topk(3).indices[[0, 0, 1, 2]]).expand(B, N).contiguous()
        r = v.verify_draft(torch.tensor([-1, 0, 0, 0], dtype=torch.int32).cuda(), ids.cuda(), p.cuda().expand(B, N, V),
                           q.cuda().expand(B, N, V) if drafted else None, u.cuda(),
                           torch.full((B,), 4 * 9 + place, dtype=torch.int32).cuda())
        want = p.double()[lo:hi] / p.double()[lo:hi].sum()
        assert share_of_target(r.tokens[:, 0].cpu().long(), (lo, hi), want)


# ---------------------------------------------------------------- flags of a tree's tiles
def test_a_tiles_flag_is_its_own(tmp_path):
    """csrc/draft.h's flags of tiles with values that are not finite, in the order that waves may take: one has gone on to the
    second tile and marks it before another has read the first one's.  Had the two one word, the second wave would take the first
    tile for marked, and wait at other barriers than the first."""
    src = tmp_path / "flags.cpp"
    src.write_text("""
#include <stdint.h>
#define __device__
static inline uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a * b) >> 32); }
#include "draft.h"
using namespace gb;
extern "C" int late_reader(int first_marked, int tile_keys) {  // what the late wave reads of the first tile
  TileFlags f;
  f.clear();
  if (first_marked) f.mark(0);
  f.mark(tile_keys);       // the wave that is ahead, in the second tile
  return f.marked(0) | f.marked(tile_keys) << 1;
}
extern "C" int early_reader(int tile_keys) {
  TileFlags f;
  f.clear();
  f.mark(0);
  return f.marked(0) | f.marked(tile_keys) << 1;
}
""")
    so = tmp_path / "flags.so"
    subprocess.run([shutil.which("g++"), "-O1", "-shared", "-fPIC", "-Wno-unknown-pragmas",
                    f"-I{os.path.join(REPO, 'pt-bpe_amd', 'csrc')}", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    assert lib.late_reader(0, 64) == 2 and lib.late_reader(1, 64) == 3
    assert lib.early_reader(64) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("N,Hq,D", [(128, 12, 128), (128, 2, 64), (100, 1, 40), (65, 3, 256), (128, 1, 24)])
@pytest.mark.parametrize("where", ["second", "first", "both"])
def test_attention_values_not_finite_by_tile(N, Hq, D, where):
    """More than 64 nodes are two tiles: a value that is not finite in either one alone, and in both."""
    c = make_attention(41, 3, N, [200, 0, 33], Hq, 1, D, 16, BF)
    if where != "first":
        c["v"][0, N - 1, 0, D - 1] = float("nan")
        c["v"][1, 64, 0, 0] = float("inf")
    if where != "second":
        c["v"][0, 63, 0, 1] = float("inf")
        c["v"][2, 5, 0, :] = -float("inf")
    want = ref_attention(**c)
    d = on(c)
    for _ in range(3):
        check_attention(attend(d), want, BF)


# ---------------------------------------------------------------- scales and scores
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, -1e300, 3e38])
def test_attention_refuses_scales_that_are_not_finite(scale):
    """NaN, infinities and what is none of float32's: a call would answer with a plain mean, or with NaN."""
    from geobpe import _native
    c = make_attention(0, 2, 3, [5, 9], 4, 2, 16, 4, BF)
    refuse(attend, c, ValueError, "scale", scale=scale)
    refuse(attend, c, TypeError, "real number|float", scale="1")
    L = _native.lib()
    args = ([256] * 9 + [64] * 15 + [1, 0] + [1, 2, 4, 2, 64, 16, 3, 2, 0])
    assert L.geobpe_tree_attention(0, None, _ATTEND.pack(*args, scale), 256, 1 << 40) == _native.E_ARG
    assert b"scale" in L.geobpe_draft_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("N", [3, 40])
@pytest.mark.parametrize("scale", [1.0, -1.0, 3.0, 1e5, 1e20, 1e30])
def test_attention_large_scores(N, scale, dtype):
    """Scores of up to 1e36 whose weights are known: keys are whole numbers times one vector, so every score is a whole number of
    steps, exact in float32, and all but the largest are at least one step of 2^10 and more below it.  Keys that share the largest
    share the row's weight."""
    c = make_attention(55, 3, N, [90, 700, 5000], 4, 2, 64, 16, dtype)
    g = np.random.default_rng(55)

    def whole(x):  # one whole number of 0 .. 7 in channels 0 and 1, nothing else
        y = torch.zeros(x.shape)
        y[..., 0] = torch.tensor(g.integers(0, 8, x.shape[:-1])).float() * 32
        y[..., 1] = y[..., 0]
        return torch.where(torch.isnan(x.float()), x.float(), y).to(dtype)

    c["k_cache"], c["k"] = whole(c["k_cache"]), whole(c["k"])
    c["q"] = torch.zeros(c["q"].shape).to(dtype)
    c["q"][..., 0] = 100
    c["q"][..., 1] = 60
    c["q"][:, 1::2, :, :2] *= -1
    c["scale"] = scale
    check_attention(attend(on(c)), ref_attention(**c), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 40])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-33, -1e-33, 1e-38, 1e-45])
def test_attention_small_scales_of_large_scores(N, scale):
    """Products q k of up to 1e33: a scale of 0 is the mean of the values all the same, and one of 1e-33 gives scores of
    some units."""
    c = make_attention(51, 2, N, [90, 600], 4, 2, 16, 16, BF)
    c["q"] = (c["q"].float() * 1e16).to(BF)
    c["k"] = (c["k"].float() * 1e16).to(BF)
    c["k_cache"] = (c["k_cache"].float() * 1e16).to(BF)
    c["scale"] = scale
    check_attention(attend(on(c)), ref_attention(**c), BF)


# ---------------------------------------------------------------- what autograd is told
def test_tangents_are_refused():
    """There is no forward derivative either: a tensor with a tangent would lose it without a word."""
    import torch.autograd.forward_ad as fw
    a, v, k = (make_attention(0, 2, 3, [5, 9], 4, 2, 16, 4, BF), make_verify(0, 2, 4, 20, torch.float32, "random"),
               make_commit(0, 2, 3, 4, [0, 5, 7], 2, 16, 4, BF))
    with fw.dual_level():
        for f, c, names in ((attend, a, ("q", "k_cache", "v_cache", "k", "v")), (verify, v, ("target", "draft")),
                            (commit, k, ("k_cache", "v_cache", "k", "v"))):
            for name in names:
                dual = fw.make_dual(c[name], torch.ones_like(c[name]))
                refuse(f, c, ValueError, "no backward", **{name: dual})
                with torch.no_grad():  # (tangents go on under no_grad)
                    refuse(f, c, ValueError, "no backward", **{name: dual})
                with torch.inference_mode():
                    refuse(f, c, ValueError, "HIP device only", **{name: dual})
            refuse(f, c, ValueError, "HIP device only")


@pytest.mark.gpu
@pytest.mark.parametrize("N,lens", [(3, [40, 5000, 0]), (40, [40, 5000, 0]), (40, [5000, 5000, 5000])])
def test_attention_rows_without_weights(N, lens):
    """A present node all of whose scores are -infinity has no weights: NaN, whether its sequence is cut into parts or not.
    An absent node's row stays 0."""
    c = make_attention(61, 3, N, lens, 2, 1, 64, 16, BF)
    used = ~torch.isnan(c["k_cache"])
    c["k_cache"][..., 0] = torch.where(used[..., 0], -1.0, float("nan")).to(BF)
    c["k"][..., 0] = -1
    c["q"][:, 1, 1, 0] = float("inf")
    c["q"][:, N - 1, 0, 0] = float("inf")
    c["parents"][:, N - 1] = -3
    want = ref_attention(**c)
    assert np.isnan(want[0][:, 1, 1]).all() and not want[0][:, N - 1].any() and np.isfinite(want[0][:, 0]).all()
    check_attention(attend(on(c)), want, BF)


# ---------------------------------------------------------------- caches that share memory
def caches_of_one(kind, L, P, S, H, D, dtype=BF, device="cpu"):
    """Keys' and values' cache in one tensor, without an element in common."""
    z = lambda *s: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    if kind == "pages":
        both = z(L, P, 2, S, H, D)
        return both[:, :, 0], both[:, :, 1]
    if kind == "heads":
        both = z(L, P, S, H, 2 * D)
        return both[..., :D], both[..., D:]
    if kind == "layers":
        both = z(2, L, P, S, H, D)
        return both[0], both[1]
    if kind == "heads first":
        both = z(L, P, 2, H, S, D).transpose(3, 4)
        return both[:, :, 0], both[:, :, 1]
    both = z(L, 2 * P, S, H, D)
    return both[:, 1::2], both[:, 0::2]


KINDS = ["pages", "heads", "layers", "heads first", "turns"]


def test_commit_refuses_caches_that_overlap():
    """One a few pages, slots or heads further on in the other's memory, rows that overlap in a cache: two writes to one
    place.  Caches that only lie in one tensor are none of these."""
    c = make_commit(0, 2, 3, 4, [0, 5, 7], 2, 16, 4, BF)
    L, P, S, H, D = c["k_cache"].shape
    for kind in KINDS:
        k, v = caches_of_one(kind, L, P, S, H, D)
        refuse(commit, c, ValueError, "HIP device only", k_cache=k, v_cache=v)
        refuse(commit, c, ValueError, "HIP device only", k_cache=v, v_cache=k)
    pages, slots, heads = (torch.zeros(L, P + a, S + b, H + h, D, dtype=BF) for a, b, h in ((1, 0, 0), (0, 1, 0), (0, 0, 1)))
    refuse(commit, c, ValueError, "partly k_cache", k_cache=pages[:, 1:], v_cache=pages[:, :-1])
    refuse(commit, c, ValueError, "partly k_cache", k_cache=pages[:, :-1], v_cache=pages[:, 1:])
    refuse(commit, c, ValueError, "partly k_cache", k_cache=slots[:, :, 1:], v_cache=slots[:, :, :-1])
    refuse(commit, c, ValueError, "partly k_cache", k_cache=heads[:, :, :, :-1], v_cache=heads[:, :, :, 1:])
    wide = torch.zeros(L, P, S, H, 2 * D, dtype=BF)
    refuse(commit, c, ValueError, "partly k_cache", k_cache=wide[..., :D], v_cache=wide[..., 8:D + 8])
    flat = torch.zeros(L * P * S * H * D, dtype=BF)
    near = torch.as_strided(flat, (L, P, S, H, D), (P * S * H * D, S * H * D, H * D, 8, 1))  # heads half a head apart
    refuse(commit, c, ValueError, "overlap", k_cache=near)
    refuse(commit, c, ValueError, "overlap", v_cache=torch.as_strided(flat, (L, P, S, H, D), (P * 8, 8, H * D, D, 1)))
    refuse(commit, c, ValueError, "expanded", v_cache=c["v_cache"][:, :, :1].expand(-1, -1, S, -1, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_commit_into_caches_of_one_tensor(kind):
    from test_draft import ref_commit
    c = make_commit(76, 3, 4, 6, [0, 15, 16, 17], 2, 48, 16, BF)
    kc, vc, want = ref_commit(c)
    d = on(c)
    k, v = caches_of_one(kind, *c["k_cache"].shape, device="cuda")
    k.copy_(d["k_cache"])
    v.copy_(d["v_cache"])
    assert torch.equal(commit({**d, "k_cache": k, "v_cache": v}).cpu(), want)
    assert torch.equal(k.cpu(), kc) and torch.equal(v.cpu(), vc)


@pytest.mark.gpu
def test_commit_tells_autograd_of_its_writes():
    """A cache that a later backward pass needs as it was: torch has to see that it was written."""
    c = on(make_commit(71, 2, 3, 4, [0, 5, 7], 2, 16, 4, torch.float32))
    before = c["k_cache"]._version, c["v_cache"]._version
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = (c["k_cache"] * w).sum() + (c["v_cache"] * w).sum()
    commit(c)
    assert c["k_cache"]._version > before[0] and c["v_cache"]._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():  # (tensors without a version)
        d = {k: v.clone() for k, v in c.items()}
        assert torch.equal(commit(d), commit({**c, "k_cache": c["k_cache"].clone(), "v_cache": c["v_cache"].clone()}))


# ---------------------------------------------------------------- long contexts, every tile visible
def level(L):
    """A position's score in powers of two: parts of 512 positions lie up to 2^12 apart."""
    return (np.arange(L) // 512 * 5) % 13 - 6


def make_visible(seed, N, L, G, Hkv, D, dtype, S=64):
    """One sequence of L positions and a chain of N nodes.  Position x's weight is nearly 2^level.  Marked positions have the value
    2^-level in one channel and 0 in the others, so that a channel of a result is the sum of a few shares that are about alike:
    the first half of the kv heads has a channel for every 512 positions, the second one for the ends of every 16 (about
    L / (4 Hkv D) of them a channel).  The level also is channel 0 of the keys."""
    g = np.random.default_rng(seed)
    M = -(-L // S)
    x, pages, half = np.arange(L), g.permutation(M + 1)[:M], Hkv // 2
    k = g.standard_normal((L, Hkv, D)) * 0.25
    k[:, :, 0] = level(L)[:, None]
    v = np.zeros((L, Hkv, D))
    v[x, x // 512 % half, x // 512 // half % D] = 2.0 ** -level(L)
    ends = x[(x % 16 == 0) | (x % 16 == 15) | (x == L - 1)]
    turn = ends // 16 * 2 + (ends % 16 > 0)
    v[ends, half + turn % half, turn // half % D] = 2.0 ** -level(L)[ends]
    kc, vc = (torch.full((M + 1, S, Hkv, D), float("nan"), dtype=dtype) for _ in range(2))
    page = torch.tensor(pages[x // S])
    kc[page, x % S], vc[page, x % S] = torch.tensor(k).to(dtype), torch.tensor(v).to(dtype)
    q = g.standard_normal((1, N, Hkv * G, D)) * 0.25
    q[..., 0] = np.log(2) * D ** 0.5
    own = g.standard_normal((1, N, Hkv, D)) * 0.25
    own[..., 0] = 0
    t = lambda y: torch.tensor(y).to(dtype)  # noqa: E731
    return dict(q=t(q), k_cache=kc, v_cache=vc, block_table=torch.tensor(pages[None], dtype=torch.int32),
                lens=torch.tensor([L], dtype=torch.int32), k=t(own), v=t(np.zeros((1, N, Hkv, D))),
                parents=torch.arange(-1, N - 1, dtype=torch.int32))


def visible_heads(c):
    """Per query head the weights (nodes x keys) and the values (keys x D), float64, of one sequence whose nodes are a chain."""
    L, S = int(c["lens"][0]), c["k_cache"].shape[1]
    x = np.arange(L)
    page = c["block_table"][0].long().numpy()[x // S]
    kc, vc = c["k_cache"].double().numpy()[page, x % S], c["v_cache"].double().numpy()[page, x % S]
    q, k, v = (c[n][0].double().numpy() for n in ("q", "k", "v"))
    N, Hq, D = q.shape
    chain = np.tril(np.ones((N, N), bool))
    for h in range(Hq):
        g = h // (Hq // k.shape[1])
        s = np.concatenate([q[:, h] @ kc[:, g].T, np.where(chain, q[:, h] @ k[:, g].T, -np.inf)], 1) * D ** -0.5
        yield np.exp(s - s.max(1, keepdims=True)), np.concatenate([vc[:, g], v[:, g]])


def ref_visible(heads, factor=1.0):
    """The result and sum w |v| / sum w, the cache's weights multiplied by ``factor`` (0: a lost key)."""
    out, mag = [], []
    for w, v in heads:
        w = w.copy()
        w[:, :w.shape[1] - w.shape[0]] *= factor
        out.append(w @ v / w.sum(1, keepdims=True))
        mag.append(w @ np.abs(v) / w.sum(1, keepdims=True))
    return np.stack(out, 1)[None], np.stack(mag, 1)[None]


VISIBLE = [  # nodes, positions, query heads a kv head, kv heads, head
    (2, 70001, 1, 8, 128), (5, 5000, 2, 4, 64), (1, 40000, 4, 8, 96), (16, 70001, 4, 8, 128), (40, 20001, 1, 8, 64),
    (100, 9000, 2, 4, 128), (3, 12345, 1, 8, 200), (20, 12345, 1, 8, 256),
]


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("L", [5000, 70001])
def test_a_lost_tile_would_be_seen(L, dtype):
    """The check passes for the result rounded to the type, and fails for one without a key at a tile's end, a tile, a part or
    the last position, and for one whose parts are joined with a weight a little off."""
    heads = list(visible_heads(make_visible(81, 1, L, 1, 8, 128, dtype)))
    want, x = ref_visible(heads), np.arange(L)
    check_attention(torch.tensor(want[0]).to(dtype), want, dtype)

    def seen(which, factor=0.0):
        got = torch.tensor(ref_visible(heads, np.where(which, factor, 1.0))[0]).to(dtype)
        try:
            check_attention(got, want, dtype)
        except AssertionError:
            return True
        return False

    for at in (0, 31, 32, 511, 512, 2047, 2048, L // 32 * 32, L - 1):
        assert seen(x == at) and seen((x >= at) & (x < at + 32)), at
    part = x // 512 == 3
    assert seen(part) and seen(part, 1.05) and seen(x // 512 == x[-1] // 512, 0.95) and not seen(part, 1.0)
    if L > 10000:
        assert seen((x >= 20000) & (x < 27000))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("shape", VISIBLE, ids=lambda s: "x".join(map(str, s)))
def test_attention_of_every_tile(shape, dtype):
    N, L, G, Hkv, D = shape
    c = make_visible(82, N, L, G, Hkv, D, dtype)
    check_attention(attend(on(c)), ref_visible(visible_heads(c)), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [2, 30])
@pytest.mark.parametrize("N", [2, 40])
def test_attention_of_every_tile_with_room_in_the_table(N, room):
    """The parts are cut for the table's positions: the same sequence under a table of ``room`` times as many."""
    c = make_visible(83, N, 5000, 1, 8, 64, FP)
    want = ref_visible(visible_heads(c))
    table = torch.full((1, c["block_table"].shape[1] * room), -1, dtype=torch.int32)
    table[:, :c["block_table"].shape[1]] = c["block_table"]
    c["block_table"] = table
    check_attention(attend(on(c)), want, FP)


# ---------------------------------------------------------------- a prompt, in chains
@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [128, 37])
def test_prompt_in_chains(chunk):
    """Prompts of 300 and 170 ids (and none) go into a DraftCache as chains of up to ``chunk`` nodes, every one attended to and kept
    whole; a sequence that has no more is absent.  The rows are those of causal attention over the whole prompt."""
    lens, L, H, Hkv, D = [300, 170, 0], 2, 4, 2, 64
    B, g = len(lens), torch.Generator().manual_seed(91)
    r = lambda h: torch.randn(L, B, max(lens), h, D, generator=g).to(BF)  # noqa: E731
    q, k, v = r(H), r(Hkv), r(Hkv)
    cache = draft.DraftCache(L, B, 320, Hkv, D, BF, page_size=16)
    got = torch.zeros(L, B, max(lens), H, D, dtype=BF)
    for at in range(0, max(lens), chunk):
        here = [max(0, min(n - at, chunk)) for n in lens]
        N = max(here)
        parents = torch.arange(-1, N - 1, dtype=torch.int32).repeat(B, 1)
        for b, n in enumerate(here):
            if n < N:
                parents[b, n] = -2  # (what hangs on it is absent too: the rest, or all of a sequence without a root)
        kk, vv = k[:, :, at:at + N].cuda(), v[:, :, at:at + N].cuda()
        for l in range(L):
            got[l, :, at:at + N] = cache.attend(l, q[l, :, at:at + N].cuda(), kk[l], vv[l], parents.cuda()).cpu()
        path = torch.arange(N, dtype=torch.int32, device="cuda").repeat(B, 1)
        cache.keep(kk, vv, draft.Verified(torch.tensor(here, dtype=torch.int32).cuda(), path, None))
    assert cache.lens.tolist() == lens
    eps = torch.finfo(BF).eps
    for l in range(L):
        for b, n in enumerate(lens):
            assert not got[l, b, n:].any()
            for h in range(H):
                kd, vd = (x[l, b, :n, h // (H // Hkv)].double() for x in (k, v))
                s = (q[l, b, :n, h].double() @ kd.t() * D ** -0.5).masked_fill(~torch.ones(n, n).tril().bool(), -torch.inf)
                w = torch.softmax(s, -1)
                want, mag = w @ vd, w @ vd.abs()
                assert ((got[l, b, :n, h].double() - want).abs() <= (eps + 2.0 ** -8) * mag + eps / 2 * want.abs() + 2.0 ** -24).all()
