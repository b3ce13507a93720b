"""The decoding operators of geobpe.draft (attention of a drafted tree over a paged cache, verification of the
drafted ids, keeping the accepted path in the cache) as measured work: cases, inputs, plain forms and 64-bit results.

A tree has N nodes; node 0 is the last decided token (not in the cache yet), parents[b, i] < i.  A GeoBPE chain of T
tokens is 4 T - 3 ids: chains of 40 to 560 residues give contexts up to 2237 ids, fewer after merges."""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the first ids of one chain, one token a step: latency alone
        dict(name="attend_one", op="attend", B=1, N=1, lo=237, hi=237, Hq=8, Hkv=8, D=64, S=16, dtype="bf16", tree="chain"),
        # a batch of chains of 40 to 560 residues, four ids drafted in a row
        dict(name="attend_chains", op="attend", B=64, N=5, lo=157, hi=2237, Hq=16, Hkv=4, D=64, S=32, dtype="fp16", tree="chain"),
        # odd everything: ragged batch, empty prefix among them, pages of 48, heads of 80, one key head per query head
        dict(name="attend_odd", op="attend", B=7, N=27, lo=0, hi=4099, Hq=12, Hkv=12, D=80, S=48, dtype="bf16", tree="random"),
        # one long context (many chains as a prompt), a small tree
        dict(name="attend_long", op="attend", B=1, N=16, lo=131071, hi=131071, Hq=32, Hkv=8, D=128, S=64, dtype="bf16", tree="random"),
        # a serving batch with wide trees: the largest
        dict(name="attend_large", op="attend", B=32, N=64, lo=8192, hi=16384, Hq=32, Hkv=8, D=128, S=64, dtype="bf16", tree="random"),
        # one chain's drafts after 1000 merges (76 residue tokens, 15 glue bins)
        dict(name="verify_one", op="verify", B=1, N=5, V=1091, dtype="fp32", tree="chain", drafted=True, grammar=False),
        # trees over the 5000-merge vocabulary, the id ranges of the grammar
        dict(name="verify_tree", op="verify", B=48, N=40, V=5123, dtype="fp32", tree="random", drafted=True, grammar=True),
        # drafts without probabilities (looked up in earlier chains), 16-bit rows of odd length
        dict(name="verify_lookup", op="verify", B=16, N=64, V=50001, dtype="bf16", tree="random", drafted=False, grammar=False),
        # a large vocabulary and batch: the rows' bytes count
        dict(name="verify_large", op="verify", B=128, N=8, V=131072, dtype="fp32", tree="chain", drafted=True, grammar=False),
        # one chain, a small model's layers
        dict(name="commit_one", op="commit", L=6, B=1, N=5, lo=237, hi=237, Hkv=8, D=64, S=16, dtype="bf16"),
        # a serving batch, every layer at once
        dict(name="commit_large", op="commit", L=16, B=64, N=16, lo=0, hi=448, Hkv=8, D=128, S=32, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "verify", "verify", "commit"])
    if op == "verify":
        drafted = rng.random() < 0.7
        grammar = rng.random() < 0.4
        V = _log(rng, 500, 6000) if grammar else _log(rng, 500, 131072)
        N = _log(rng, 1, 64)
        B = min(_log(rng, 1, 128), max(1, (128 * 8 * 131072) // (N * V)))
        return dict(op=op, B=B, N=N, V=V, dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    tree=rng.choice(["chain", "random"]), drafted=drafted, grammar=grammar)
    Hkv = rng.choice([1, 2, 4, 8, 12])
    D = rng.choice([32, 64, 80, 96, 128])
    S = rng.choice([16, 24, 32, 64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "commit":
        L, B, N = rng.randint(1, 16), _log(rng, 1, 64), _log(rng, 1, 24)
        hi = _log(rng, 16, 448)
        return dict(op=op, L=L, B=B, N=N, lo=0, hi=hi, Hkv=min(Hkv, 8), D=D, S=S, dtype=dtype)
    G = rng.choice([1, 2, 4, 7, 8])
    N = _log(rng, 1, 64)
    hi = _log(rng, 16, 131072)
    most = 32 * 16384 * 8 * 128  # no more keys, and no more scores, than the largest listed case
    B = min(_log(rng, 1, 96), max(1, most // (hi * Hkv * D)), max(1, 32 * 16384 * 32 * 64 // (hi * Hkv * G * N)))
    return dict(op=op, B=B, N=N, lo=rng.choice([0, hi // 2, hi]), hi=hi, Hq=Hkv * G, Hkv=Hkv, D=D, S=S, dtype=dtype,
                tree=rng.choice(["chain", "random"]))


def _parents(case, seed):
    """[B, N]: a row of drafts, or a tree whose nodes hang on any earlier one, the nearer the likelier."""
    rng, N = random.Random(seed * 7919 + 1), case["N"]
    rows = []
    for _ in range(case["B"]):
        chain = case.get("tree", "chain") == "chain"
        rows.append([-1] + [i - 1 if chain else max(0, i - 1 - int(rng.random() ** 2 * i)) for i in range(1, N)])
    return rows


def _depths(parents):
    d = [0]
    for p in parents[1:]:
        d.append(d[p] + 1)
    return d


def _lens(case, seed):
    rng = random.Random(seed * 7919 + 2)
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def _ranges(V):
    """The ids of a vocabulary with five bins an angle: motifs, omega, phi, C:1N:1CA, by the place in the chain."""
    K = V - 15
    return [[0, K], [K + 5, K + 10], [K + 10, K + 15], [K, K + 5]]


def _pages(case, lens, gen, layers=()):
    """A paged cache whose sequences' pages lie in any order: values, block table, lengths."""
    B, S = case["B"], case["S"]
    M = (case["hi"] + case["N"] + S - 1) // S
    order = torch.randperm(B * M, device="cuda", generator=gen).to(torch.int32).view(B, M)
    shape = (*layers, B * M, S, case["Hkv"], case["D"])
    t = TYPES[case["dtype"]]
    k = torch.empty(shape, device="cuda", dtype=t).normal_(generator=gen)
    v = torch.empty(shape, device="cuda", dtype=t).normal_(generator=gen)
    return k, v, order, torch.tensor(lens, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, N, t = case["B"], case["N"], TYPES[case["dtype"]]
    st = {"op": case["op"]}
    if case["op"] != "commit":
        st["parents"] = torch.tensor(_parents(case, seed), device="cuda", dtype=torch.int32)
    if case["op"] == "attend":
        st["k_cache"], st["v_cache"], st["table"], st["lens"] = _pages(case, _lens(case, seed), gen)
        st["q"] = torch.empty(B, N, case["Hq"], case["D"], device="cuda", dtype=t).normal_(std=1.5, generator=gen)
        st["k"] = torch.empty(B, N, case["Hkv"], case["D"], device="cuda", dtype=t).normal_(generator=gen)
        st["v"] = torch.empty(B, N, case["Hkv"], case["D"], device="cuda", dtype=t).normal_(generator=gen)
    elif case["op"] == "verify":
        V = case["V"]
        st["u"] = torch.rand(B, N, device="cuda", generator=gen)
        st["ranges"] = st["start"] = None
        ok = None
        if case["grammar"]:
            st["ranges"] = torch.tensor(_ranges(V), device="cuda", dtype=torch.int32)
            st["start"] = torch.randint(0, 2237, (B,), device="cuda", generator=gen).to(torch.int32)
            depth = torch.tensor([_depths(p) for p in _parents(case, seed)], device="cuda")
            lo, hi = st["ranges"][(st["start"].long()[:, None] + depth) % 4].unbind(-1)
            x = torch.arange(V, device="cuda")
            ok = (x >= lo[..., None]) & (x < hi[..., None])
        # a sharp target and a draft that mostly agrees with it, each node's id drawn from its parent's draft row
        logits = torch.empty(B, N, V, device="cuda").normal_(std=2.5, generator=gen)
        near = logits + torch.empty_like(logits).normal_(std=0.5, generator=gen)
        if ok is not None:
            logits.masked_fill_(~ok, -math.inf)
            near.masked_fill_(~ok, -math.inf)
        st["target"] = torch.softmax(logits, -1).to(t)
        del logits
        q = torch.softmax(near, -1).to(t)
        del near
        up = st["parents"].long().clamp(min=0)
        at = q.double().cumsum(-1).gather(1, up[..., None].expand(B, N, V)) if B * N * V < 1 << 26 else None
        w = torch.rand(B, N, 1, device="cuda", generator=gen, dtype=torch.float64)
        ids = []
        for i in range(N):  # (row by row: the cumulative sums of the largest rows would not fit at once)
            c = at[:, i].contiguous() if at is not None else q[torch.arange(B, device="cuda"), up[:, i]].double().cumsum(-1)
            ids.append(torch.searchsorted(c, w[:, i] * c[:, -1:], right=True).clamp(max=V - 1)[:, 0])
        st["ids"] = torch.stack(ids, 1)
        st["draft"] = q if case["drafted"] else None
    else:
        shape = (case["L"], B, N, case["Hkv"], case["D"])
        st["k_cache"], st["v_cache"], st["table"], st["lens"] = _pages(case, _lens(case, seed), gen, (case["L"],))
        st["k"] = torch.empty(shape, device="cuda", dtype=t).normal_(generator=gen)
        st["v"] = torch.empty(shape, device="cuda", dtype=t).normal_(generator=gen)
        rng = random.Random(seed * 7919 + 3)
        n = [rng.randint(1, N) for _ in range(B)]
        path = [[0] + sorted(rng.sample(range(1, N), m - 1)) + [-1] * (N - m) for m in n]
        st["n"] = torch.tensor(n, device="cuda", dtype=torch.int32)
        st["path"] = torch.tensor(path, device="cuda", dtype=torch.int32)
    return st


# ---------------------------------------------------------------- plain forms
def _present(parents):
    """[B, N] nodes that hang on the root, and [B, N, N] truth of j being on the path from the root to i."""
    B, N = parents.shape
    on = torch.zeros(B, N, N, device=parents.device, dtype=torch.bool)
    row = torch.arange(B, device=parents.device)
    on[:, 0, 0] = parents[:, 0] == -1
    for i in range(1, N):
        p = parents[:, i].long()
        good = (p >= 0) & (p < i)
        up = on[row, p.clamp(0, N - 1)] & good[:, None]
        up[:, i] = up.any(1)
        on[:, i] = up
    return on.diagonal(dim1=1, dim2=2), on


def _attend(st):
    q, k, v = st["q"], st["k"], st["v"]
    B, N, Hq, D = q.shape
    Hkv = k.shape[2]
    here, on = _present(st["parents"])
    cap = st["table"].shape[1] * st["k_cache"].shape[1]
    table = st["table"].long()
    K = torch.cat([st["k_cache"][table].view(B, cap, Hkv, D), k], 1).float()
    V = torch.cat([st["v_cache"][table].view(B, cap, Hkv, D), v], 1).float()
    seen = torch.arange(cap, device=q.device)[None] < st["lens"][:, None]
    V = torch.where(torch.cat([seen, here], 1)[:, :, None, None], V, 0.0)
    mask = torch.cat([seen[:, None].expand(B, N, cap), on], 2)[:, None, :, None]  # [B, 1, N, 1, keys]
    rows = q.float().view(B, N, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    s = torch.matmul(rows, K.permute(0, 2, 3, 1)).mul_(D ** -0.5)
    del K
    s = s.view(B, Hkv, N, Hq // Hkv, -1).masked_fill_(~mask, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, Hkv, -1, s.shape[-1]), V.permute(0, 2, 1, 3)).view(B, Hkv, N, -1, D)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(B, N, Hq, D).to(q.dtype)


def _verify(st):
    target, draft, ids, parents, u = st["target"], st["draft"], st["ids"].long(), st["parents"], st["u"].double()
    B, N, V = target.shape
    dev = target.device
    row, x = torch.arange(B, device=dev), torch.arange(V, device=dev)
    here, _ = _present(parents)

    def probabilities(p, c, depth):  # a context's row: 64 bits, nothing but finite positive entries of its range
        p = p[row, c].double()
        good = (p > 0) & (p < math.inf)
        if st["ranges"] is not None:
            lo, hi = st["ranges"].long()[(st["start"].long() + depth) % st["ranges"].shape[0]].unbind(-1)
            good &= (x >= lo[:, None]) & (x < hi[:, None])
        return torch.where(good, p, 0.0)

    c = torch.zeros(B, device=dev, dtype=torch.long)
    depth = torch.zeros_like(c)
    n = here[:, 0].long()
    path = torch.full((B, N + 1), -1, device=dev, dtype=torch.long)
    tokens = torch.full((B, N + 1), -1, device=dev, dtype=torch.long)
    path[:, 0] = n - 1
    r = probabilities(target, c, depth)
    Z = torch.ones(B, device=dev, dtype=torch.float64)
    fresh = torch.ones(B, device=dev, dtype=torch.bool)
    for i in range(1, N):
        tried = here[:, i] & (parents[:, i].long() == c)
        good = (ids[:, i] >= 0) & (ids[:, i] < V)
        y = ids[:, i].clamp(0, V - 1)[:, None]
        if draft is None:
            q = ((x == y) & good[:, None]).double()
        else:
            q = probabilities(draft, c, depth)
        ry, qy = r.gather(1, y)[:, 0] * good, q.gather(1, y)[:, 0]
        if draft is None:
            qy = torch.ones_like(ry)
        yes = tried & (u[:, i] * qy * Z < ry)
        no = tried & ~yes
        left = (r - Z[:, None] * q).clamp(min=0)
        r = torch.where(no[:, None], left, r)
        Z = torch.where(no, left.sum(1), Z)
        fresh &= ~no
        path.scatter_(1, torch.where(yes, n, N)[:, None], torch.full_like(y, i))  # column N takes what is not kept
        tokens.scatter_(1, torch.where(yes, n - 1, N)[:, None], y)
        c = torch.where(yes, i, c)
        depth += yes
        n = n + yes
        r = torch.where(yes[:, None], probabilities(target, c, depth), r)
        Z = torch.where(yes, 1.0, Z)
        fresh |= yes
    r = torch.where((r.sum(1) > 0)[:, None], r, probabilities(target, c, depth))
    mass = r.cumsum(1)
    nxt = (mass <= u[:, :1] * mass[:, -1:]).sum(1)
    last = torch.where(r > 0, x, -1).amax(1)
    nxt = torch.minimum(nxt, last)
    col = torch.arange(N + 1, device=dev)[None]
    tokens = torch.where(col < (n - 1)[:, None], tokens, -1)
    tokens = torch.where((col == (n - 1)[:, None]) & (n > 0)[:, None], nxt[:, None], tokens)
    path = torch.where(col < n[:, None], path, -1)
    return n.to(torch.int32), path[:, :N].to(torch.int32), tokens[:, :N].to(torch.int32)


def _commit(st):
    L, B, N, Hkv, D = st["k"].shape
    S = st["k_cache"].shape[2]
    t = torch.arange(N, device=st["k"].device)[None]
    keep = t < st["n"][:, None]
    at = st["lens"].long()[:, None] + t
    page = st["table"].long().gather(1, (at // S).clamp(max=st["table"].shape[1] - 1))
    b = torch.arange(B, device=t.device)[:, None].expand(B, N)[keep]
    node, page, slot = st["path"].long()[keep], page[keep], (at % S)[keep]
    st["k_cache"][:, page, slot] = st["k"][:, b, node]
    st["v_cache"][:, page, slot] = st["v"][:, b, node]
    return st["k_cache"], st["v_cache"], st["lens"] + st["n"]


def run(state):
    if not own:
        return {"attend": _attend, "verify": _verify, "commit": _commit}[state["op"]](state)
    geobpe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pt-bpe_amd")
    if geobpe not in sys.path:
        sys.path.insert(0, geobpe)
    from geobpe import draft
    st = state
    if st["op"] == "attend":
        return draft.tree_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], st["k"], st["v"],
                                    st["parents"])
    if st["op"] == "verify":
        r = draft.verify(st["parents"], st["ids"], st["target"], st["draft"], st["u"], ranges=st["ranges"], start=st["start"])
        return r.n, r.path, r.tokens
    lens = draft.commit(st["k_cache"], st["v_cache"], st["table"], st["lens"], st["k"], st["v"], st["path"], st["n"])
    return st["k_cache"], st["v_cache"], lens


def work(case):
    B, N, e = case["B"], case["N"], TYPES[case["dtype"]].itemsize
    if case["op"] == "verify":
        # the ids, parents and numbers, an entry or two a node, and the row that the next id is drawn from
        rows = 2 if case["drafted"] else 1
        return {"bytes": B * (N * (8 + 4 + 4 + rows * e + 8) + rows * e * case["V"]), "flops": B * 4 * case["V"]}
    row = case["Hkv"] * case["D"] * e
    mean = (case["lo"] + case["hi"]) / 2
    if case["op"] == "commit":
        return {"bytes": int(case["L"] * B * (N + 1) / 2 * row * 4), "flops": 0}
    keys = B * (mean + N)
    return {"bytes": int(2 * keys * row + 2 * B * N * case["Hq"] * case["D"] * e),
            "flops": int(4 * keys * N * case["Hq"] * case["D"])}


# ---------------------------------------------------------------- results in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(st, _parents(case, seed), _lens(case, seed))
    if case["op"] == "verify":
        if case["B"] * case["N"] > 4096:
            return None
        return _exact_verify(st, _parents(case, seed), case)
    k, v, S = st["k_cache"], st["v_cache"], case["S"]
    table, path = st["table"].tolist(), st["path"].tolist()
    for b, (n, m) in enumerate(zip(st["n"].tolist(), _lens(case, seed))):
        for t in range(n):
            page, slot = table[b][(m + t) // S], (m + t) % S
            k[:, page, slot] = st["k"][:, b, path[b][t]]
            v[:, page, slot] = st["v"][:, b, path[b][t]]
    return k, v, st["lens"] + st["n"]


def _exact_attend(st, parents, lens):
    q, out = st["q"], torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64)
    B, N, Hq, D = q.shape
    G = Hq // st["k"].shape[2]
    for b in range(B):
        anc = torch.zeros(N, N, dtype=torch.float64)
        for i in range(N):
            j = i
            while j >= 0:
                anc[i, j] = 1
                j = parents[b][j]
        hidden = torch.where(anc > 0, 0.0, -math.inf).cuda()
        pages = st["table"][b].long()
        for h in range(Hq // G):
            old_k = st["k_cache"][pages][:, :, h].reshape(-1, D)[:lens[b]].double()
            old_v = st["v_cache"][pages][:, :, h].reshape(-1, D)[:lens[b]].double()
            new_k, new_v = st["k"][b, :, h].double(), st["v"][b, :, h].double()
            for g in range(h * G, h * G + G):
                x = q[b, :, g].double() / math.sqrt(D)
                s = torch.cat([x @ old_k.t(), x @ new_k.t() + hidden], 1)
                out[b, :, g] = torch.softmax(s, 1) @ torch.cat([old_v, new_v])
    return out


def _exact_verify(st, parents, case):
    ids, u = st["ids"].tolist(), st["u"].double().tolist()
    V, N = case["V"], case["N"]
    start = st["start"].tolist() if case["grammar"] else None
    n, paths, tokens = [], [], []
    for b in range(case["B"]):
        def row(rows, c, depth):
            p = rows[b, c].double()
            if start is None:
                return p
            lo, hi = _ranges(V)[(start[b] + depth) % 4]
            z = torch.zeros_like(p)
            z[lo:hi] = p[lo:hi]
            return z

        path, got = [0], []
        while True:
            rest, mass = row(st["target"], path[-1], len(got)), 1.0
            q = row(st["draft"], path[-1], len(got)) if case["drafted"] else None
            taken = None
            for i in range(path[-1] + 1, N):
                if parents[b][i] != path[-1]:
                    continue
                x = ids[b][i]
                chance = float(q[x]) if case["drafted"] else 1.0
                if u[b][i] * chance * mass < float(rest[x]):
                    taken = i
                    break
                if case["drafted"]:
                    rest = torch.relu(rest - mass * q)
                else:
                    rest[x] = 0
                mass = float(rest.sum())
            if taken is None:
                break
            path.append(taken)
            got.append(ids[b][taken])
        sums = torch.cumsum(rest, 0)
        got.append(int(torch.searchsorted(sums, sums[-1:] * u[b][0], right=True)))
        n.append(len(path))
        paths.append(path + [-1] * (N - len(path)))
        tokens.append(got + [-1] * (N - len(got)))
    return tuple(torch.tensor(z, device="cuda", dtype=torch.int32) for z in (n, paths, tokens))
