"""Decoding over GeoBPE ids with drafted trees: the device operators between a model and
``BPE.dequantize`` / ``recover`` (the reference's sampler draws ids one by one, bin/train.py:715-716).

  tree_attention   attention of the tree's nodes over a paged cache and their own ancestors
  verify           the drafted ids against the target's probabilities, from given random numbers
  commit           the kept nodes' keys and values into the cache, every layer at once
  DraftCache       a paged cache with its lengths that calls the two cache operators

A tree has N <= 128 nodes.  Node 0 is the last decided token (its key and value are not in the cache
yet): ``parents[0] == -1``, anything else: the whole sequence is absent (a padded batch).  Node i > 0
hangs on the present node ``parents[i] < i``, else it is absent.  ``parents`` is int32, (N,) for one
tree or (batch, N).

The tensors are torch tensors of one device.  Calls are ordered on the current stream of that device,
wait for nothing, take their outputs from torch's allocator and can be captured.  There is no
CPU fallback and no backward: inputs that require gradients are refused unless gradients are off.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _native

MAX_NODES = 128
MAX_VOCAB = 1 << 22
MAX_POSITIONS = (1 << 31) - 64

_HALF = {torch.bfloat16: 0, torch.float16: 1}
_PROB = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ATTEND = struct.Struct("35qd")  # include/geobpe.h geobpe_attend_args
_VERIFY = struct.Struct("23q")   # geobpe_verify_args
_COMMIT = struct.Struct("35q")   # geobpe_commit_args


class Verified(NamedTuple):
    """n (batch,): kept nodes, the root included (0: an absent sequence); path (batch, N): their
    indices; tokens (batch, N): the n - 1 accepted ids, then the next id.  int32, -1 behind."""
    n: torch.Tensor
    path: torch.Tensor
    tokens: torch.Tensor


def _tensor(name, x, shape, dtypes, device):
    """x as an operand: its shape (None: any size), its type, its device."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: a torch tensor is expected, not {type(x).__name__}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name}: {x.dtype} is not one of {', '.join(map(str, dtypes))}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, not on {device}")
    if x.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, x.shape)):
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {tuple('any' if s is None else s for s in shape)}")


def _rows(name, x):
    """A tensor read in 16-byte pieces of its last dimension."""
    unit = 16 // x.element_size()
    st = x.stride()
    if st[-1] != 1 or x.data_ptr() % 16 or any(s % unit for s, n in zip(st[:-1], x.shape) if n > 1):
        raise ValueError(f"{name}: rows must be contiguous and 16-byte aligned (strides {st}, "
                         f"address {x.data_ptr() % 16} past 16 bytes): pass {name}.contiguous()")
    return [s if n > 1 else 0 for s, n in zip(st[:-1], x.shape)]


def _first(name, x):
    """The device of an operator's first operand: the others have to be there too."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: a torch tensor is expected, not {type(x).__name__}")
    return x.device


def _stream(device):
    if device.type != "cuda":
        raise ValueError(f"tensors on {device}: the decoding operators run on a HIP device only")
    return torch.cuda.current_stream(device).cuda_stream


def _no_grad(*xs):
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in xs):
        raise ValueError("the decoding operators have no backward: call them under torch.no_grad()")


def _parents(parents, B, N, device):
    _tensor("parents", parents, (N,) if isinstance(parents, torch.Tensor) and parents.dim() == 1 else (B, N),
            (torch.int32,), device)
    if N > 1 and parents.stride(-1) != 1:
        raise ValueError("parents: the nodes must be contiguous")
    return parents.stride(0) if parents.dim() == 2 else 0


def _nodes(N):
    if not 1 <= N <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, not {N}")


def _cache(k_cache, v_cache, table, lens, lead, dtypes, device):
    """The paged cache's checks; returns its page count, page size, table width."""
    shape = tuple(k_cache.shape) if isinstance(k_cache, torch.Tensor) else None
    _tensor("k_cache", k_cache, (*lead, None, None, None, None), dtypes, device)
    _tensor("v_cache", v_cache, shape, (k_cache.dtype,), device)
    B = lens.shape[0] if isinstance(lens, torch.Tensor) and lens.dim() == 1 else None
    _tensor("lens", lens, (B,), (torch.int32,), device)
    _tensor("block_table", table, (B, None), (torch.int32,), device)
    P, S, M = shape[-4], shape[-3], table.shape[1]
    if P < 1 or S < 1:
        raise ValueError("k_cache: a cache has at least one page of one position")
    if M * S > MAX_POSITIONS:
        raise ValueError(f"block_table: {M} pages of {S} positions are more than {MAX_POSITIONS}")
    if M > 1 and table.stride(1) != 1:
        raise ValueError("block_table: a sequence's pages must be contiguous")
    if B > 1 and lens.stride(0) != 1:
        raise ValueError("lens must be contiguous")
    return B, P, S, M


def _call(rc):
    if rc:
        msg = (_native.lib().geobpe_draft_error() or b"").decode()
        raise (ValueError if rc == _native.E_ARG else _native.GeoBPEError)(f"{msg} (code {rc})")


def tree_attention(q, k_cache, v_cache, block_table, lens, k, v, parents, scale: Optional[float] = None):
    """Attention of every node over the committed prefix and its own path in the tree.

    q (B, N, Hq, D), k and v (B, N, Hkv, D): the nodes' queries, keys and values, bfloat16 or float16, D a
    multiple of 8 up to 256, Hq a multiple of Hkv (query head h reads kv head h // (Hq // Hkv)).
    k_cache, v_cache (pages, page size, Hkv, D): position x of sequence b is slot x % page size of page
    block_table[b, x // page size]; lens (B,): its committed positions.  Other orders of the cache's
    dimensions are views with strides (16-byte aligned rows).  scale: D ** -0.5 if None.

    Returns (B, N, Hq, D).  Rows of absent nodes are 0 whatever their keys and values hold, and so does
    nothing outside a node's own path reach its row.  A length outside the table, or a page outside the cache
    among those needed, makes the sequence's present rows NaN."""
    dev = _first("q", q)
    _tensor("q", q, (None,) * 4, tuple(_HALF), dev)
    B, N, Hq, D = q.shape
    _nodes(N)
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"head dimension {D}: a multiple of 8 up to 256 is expected")
    nb, P, S, M = _cache(k_cache, v_cache, block_table, lens, (), (q.dtype,), dev)
    Hkv = k_cache.shape[2]
    if nb != B or k_cache.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)} does not fit {nb} sequences and heads of {k_cache.shape[3]}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads over {Hkv} key heads")
    _tensor("k", k, (B, N, Hkv, D), (q.dtype,), dev)
    _tensor("v", v, (B, N, Hkv, D), (q.dtype,), dev)
    ps = _parents(parents, B, N, dev)
    _no_grad(q, k_cache, v_cache, k, v)
    rows = [*_rows("q", q), *_rows("k", k), *_rows("v", v), *_rows("k_cache", k_cache), *_rows("v_cache", v_cache)]
    stream = _stream(dev)
    out = torch.empty((B, N, Hq, D), dtype=q.dtype, device=dev)
    args = _ATTEND.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        block_table.data_ptr(), lens.data_ptr(), parents.data_ptr(), *rows, block_table.stride(0), ps,
        B, N, Hq, Hkv, D, S, P, M,
        _HALF[q.dtype], D ** -0.5 if scale is None else float(scale))
    lib = _native.lib()
    need = lib.geobpe_tree_attention_work(args)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _call(lib.geobpe_tree_attention(dev.index, stream, args, work.data_ptr() if need > 0 else None, need))
    return out


def verify(parents, ids, target, draft, u, ranges=None, start=None) -> Verified:
    """Which drafted ids stand, and the next id: node by node from the root, the children of the last kept
    node in their order.  Child i with id x is kept when

        u[b, i] * draft[b, c, x] * Z < r(x),

    c the last kept node, r = target[b, c] and Z = 1 at first; a rejected one leaves r <- max(r - Z draft[b, c], 0),
    Z <- sum r.  When no child is kept, the next id is the first x whose cumulative r passes u[b, 0] * sum r; where
    r has no mass it is drawn from target[b, c], and it is -1 where that has none either.  The ids kept and drawn
    are distributed as the target's when every node's id was drawn from draft[b, parent] and u is uniform on [0, 1).

    ids (B, N) int32 or int64 (ids[:, 0] is not read; an id outside the vocabulary is rejected), target and draft
    (B, N, V) of one type (float32, bfloat16, float16; the rows are used as they are, entries that are not finite and
    positive count as 0), row i the distribution after node i; draft None: drafts without probabilities, draft(x)
    is 1 at the drafted id.  u (B, N) float32.
    ranges (C, 2) int32 and start (B,) int32: the token after node i is at place start[b] + depth(i), and outside
    ranges[place % C] = [lo, hi) a row's entries are taken as 0 and not read (``BPE.id_ranges``)."""
    dev = _first("target", target)
    _tensor("target", target, (None,) * 3, tuple(_PROB), dev)
    B, N, V = target.shape
    _nodes(N)
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"a vocabulary of {V}: 1 to {MAX_VOCAB} are expected")
    _tensor("ids", ids, (B, N), (torch.int64, torch.int32), dev)
    _tensor("u", u, (B, N), (torch.float32,), dev)
    if draft is not None:
        _tensor("draft", draft, (B, N, V), (target.dtype,), dev)
    ps = _parents(parents, B, N, dev)
    if (ranges is None) != (start is None):
        raise ValueError("ranges and start belong together")
    C = 0
    if ranges is not None:
        _tensor("ranges", ranges, (None, 2), (torch.int32,), dev)
        _tensor("start", start, (B,), (torch.int32,), dev)
        C = ranges.shape[0]
        if C < 1 or not ranges.is_contiguous() or not start.is_contiguous():
            raise ValueError("ranges and start must be contiguous and not empty")
    for name, x in (("ids", ids), ("u", u), ("target", target), ("draft", draft)):
        if x is not None and x.shape[-1] > 1 and x.stride(-1) != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
    _no_grad(target, draft)
    stream = _stream(dev)
    out = torch.empty((2 * N + 1, B), dtype=torch.int32, device=dev)
    n, path, tokens = out[0], out[1:N + 1].view(B, N), out[N + 1:].view(B, N)
    ts = target.stride()
    ds = draft.stride() if draft is not None else (0, 0)
    args = _VERIFY.pack(
        parents.data_ptr(), ids.data_ptr(), target.data_ptr(), draft.data_ptr() if draft is not None else 0,
        u.data_ptr(), ranges.data_ptr() if C else 0, start.data_ptr() if C else 0, n.data_ptr(), path.data_ptr(),
        tokens.data_ptr(), ts[0], ts[1], ds[0], ds[1], ps, ids.stride(0), u.stride(0), B, N, V, C,
        ids.dtype == torch.int64, _PROB[target.dtype])
    _call(_native.lib().geobpe_verify_draft(dev.index, stream, args))
    return Verified(n, path, tokens)


def commit(k_cache, v_cache, block_table, lens, k, v, path, n):
    """Node path[b, t] becomes position lens[b] + t of sequence b, t < n[b], in place; returns the new lengths
    lens + n (int32; lens itself stays as it is, for the other layers' calls).

    k_cache, v_cache (pages, page size, Hkv, D) and k, v (B, N, Hkv, D), or with a leading dimension of layers, of
    any type whose rows are multiples of 16 bytes; path (B, N) and n (B,) as ``verify`` returns them.  The table has
    to have the pages for the new positions.  A kept node outside the tree, the table or the cache is not written,
    and that sequence's new length is -1.  Pages that sequences share must not be among the written ones."""
    dev = _first("k_cache", k_cache)
    lead = (None,) if k_cache.dim() == 5 else ()
    B, P, S, M = _cache(k_cache, v_cache, block_table, lens, lead, (k_cache.dtype,), dev)
    Hkv, D = k_cache.shape[-2:]
    _tensor("path", path, (B, None), (torch.int32,), dev)
    N = path.shape[1]
    _nodes(N)
    lead = tuple(k_cache.shape[:-4])
    _tensor("k", k, (*lead, B, N, Hkv, D), (k_cache.dtype,), dev)
    _tensor("v", v, (*lead, B, N, Hkv, D), (k_cache.dtype,), dev)
    _tensor("n", n, (B,), (torch.int32,), dev)
    if (N > 1 and path.stride(1) != 1) or not n.is_contiguous():
        raise ValueError("path and n must be contiguous")
    e = k_cache.element_size()
    if Hkv < 1 or D < 1 or D * e % 16 or D * e > 65536:
        raise ValueError(f"heads of {D} x {e} bytes: a multiple of 16 bytes is expected")
    _no_grad(k_cache, v_cache, k, v)
    st = []
    for name, x in (("k", k), ("v", v), ("k_cache", k_cache), ("v_cache", v_cache)):
        s = [i * e for i in _rows(name, x)]
        st += s if len(s) == 4 else [0, *s]
    for name, x in (("k_cache", k_cache), ("v_cache", v_cache)):
        if any(s == 0 and m > 1 for s, m in zip(x.stride(), x.shape)):
            raise ValueError(f"{name} is expanded: its rows share memory")
    stream = _stream(dev)
    out = torch.empty(B, dtype=torch.int32, device=dev)
    args = _COMMIT.pack(
        k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), lens.data_ptr(),
        path.data_ptr(), n.data_ptr(), out.data_ptr(), *st, block_table.stride(0), path.stride(0),
        lead[0] if lead else 1, B, N, Hkv, D * e, S, P, M)
    _call(_native.lib().geobpe_commit_draft(dev.index, stream, args))
    return out


class DraftCache:
    """The keys and values of ``batch`` sequences of up to ``max_len`` committed positions, every layer's, in pages,
    with their lengths.  A model's step over a drafted tree is, per layer, ``attend`` and, once the ids are verified
    (``verify``, ``BPE.verify_draft``), one ``keep``; ``lens`` is a device tensor throughout."""

    def __init__(self, layers: int, batch: int, max_len: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
                 device="cuda", page_size: int = 64):
        if min(layers, batch, max_len, kv_heads, head_dim, page_size) < 1:
            raise ValueError("a cache has layers, sequences, positions, heads and pages")
        if dtype not in _HALF:
            raise TypeError(f"{dtype} is not one of {', '.join(map(str, _HALF))}")
        pages = -(-max_len // page_size)
        shape = (layers, batch * pages, page_size, kv_heads, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.block_table = torch.arange(batch * pages, dtype=torch.int32, device=device).view(batch, pages)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)

    def attend(self, layer: int, q, k, v, parents, scale: Optional[float] = None):
        """``tree_attention`` of one layer's nodes over what is kept so far."""
        return tree_attention(q, self.k[layer], self.v[layer], self.block_table, self.lens, k, v, parents, scale)

    def keep(self, k, v, verified: Verified):
        """The kept nodes of every layer, k and v (layers, B, N, Hkv, D), into the cache; the lengths grow."""
        self.lens.copy_(commit(self.k, self.v, self.block_table, self.lens, k, v, verified.path, verified.n))
