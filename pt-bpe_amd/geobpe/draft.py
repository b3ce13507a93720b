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
CPU fallback and no backward: inputs that require gradients are refused unless gradients are off, and so are
inputs with tangents (forward mode) outside inference mode.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native

MAX_NODES = 128
MAX_VOCAB = 1 << 22
MAX_POSITIONS = (1 << 31) - 4096

_HALF = (torch.bfloat16, torch.float16)
_bound = None


def _ops():
    """geobpe._draft (csrc/draft_py.cpp: the checks and the calls), bound to libgeobpe.so."""
    global _bound
    if _bound is None:
        import ctypes
        lib = _native.lib()
        try:
            from . import _draft
        except ImportError as e:
            raise _native.GeoBPEError(f"the decoding operators' extension (_draft.so) is not built: "
                                      f"geobpe.build.build_draft() ({e})")
        _draft.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in (
            "geobpe_tree_attention", "geobpe_tree_attention_work", "geobpe_verify_draft", "geobpe_commit_draft",
            "geobpe_draft_error")), _native.GeoBPEError)
        _bound = _draft
    return _bound


class Verified(NamedTuple):
    """n (batch,): kept nodes, the root included (0: an absent sequence); path (batch, N): their
    indices; tokens (batch, N): the n - 1 accepted ids, then the next id.  int32, -1 behind."""
    n: torch.Tensor
    path: torch.Tensor
    tokens: torch.Tensor


def tree_attention(q, k_cache, v_cache, block_table, lens, k, v, parents, scale: Optional[float] = None):
    """Attention of every node over the committed prefix and its own path in the tree.

    q (B, N, Hq, D), k and v (B, N, Hkv, D): the nodes' queries, keys and values, bfloat16 or float16, D a
    multiple of 8 up to 256, Hq a multiple of Hkv (query head h reads kv head h // (Hq // Hkv)).
    k_cache, v_cache (pages, page size, Hkv, D): position x of sequence b is slot x % page size of page
    block_table[b, x // page size]; lens (B,): its committed positions.  Other orders of the cache's
    dimensions are views with strides (16-byte aligned rows).  scale: D ** -0.5 if None, else a
    finite number up to 2e38 in size.  A call has at most
    2^23 - 1 query rows (B N Hq) and a table MAX_POSITIONS positions.  The work is cut for the table's positions, whatever
    the lengths: a table far longer than its sequences costs time (some 6 times at 16 times the length), so pass the part of
    it that can be in use (``block_table[:, :pages]``).

    Returns (B, N, Hq, D).  Rows of absent nodes are 0 whatever their keys and values hold, and so does
    nothing outside a node's own path reach its row.  A length outside the table, or a page outside the cache
    among those needed, makes the sequence's present rows NaN."""
    return (_bound or _ops()).tree_attention(q, k_cache, v_cache, block_table, lens, k, v, parents, scale)


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
    is 1 at the drafted id.  u (B, N) float32 (NaN keeps no child; beyond [0, 1) the next id is the first or last one with mass).
    ranges (C, 2) int32 and start (B,) int32: the token after node i is at place start[b] + depth(i), and the rows after it
    count as what they are inside ranges[place % C] = [lo, hi) (``BPE.id_ranges``), divided by their mass there (a mass
    that is 1 but for the type's rounding changes nothing): what lies outside is not read, and need not be 0.  So the ids kept and drawn are distributed as the target held to the range,
    whether the drafts were drawn from the whole row or inside the range: one outside is passed over, as is every child
    of a draft row without mass inside."""
    return Verified(*(_bound or _ops()).verify(parents, ids, target, draft, u, ranges, start))


def commit(k_cache, v_cache, block_table, lens, k, v, path, n):
    """Node path[b, t] becomes position lens[b] + t of sequence b, t < n[b], in place; returns the new lengths
    lens + n (int32; lens itself stays as it is, for the other layers' calls).

    k_cache, v_cache (pages, page size, Hkv, D) and k, v (B, N, Hkv, D), or with a leading dimension of layers, of
    any type whose rows are multiples of 16 bytes; path (B, N) and n (B,) as ``verify`` returns them.  The table has
    to have the pages for the new positions.  A kept node outside the tree, the table or the cache is not written,
    and that sequence's new length is -1.  Pages that sequences share must not be among the written ones, k and v not lie
    in the cache's own memory; a cache for both keys and values, or one whose rows overlap, is refused."""
    return (_bound or _ops()).commit(k_cache, v_cache, block_table, lens, k, v, path, n)


class DraftCache:
    """The keys and values of ``batch`` sequences of up to ``max_len`` committed positions, every layer's, in pages,
    with their lengths.  A model's step over a drafted tree is, per layer, ``attend`` and, once the ids are verified
    (``verify``, ``BPE.verify_draft``), one ``keep``; ``lens`` is a device tensor throughout.  A prompt goes in as chains of
    up to MAX_NODES nodes, each kept whole: ``keep(k, v, Verified(n, path, None))``, path[b] = 0, 1, ..., n[b] its nodes."""

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
