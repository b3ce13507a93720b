"""More of the decoding operators (geobpe.draft) against plain 64-bit implementations: rows held to id ranges that have
mass outside them, scales and scores at the ends of float32, long contexts with every tile visible, what autograd is told.

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
                        make_parents, make_verify, on, ref_attention, ref_verify, refuse, tree_paths, verify)

BF, FP = torch.bfloat16, torch.float16


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
