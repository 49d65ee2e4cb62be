"""CPU tests of how a call behind a shared prefix is laid out: accepted sizes give a workspace, none ends the process."""
from __future__ import annotations

import math
import random
import subprocess
import sys

import pytest

from lynnreal_omni_b200 import _lib


def needed(*sizes):
    """lr_attention_shared_workspace_bytes(seqs, queries, own keys, prefix, heads, kv_heads, D)."""
    return _lib.load().lr_attention_shared_workspace_bytes(*sizes)


@pytest.mark.parametrize("kv_heads", [592, 593, 600, 4096, 65535])
@pytest.mark.parametrize("queries", [1, 10, 16, 17])
def test_many_key_heads(kv_heads, queries):
    """More key/value heads than the GPU has places for blocks. In a process of its own: it used to divide by zero."""
    code = ("import ctypes, sys\n"
            f"need = ctypes.CDLL({str(_lib.LIBRARY)!r}).lr_attention_shared_workspace_bytes\n"
            "need.restype, need.argtypes = ctypes.c_int64, [ctypes.c_int64] * 7\n"
            f"print(need(1, {queries}, 10, 100, {kv_heads}, {kv_heads}, 128))")
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0, (got.returncode, got.stderr)
    # at least the prefix's part and the own one of every row, at most one of each 64 keys of the prefix more
    row = queries * kv_heads * (128 + 2) * 4
    assert 2 * row <= int(got.stdout) <= 3 * row + 64


def test_too_many_rows_are_refused_before_anything_runs():
    """2^32 rows: no grid counts them. The pointers are never followed."""
    seqs, heads, lib = 1 << 20, 4096, _lib.load()
    need = needed(seqs, seqs, 0, 100, heads, heads, 64)
    operand = (4096, heads * 64, 64)
    status = lib.lr_attention_shared(*operand, *operand, *operand, *operand, *operand, 4096, 4096, seqs, seqs, 0, 100, heads, heads, 64, 1,
                                     0.125, 4096, 4096, need, None)
    assert status == _lib.LR_ERR_INVALID_ARGUMENT and b"rows" in lib.lr_last_error()


def room(seqs, tq, tk, prefix, h, hk, d):
    """A bound on the workspace: a few fp32 parts a row of queries, a quarter of the own keys and values, and what fills the GPU
    (148 blocks of 256 rows of the prefix's parts; the places of a wave for the own keys' of few sequences)."""
    row = (d + 2) * 4
    return row * (8 * tq * h + 2 ** 18 + 256 * hk) + int(0.26 * 4 * tk * hk * d)


def test_pieces_of_prompts_behind_long_own_keys():
    """Queries against longer own keys: the workspace stays below what the call reads and writes."""
    for sizes in ((1, 256, 8192, 8192, 32, 8, 128), (1, 128, 32768, 8192, 32, 8, 128), (1, 128, 131072, 512, 32, 8, 128),
                  (1, 147, 972915, 26, 32, 2, 128), (64, 64 * 80, 64 * 1080, 32768, 64, 8, 128), (16, 16 * 17, 16 * 4017, 32768, 64, 8, 128),
                  (512, 512 * 17, 512 * 4017, 32768, 64, 8, 128), (64, 64 * 8, 64 * 4096, 8192, 64, 8, 128), (1, 1, 1 << 23, 1000, 32, 8, 128)):
        seqs, tq, tk, prefix, h, hk, d = sizes
        assert needed(*sizes) <= (4 * tq * h * d + 4 * (tk + prefix) * hk * d) // 2, sizes


def test_workspaces_over_the_whole_range():
    rng = random.Random(7)

    def spread(high):
        return int(round(2 ** rng.uniform(0, math.log2(high))))

    for _ in range(20000):
        hk, group, d = spread(64), spread(128), rng.choice((64, 128))
        seqs, tq = spread(4096), spread(1 << 17)
        tk, prefix = rng.choice((0, spread(1 << 24))), spread(1 << 20)
        sizes = (seqs, tq, tk, prefix, hk * group, hk, d)
        assert needed(*sizes) <= room(*sizes), (sizes, needed(*sizes), room(*sizes))
