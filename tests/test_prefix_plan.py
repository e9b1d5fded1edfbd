"""How a shared prefix is cut into pieces (csrc/prefix_plan.h), built for the CPU."""

import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-practice_amd", "csrc")

HEADS = [(16, 8), (32, 8), (64, 8), (16, 16), (8, 1), (6, 2), (12, 4), (40, 1)]
SEQS = [1, 3, 8, 13, 32, 33, 54, 56, 64, 65, 100, 128, 129, 192, 200, 256, 300, 1000, 65535]


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(
        '#include "prefix_plan.h"\n'
        'extern "C" void plan(int b, int h, int kvh, int group, int rows, int keys, int tail, int cus, int* out) {\n'
        "    const femto::PrefixPieces p = femto::prefix_pieces(b, h, kvh, group, rows, keys, tail, cus);\n"
        "    out[0] = p.pieces; out[1] = p.piece_keys; out[2] = p.longest;\n}\n")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "plan.cpp"), "-o",
                    str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    out = (ctypes.c_int * 3)()

    def call(seqs, heads, kv_heads, keys, tail=512, cus=256):
        """(pieces, keys of a piece, the tiles are the longest work)"""
        n_rep = heads // kv_heads
        group = next(g for g in (4, 2, 1) if n_rep % g == 0)
        lib.plan(seqs, heads, kv_heads, group, 32 * (4 // group), keys, tail, cus, out)
        return out[0], out[1], bool(out[2])

    return call


@pytest.mark.parametrize("heads", HEADS)
def test_pieces_are_one_even_cut(plan, heads):
    """Every key of a prefix is in one of its pieces, none of them is empty, and the cut is the even one: ceil(tiles /
    pieces) key tiles each, so whoever cuts a prefix evenly and whoever counts a context's pieces by piece_keys agree."""
    for seqs in SEQS:
        for pages in range(1, 1025):
            keys = 16 * pages
            pieces, piece_keys, _ = plan(seqs, *heads, keys)
            where = (seqs, heads, keys, pieces, piece_keys)
            assert 1 <= pieces <= 64 and piece_keys > 0 and piece_keys % 64 == 0, where
            assert (pieces - 1) * piece_keys < keys <= pieces * piece_keys, where
            tiles = -(-keys // 64)
            assert piece_keys == 64 * -(-tiles // pieces), where


def test_without_a_prefix(plan):
    assert plan(8, 16, 8, 0) == (0, 0, False)


def test_largest_prefix(plan):
    pieces, piece_keys, _ = plan(65535, 64, 8, 1 << 30)
    assert (pieces - 1) * piece_keys < 1 << 30 <= pieces * piece_keys and pieces <= 64


# (sequences, heads, KV heads, prefix, longest tail): measured with and without the tiles' waves ahead, the faster one.
AHEAD = [
    ((256, 32, 8, 16384, 1024), True), ((256, 32, 8, 16384, 1365), True), ((256, 32, 8, 16384, 1638), False),
    ((256, 32, 8, 16384, 4096), False), ((128, 32, 8, 16384, 1170), True), ((128, 32, 8, 16384, 1638), False),
    ((256, 16, 8, 16384, 1024), False), ((256, 16, 8, 16384, 819), False), ((256, 16, 8, 16384, 256), True),
    ((128, 16, 8, 16384, 819), False), ((128, 16, 8, 16384, 256), True), ((256, 16, 8, 8192, 512), False),
    ((256, 64, 8, 16384, 2048), True), ((256, 64, 8, 16384, 4096), False), ((128, 64, 8, 8192, 1024), True),
    ((64, 32, 8, 16384, 819), True), ((64, 32, 8, 16384, 2048), False),
]


@pytest.mark.parametrize("shape,ahead", AHEAD)
def test_tiles_ahead(plan, shape, ahead):
    assert plan(*shape)[2] == ahead


def test_short_chains_are_never_ahead(plan):
    for seqs in (1, 8, 64, 256):
        for keys in range(16, 1024, 48):
            pieces, piece_keys, ahead = plan(seqs, 16, 8, keys, 1)
            assert not (ahead and piece_keys < 5 * 64)
