"""Index arithmetic of the decode operators on the CPU: pcp_b200/csrc/decode_index.h compiled by the host compiler and run over good
and bad lengths, pages and parents, and over the split of tiles into equal shares."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = r'''
#include "decode_index.h"
using namespace pcpb;
extern "C" {
void t_clip_seq(int lo, int hi, int ctx, int rows, int nodes, int top, int* o) { SeqLen s = clip_seq(lo, hi, ctx, rows, nodes, top); o[0] = s.n0; o[1] = s.n; o[2] = s.ctx; o[3] = s.bad; }
int t_clip_parent(int p, int i, int* bad) { return clip_parent(p, i, bad); }
int t_clip_page(int p, int n) { return clip_page(p, n); }
long long t_page_row(int p, long long st, int h, int pt, int off, int w) { return page_row(p, st, h, pt, off, w); }
long long t_share(long long total, int blocks) { return tile_share(total, blocks); }
void t_parts(long long first, int count, long long share, int* o) { Parts p = parts_of(first, count, share); o[0] = p.c0; o[1] = p.c1; o[2] = p.slot0; }
}
'''


@pytest.fixture(scope="module")
def idx(tmp_path_factory):
    d = tmp_path_factory.mktemp("idx")
    (d / "t.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-I", os.path.join(ROOT, "pcp_b200", "csrc"), str(d / "t.cpp"), "-o", str(d / "t.so")], check=True)
    lib = C.CDLL(str(d / "t.so"))
    lib.t_page_row.argtypes = [C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_int]
    lib.t_page_row.restype = lib.t_share.restype = C.c_longlong
    lib.t_share.argtypes = [C.c_longlong, C.c_int]
    lib.t_parts.argtypes = [C.c_longlong, C.c_int, C.c_longlong, C.c_void_p]
    return lib


EDGE = [-2 ** 31, -5, -1, 0, 1, 7, 8, 9, 64, 255, 256, 257, 10 ** 6, 2 ** 31 - 1]


def test_lengths_are_clipped_into_what_there_is(idx):
    o = (C.c_int * 4)()
    for rows in (1, 8, 64):
        for nodes in (1, 7, 256):
            for top in (16, 10 ** 6):
                for lo in EDGE:
                    for hi in EDGE:
                        for ctx in EDGE:
                            idx.t_clip_seq(lo, hi, ctx, rows, nodes, top, o)
                            n0, n, c, bad = o
                            assert 0 <= n0 <= rows and 0 <= n <= nodes and n0 + n <= rows and 0 <= c <= top
                            good = 0 <= lo <= hi <= rows and hi - lo <= nodes and 0 <= ctx <= top
                            assert bool(bad) == (not good)
                            if good:
                                assert (n0, n, c) == (lo, hi - lo, ctx)


def test_parents_and_pages(idx):
    bad = C.c_int(0)
    for i in (0, 1, 5, 255):
        for p in EDGE:
            bad.value = 0
            got = idx.t_clip_parent(p, i, C.byref(bad))
            assert got == (p if -1 <= p < i else -1) and bool(bad.value) == (not -1 <= p < i)
    for n in (1, 8, 2 ** 31 - 1):
        for p in EDGE:
            assert idx.t_clip_page(p, n) == (p if 0 <= p < n else -1)


def test_offsets_pass_32_bits(idx):
    assert idx.t_page_row(2 ** 31 - 2, 8 * 16 * 128, 7, 16, 15, 128) == (2 ** 31 - 2) * 16384 + (7 * 16 + 15) * 128


@pytest.mark.parametrize("seed", range(8))
def test_every_tile_belongs_to_one_block_and_its_part_is_found(idx, seed):
    """The loop of the attention kernels (segment by segment, a part goes to slot 0 if the block begins with it, else to slot 1) against the
    lookup of the kernel that joins the parts."""
    r = random.Random(seed)
    for _ in range(40):
        blocks = r.choice([1, 2, 7, 148, 296])
        items = [r.choice([1, 1, 2, 5, 33, 400]) for _ in range(r.randrange(1, 60))]
        first = [sum(items[:i]) for i in range(len(items))]
        total = sum(items)
        share = idx.t_share(total, blocks)
        held, finished = {}, {}
        for c in range(blocks):
            w, w1 = share * c, min(total, share * (c + 1))
            w0, used = w, set()
            while w < w1:
                i = max(k for k in range(len(items)) if first[k] <= w)
                t0, t1 = w - first[i], min(items[i], w - first[i] + (w1 - w))
                if t0 == 0 and t1 == items[i]:
                    finished[i] = c
                else:
                    slot = 2 * c + (0 if w == w0 else 1)
                    assert slot not in used
                    used.add(slot)
                    held.setdefault(i, []).append((slot, t1 - t0))
                w += t1 - t0
        o = (C.c_int * 3)()
        for i, n in enumerate(items):
            idx.t_parts(first[i], n, share, o)
            c0, c1, slot0 = o
            if c0 == c1:
                assert finished[i] == c0 and i not in held
            else:
                assert [s for s, _ in held[i]] == [slot0 if c == c0 else 2 * c for c in range(c0, c1 + 1)]
                assert sum(k for _, k in held[i]) == n and i not in finished
