"""How the attention over pages cuts a sequence's keys over blocks: sizes of clusters that the device does not run are not chosen.  The rule is host code of the kernels' header,
compiled here with the library's compiler; no GPU."""
import os
import shutil
import subprocess

import pytest

from pygpukit_b200 import build

PROGRAM = r'''
#include <cstdio>
#include "paged.cuh"
int main() {
    // sequences, tiles, key heads, keys, tile, cost of the ends in tiles, then how many clusters of 1 ... 16 blocks run at once
    int n[6];
    while (scanf("%d %d %d %d %d %d", n, n + 1, n + 2, n + 3, n + 4, n + 5) == 6) {
        int at_once[17] = {};
        for (int i = 1; i <= 16; ++i) if (scanf("%d", at_once + i) != 1) return 1;
        pgk::PagedParams p = {};
        p.seqs = n[0]; p.tiles = n[1]; p.kv_heads = n[2]; p.max_keys = n[3];
        const pgk::PagedSplit s = pgk::paged_split(p, n[4], at_once, pgk::PAGED_CLUSTER, n[5]);
        printf("%d %d\n", s.splits, s.apart ? 1 : 0);
    }
}
'''


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    if not (os.path.exists(build.NVCC) or shutil.which(build.NVCC)):
        pytest.skip("no compiler")
    d = tmp_path_factory.mktemp("split")
    (d / "split.cu").write_text(PROGRAM)
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "-I", build.CSRC, str(d / "split.cu"), "-o", str(d / "split")], check=True, capture_output=True)

    def run(*calls):
        text = "\n".join(" ".join(map(str, (*call, *at_once))) for call, at_once in calls)
        out = subprocess.run([str(d / "split")], input=text, text=True, check=True, capture_output=True).stdout.split()
        return [(int(a), bool(int(b))) for a, b in zip(out[::2], out[1::2])]
    return run


FITS = [148, 74, 48, 36, 28, 24, 20, 17, 15, 14, 12, 11, 10, 9, 8, 8]


def test_sizes_that_do_not_run_are_not_chosen(split):
    one = (1, 1, 1, 2000, 128, 4)                      # one head of one sequence, 16 tiles: any cluster is one round
    upto8 = FITS[:8] + [0] * 8
    gaps = [n if i % 3 else 0 for i, n in enumerate(FITS)]
    gaps[0] = 148
    full, eight, gap, alone = split((one, FITS), (one, upto8), (one, gaps), (one, [148] + [0] * 15))
    assert full == (16, False) and eight == (8, False)
    assert gap == (8, False)                           # of 2, 3, 5, 6, 8, 9, 11, 12, 14, 15: two tiles a block from 8 to 15
    assert alone[1] and alone[0] > 1                   # blocks that leave their sums in memory need no cluster


def test_calls_that_fill_the_device_are_not_cut(split):
    assert split(((148, 1, 8, 4000, 128, 4), FITS), ((5, 1, 1, 0, 128, 4), FITS), ((1, 1, 1, 100, 128, 4), [0] * 16)) == [(1, False)] * 3
