"""Which tile a prompt's or chunk's attention takes and what it asks of the context (sq8_text_plan.hip), compiled for the host (no
GPU), and the new entries' checks that answer without one."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT
from siliconed_amd import _abi as abi

CSRC = os.path.join(ROOT, "siliconed_amd", "csrc")
PROBE = r"""
#include "sq8_text_plan.hip"
#include <stdio.h>
int main() {
    int paged, e4m3;
    sq8::AttendArgs p = {};
    while (scanf("%d %d %d %d %d %d %d %d %d", &paged, &e4m3, &p.tokens, &p.sequences, &p.kv_heads, &p.group, &p.dim, &p.page, &p.max_pages) == 9) {
        static const int32_t pages = 0;
        p.pages = paged ? &pages : nullptr;
        const sq8::AttendPlan plan = sq8::attend_plan(p, e4m3 != 0, 256);
        printf("%d %d %d %lld %lld %.0f\n", plan.rows, plan.narrow, plan.groups, (long long)plan.part_bytes, (long long)plan.marks, plan.tiles);
    }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    from siliconed_amd.build import HIPCC
    d = tmp_path_factory.mktemp("attend_plan")
    src, exe = str(d / "probe.hip"), str(d / "probe")
    with open(src, "w") as f:
        f.write(PROBE)
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-ftrapv", "-ffunction-sections",
                        "-I", CSRC, "-Wl,--gc-sections", src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def ask(tokens, sequences, *, kv=8, group=4, dim=128, page=0, most=0, e4m3=False):
        line = f"{int(page > 0)} {int(e4m3)} {tokens} {sequences} {kv} {group} {dim} {max(page, 1)} {most}\n"
        r = subprocess.run([exe], input=line, capture_output=True, text=True)
        assert r.returncode == 0
        rows, narrow, groups, part, marks, tiles = r.stdout.split()
        return int(rows), int(narrow), int(groups), int(part), int(marks), float(tiles)
    return ask


def test_prompts(plan):
    """Of long sequences tiles of 256 rows, else of 128, if they are as many as the card's 256 units; else of 64; heads of 256: 128."""
    assert plan(8192, 1)[:2] == (256, 0) and plan(4096, 1)[:2] == (256, 0) and plan(4095, 1)[:2] == (128, 0)
    assert plan(8192, 2)[:2] == (256, 0) and plan(8192, 3)[:2] == (128, 0) and plan(4096, 1, kv=1, group=1)[0] == 64
    assert plan(1000, 1)[0] == 128 and plan(900, 1)[0] == 64 and plan(700, 1)[0] == 64 and plan(1, 1)[0] == 64
    assert plan(8192, 1, dim=256)[0] == 128 and plan(5, 1, dim=200)[0] == 128
    assert plan(8192, 1)[2:5] == (8 * (32768 // 256 + 1), 0, 0)  # a workgroup a tile, nothing of the context
    assert plan(0, 3)[2] == 0 and plan(7, 0)[2] == 0


def test_chunks(plan):
    def chunk(new, sequences, length, **kw):
        return plan(new * sequences, sequences, page=16, most=-(-length // 16), **kw)[:2]
    assert chunk(1, 32, 8192) == (16, 1) and chunk(4, 32, 8192) == (16, 1)
    assert chunk(16, 32, 8192) == (64, 1) and chunk(16, 1, 500) == (16, 1) and chunk(8, 32, 8192) == (32, 1)
    assert chunk(64, 1, 8192) == (16, 1) and chunk(64, 8, 8192) == (256, 0) and chunk(2048, 1, 32768) == (256, 0)
    assert chunk(32, 32, 8192) == (128, 0) and chunk(32, 8, 8192) == (64, 1)
    assert chunk(64, 8, 16384, dim=256) == (128, 0) and chunk(8, 32, 8192, dim=256) == (32, 1)
    assert chunk(64, 8, 16384, dim=64, e4m3=True) == (128, 0) and chunk(64, 8, 16384, dim=64) == (256, 0)
    # Heads of 130 to 256 that are no multiple of 16 have no narrow tile.
    assert chunk(4, 32, 8192, dim=136) == (128, 0) and chunk(4, 32, 8192, dim=144) == (16, 1)


@pytest.mark.parametrize("new,sequences,length,dim", [(1, 1, 1, 64), (16, 1, 500, 128), (7, 33, 900, 256), (2048, 1, 32768, 128),
                                                      (64, 8, 8192, 128), (1, 4096, 131072, 128), (300, 5, 1 << 20, 64)])
def test_what_a_chunk_asks_of_the_context(plan, new, sequences, length, dim):
    """No more workgroups than the card holds, two slots of a tile's maxima, sums and outputs and a counter's line for each."""
    rows, narrow, groups, part, marks, tiles = plan(new * sequences, sequences, page=16, most=-(-length // 16), dim=dim)
    padded = 64 if dim <= 64 else 128 if dim <= 128 else 256
    assert 1 <= groups <= 4 * 256 and groups <= tiles
    assert part == 2 * groups * rows * (2 + padded) * 4 and marks % groups == 0 and marks >= groups


def test_the_most_tiles_are_counted_without_overflow(plan):
    assert plan(1 << 20, 1, page=1, most=(1 << 31) - 1)[5] > 2 ** 31
    assert plan(2 ** 31 - 1, 2 ** 31 - 1, page=2 ** 15, most=2 ** 31 - 1, kv=128, group=1)[5] > 2 ** 31
    assert plan(2 ** 31 - 1, 1, kv=1, group=1)[2] > 0


def test_null_contexts_are_refused():
    lib = abi.load()
    cache = ctypes.byref(abi.PagedCacheArgs())
    assert lib.sq8_norm_append_kv(None, None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, cache, None, None, None, 0, 0, 0, 0, None,
                                  None, 0.0, 1, 1) == abi.EINVAL
    assert lib.sq8_norm_rotate(None, None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, None, 0, 0, 0, 0, None, None, 0.0, 1, 1,
                               1, 64) == abi.EINVAL
    assert lib.sq8_prompt_attention(None, None, 0, 0, None, 0, 0, None, 0, 0, None, 1, 1.0, 0.0, 0, 1, None, 0, 0, 1, 1, 1,
                                    64) == abi.EINVAL
    assert lib.sq8_chunk_attention(None, None, 0, 0, cache, None, 0, 1, None, None, 1, 1.0, 0.0, 0, None, 0, 0, 1, 1) == abi.EINVAL
    assert lib.sq8_sample_tokens(None, None, 0, 0, None, None, None, None, None, None, None, 1, 1) == abi.EINVAL
