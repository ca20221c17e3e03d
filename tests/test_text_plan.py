"""The text decoder operators' launches (sq8_text_plan.hip), compiled for the host (no GPU): which kernel, tile and split a
block-scaled product takes, and how many workgroups a paged attention."""
import os
import subprocess

import pytest

from conftest import ROOT
from f8_shapes import FEW, LONG, VALUES

CSRC = os.path.join(ROOT, "siliconed_amd", "csrc")
PROBE = r"""
#include "sq8_text_plan.hip"
#include <stdio.h>
int main() {
    const char *const names[] = {"256", "128", "128 one", "64x128", "64", "short", "short wide", "far", "staged", "staged wide"};
    char what;
    while (scanf(" %c", &what) == 1) {
        if (what == 'a') {
            sq8::PagedArgs p = {};
            if (scanf("%d %d %d %d %d %d %d", &p.batch, &p.q_heads, &p.kv_heads, &p.dim, &p.page, &p.max_pages, &p.window) != 7) return 1;
            printf("%d\n", sq8::paged_groups(p, 256));
            continue;
        }
        sq8::F8Args p = {};
        int glu, f32, values;
        if (scanf("%d %d %d %d %d %d", &p.M, &p.K, &p.N, &glu, &f32, &values) != 6) return 1;
        static const uint16_t x = 0;
        p.H = glu ? p.N / 2 : p.N;
        p.KB = (p.K + 127) / 128;
        p.lda = p.ldw = p.ldx = p.K;
        p.ldsx = p.KB;
        if (values) p.x = &x;
        const sq8::F8Plan plan = sq8::f8_plan(p, glu != 0, f32 != 0, 256);
        printf("%s/%d\n", names[plan.kernel], plan.splits);
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    """The probe's answer, a line, to a line of numbers. An int that overflows ends it."""
    from siliconed_amd.build import HIPCC
    d = tmp_path_factory.mktemp("text_plan")
    src, exe = str(d / "probe.hip"), str(d / "probe")
    with open(src, "w") as f:
        f.write(PROBE)
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-ftrapv", "-ffunction-sections",
                        "-I", CSRC, "-Wl,--gc-sections", src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def run(*line):
        out = subprocess.run([exe], input=" ".join(map(str, line)) + "\n", capture_output=True, text=True)
        assert out.returncode == 0, f"{line}: ended with {out.returncode}"
        return out.stdout.strip()

    return run


@pytest.fixture(scope="module")
def plan(ask):
    """(M, K, N, GLU, fp32 out, values) → "kernel/parts of K" on 256 CUs."""
    return lambda m, k, n, glu=False, f32=False, values=False: ask("f", m, k, n, int(glu), int(f32), int(values))


@pytest.mark.parametrize("m,k,n,want", [(2100, 528, 4100, "256/1"), (1000, 656, 6100, "128/1"), (1000, 1040, 4000, "128 one/1"),
                                        (250, 400, 8100, "64x128/1"), (200, 272, 2500, "64/1"), (64, 12288, 4096, "64/4"),
                                        (48, 4096, 24576, "64x128/1"), (8192, 4096, 24576, "256/1")])
def test_tiles_of_many_rows(plan, m, k, n, want):
    assert plan(m, k, n) == want


def test_short_products(plan):
    assert plan(1, 4096, 6144) == "short wide/1" and plan(16, 4096, 4096) == "short/1"
    assert plan(1, 4096, 4096, values=True) == "staged/1" and plan(1, 4096, 6144, values=True) == "staged wide/1"
    assert plan(1, 16385, 4096, values=True) == "short/1" and plan(17, 128, 128, values=True) == "64/1"
    assert plan(4, 4096, 24576, glu=True, values=True) == "short/1"


def test_windows_past_the_table_change_nothing(ask):
    for case in ((2, 2, 1, 128, 16, 300), (1, 32, 8, 128, 64, 2048), (48, 40, 8, 64, 1, 100)):
        want = int(ask("a", *case, 0))
        assert want > 1
        for window in (2 ** 31 - 1, 2 ** 31 - 31, 2 ** 31 - 32, 2 ** 30):
            assert int(ask("a", *case, window)) == want, window


def test_a_window_bounds_the_workgroups(ask):
    assert ask("a", 1, 8, 1, 128, 16, 1000, 128) == "2"  # 159 tokens at most: two tiles
    assert ask("a", 1, 8, 1, 128, 16, 1000, 1) == "1"
    assert ask("a", 3, 8, 2, 128, 16, 0, 0) == "1"


def test_the_kernels_that_the_gpu_tests_are_for(plan):
    """The shapes of test_gpu_text_few_rows.py and test_gpu_text_long_k.py reach what they are named after."""
    for shape, want in FEW:
        assert plan(*shape) == plan(*shape, f32=True) == want, shape
    for shape, want in VALUES:
        assert plan(*shape, values=True) == plan(*shape, f32=True, values=True) == want, shape
    for shape, bf16, f32 in LONG:
        assert (plan(*shape), plan(*shape, f32=True)) == (bf16, f32), shape


def test_tall_products_sum_in_one_sequence(plan):
    """From 4096 rows on and past 1024 columns a product's rows have the same bits however they are chunked."""
    for n in (1025, 1500, 2048, 4098, 24576):
        for m in (4096, 4097, 5000, 8192, 20000):
            for k in (1024, 8192, 16384):
                for glu in (False, True)[:2 - n % 2]:
                    for f32 in (False, True):
                        assert plan(m, k, n, glu, f32).endswith("/1"), (m, k, n, glu, f32)
