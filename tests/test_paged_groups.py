"""The paged attention's launch sizes, compiled for the host (no GPU)."""
import os
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "siliconed_amd", "csrc")
PROBE = r"""
#include "sq8_paged.hip"
#include <stdio.h>
int main() {
    sq8::PagedArgs p = {};
    while (scanf("%d %d %d %d %d %d %d", &p.batch, &p.q_heads, &p.kv_heads, &p.dim, &p.page, &p.max_pages, &p.window) == 7)
        printf("%d\n", sq8::paged_groups(p, 256));
}
"""


@pytest.fixture(scope="module")
def groups(tmp_path_factory):
    """(batch, q heads, kv heads, dim, page, most pages, window) → the workgroups of a launch on 256 CUs. Overflows of ints stop it."""
    from siliconed_amd.build import HIPCC
    d = tmp_path_factory.mktemp("paged_groups")
    src, exe = str(d / "probe.hip"), str(d / "probe")
    with open(src, "w") as f:
        f.write(PROBE)
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-ffunction-sections", "-ftrapv", "-fgpu-rdc",
                        "-I", CSRC, "-Wl,--gc-sections", src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def run(*case):
        out = subprocess.run([exe], input=" ".join(map(str, case)) + "\n", capture_output=True, text=True)
        assert out.returncode == 0, f"{case}: ended with {out.returncode}"
        return int(out.stdout)

    return run


def test_windows_past_the_table_change_nothing(groups):
    for case in ((2, 2, 1, 128, 16, 300), (1, 32, 8, 128, 64, 2048), (48, 40, 8, 64, 1, 100)):
        want = groups(*case, 0)
        assert want > 1
        for window in (2 ** 31 - 1, 2 ** 31 - 31, 2 ** 31 - 32, 2 ** 30):
            assert groups(*case, window) == want, window


def test_a_window_bounds_the_workgroups(groups):
    assert groups(1, 8, 1, 128, 16, 1000, 128) == 2  # 159 tokens at most: two tiles
    assert groups(1, 8, 1, 128, 16, 1000, 1) == 1
    assert groups(3, 8, 2, 128, 16, 0, 0) == 1
