# SPDX-License-Identifier: MIT
"""Workspaces of attention over a paged cache, by a C program that launches
nothing: what they may grow to, and sizes that no launch takes."""

import os
import subprocess

from beamgrad_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROBE = r"""
#include <stdio.h>
#include <string.h>
#include "beamgrad_state.h"
static int32_t shared[4096];
static int64_t bytes(int type, int groups, int beams, int tokens, int heads, int kv_heads, int dim) {
    BeamgradAttention a; memset(&a, 0, sizeof a);
    a.data_type = type; a.sequences = groups * beams; a.tokens = tokens; a.heads = heads; a.kv_heads = kv_heads; a.head_dim = dim;
    a.beams = beams; a.page_tokens = 16; a.n_pages = 100000; a.table_pages = 8000; a.scale = 0.125f;
    a.shared = beams > 1 ? shared : 0;
    return beamgrad_tree_attention_workspace_size(&a);
}
#define AT_MOST(mb, n) do { const int64_t got = n; if (got <= 0 || got > (int64_t)(mb) << 20) { printf("%s: %lld\n", #n, (long long)got); return 1; } } while (0)
int main(void) {
    /* two results of 128 rows (float32 in 32 bits: 64) for each of 512 workgroups */
    AT_MOST(100, bytes(2, 1, 1, 100000, 32, 8, 128));
    AT_MOST(100, bytes(2, 16, 16, 64, 64, 8, 128));
    AT_MOST(100, bytes(2, 4, 8, 4000, 64, 8, 128));
    AT_MOST(100, bytes(2, 32, 8, 4000, 64, 8, 128));
    AT_MOST(100, bytes(0, 32, 8, 500, 64, 8, 128));
    /* groups that share: 256 MB and those of the workgroups */
    AT_MOST(400, bytes(2, 200, 16, 5, 64, 8, 256));
    AT_MOST(400, bytes(1, 16, 16, 12, 64, 8, 256));
    AT_MOST(400, bytes(0, 16, 16, 33, 64, 32, 256));
    /* sizes of no launch: refused, and in finite time */
    if (bytes(2, 256, 1, 1, 4000000, 4000000, 8) <= 0) return 2; /* several launches of fewer sequences */
    if (bytes(2, 1, 1, 1, 40000000, 40000000, 8) != -1) return 3;
    if (bytes(2, 4, 2, 1, 16000000, 16000000, 8) != -1) return 4;
    if (bytes(2, 1, 1, 30000000, 32, 1, 64) <= 0) return 5;
    return 0;
}
"""


def test_sizes(tmp_path):
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(PROBE)
    lib = os.path.dirname(_build.lib_path())
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), f"-L{lib}", "-ldbs_hip",
                    f"-Wl,-rpath,{lib}", f"-L{_build.ROCM}/lib", f"-Wl,-rpath,{_build.ROCM}/lib", "-lamdhip64", "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=20)
    assert done.returncode == 0, done.stdout
