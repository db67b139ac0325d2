# SPDX-License-Identifier: MIT
"""The C entries of the cache's pages: a new table in the old one's place is refused.
By a C program that launches nothing."""

import os
import subprocess

from beamgrad_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_new_tables_in_the_place_of_old_ones(tmp_path):
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(r"""
#include "beamgrad_state.h"
static int32_t ints[200];
static char memory[4096];
int main(void) {
    void* base[1] = {memory};
    int64_t row[1] = {16}, page[1] = {64}, token[1] = {16};
    BeamgradPools p = {base, row, page, token, 1, 4, 4, 0};
    /* pages [4, 4], lengths [4], refs [4] */
    BeamgradTable from = {ints, ints + 16, ints + 20};
    int32_t* const old[3] = {ints, ints + 16, ints + 20};
    const int size[3] = {16, 4, 4};
    for (int field = 0; field < 3; ++field)
        for (int other = 0; other < 3; ++other)
            for (int end = 0; end < 2; ++end) {
                int32_t* new[3] = {ints + 100, ints + 116, ints + 120};
                /* its last entry is the other's first, or its first the other's last */
                new[field] = end ? old[other] + size[other] - 1 : old[other] - (size[field] - 1);
                if (new[field] < ints) new[field] = ints;
                BeamgradTable to = {new[0], new[1], new[2]};
                if (beamgrad_fork_pages(&p, &from, ints + 150, 0, 4, 4, &to, ints + 160, 4096, 0) != 2) return 1;
                if (beamgrad_extend_pages(&from, ints + 150, 4, 4, 4, 4, &to, ints + 160, 4096, 0) != 2) return 2;
                if (beamgrad_keep_tokens(&p, &from, ints + 150, ints + 154, ints + 158, 4, 4, 1, &to, 0) != 2) return 3;
            }
    /* the parts of the new table among each other */
    BeamgradTable to = {ints + 100, ints + 115, ints + 120};
    if (beamgrad_extend_pages(&from, ints + 150, 4, 4, 4, 4, &to, ints + 160, 4096, 0) != 2) return 4;
    return 0;
}
""")
    lib = os.path.dirname(_build.lib_path())
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), f"-L{lib}", "-ldbs_hip",
                    f"-Wl,-rpath,{lib}", f"-L{_build.ROCM}/lib", f"-Wl,-rpath,{_build.ROCM}/lib", "-lamdhip64", "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0


def test_tables_of_more_entries_than_ranks_hold(tmp_path):
    """2^30 entries are the most: the pages that all sequences want together are
    counted in 31 bits."""
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(r"""
#include "beamgrad_state.h"
static int32_t ints[64];
static char memory[64];
int main(void) {
    /* addresses as far apart as such tables are, none of which is touched */
    char* const far = (char*)0 + (1ll << 40);
    void* base[1] = {memory};
    int64_t row[1] = {16}, page[1] = {16}, token[1] = {16};
    BeamgradPools p = {base, row, page, token, 1, 4, 1, 0};
    BeamgradTable from = {(int32_t*)far, (int32_t*)(far + (1ll << 38)), ints};
    BeamgradTable to = {(int32_t*)(far + (1ll << 39)), (int32_t*)(far + (3ll << 38)), ints + 16};
    for (int log = 0; log <= 12; log += 6) {
        const int P = (1 << log) + 1, S = 1 << (30 - log);
        if (beamgrad_fork_pages(&p, &from, ints, 0, S, P, &to, ints, 1ll << 40, 0) != 2) return 1;
        if (beamgrad_extend_pages(&from, ints, S, P, 4, 1, &to, ints, 1 << 20, 0) != 2) return 2;
        if (beamgrad_keep_tokens(&p, &from, ints, ints, ints, S, P, 1, &to, 0) != 2) return 3;
    }
    return 0;
}
""")
    lib = os.path.dirname(_build.lib_path())
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), f"-L{lib}", "-ldbs_hip",
                    f"-Wl,-rpath,{lib}", f"-L{_build.ROCM}/lib", f"-Wl,-rpath,{_build.ROCM}/lib", "-lamdhip64", "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0


def test_large_tables_are_refused_by_name():
    import pytest
    import torch

    import beamgrad_amd as bg

    table = bg.PageTable(torch.empty(1, 1, dtype=torch.int32).expand(1 << 15, (1 << 15) + 1), torch.zeros(1 << 15, dtype=torch.int32),
                         torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="2\\*\\*30 entries"):
        bg.extend_pages(table, torch.zeros(1 << 15, dtype=torch.int32), 1)
