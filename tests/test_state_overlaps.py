# SPDX-License-Identifier: MIT
"""What one call writes has to lie apart: pools and states given twice or
overlapping are refused, however they are interleaved otherwise. On the CPU."""

import os
import subprocess

import pytest
import torch

import beamgrad_amd as bg
from beamgrad_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ONES = torch.ones(4, dtype=torch.int32)


def table():
    return bg.PageTable.empty(4, 5, 20, device="cpu")


def pool_calls(pools):
    keep = torch.zeros(4, 2, dtype=torch.int32)
    yield lambda: bg.fork_pages(pools, table(), ONES)
    yield lambda: bg.keep_tokens(pools, table(), ONES, keep, ONES)
    yield lambda: bg.write_tokens(pools, [torch.zeros(4, 2, *p.shape[2:], dtype=p.dtype) for p in pools], table())


BUFFER = torch.zeros(20 * 8 * 64)


@pytest.mark.parametrize("pools, which", [
    ([BUFFER.view(20, 8, 64)] * 2, "0. and pools.1"),
    ([torch.zeros(20, 8, 4), BUFFER[:20 * 8 * 4].view(20, 8, 4), BUFFER[4:20 * 8 * 4 + 4].view(20, 8, 4)], "1. and pools.2"),
    ([BUFFER.view(20, 8, 64)[..., :33], BUFFER.view(20, 8, 64)[..., 32:]], "0. and pools.1"),
    ([BUFFER.view(20, 8, 2, 32)[:, :, 1], BUFFER.view(20, 8, 2, 32)[:, :, 0], BUFFER.view(20, 8, 4, 16)[:, :, 3]], "0. and pools.2"),
    ([BUFFER.view(20, 8, 64), BUFFER.view(torch.int32).view(20, 8, 64)[..., 5:6]], "0. and pools.1"),
    ([BUFFER.as_strided((20, 8, 4), (16, 4, 1))], "pages and tokens of pools.0"),
])
def test_pools_that_meet_are_refused(pools, which):
    for call in pool_calls(pools):
        with pytest.raises(ValueError, match=which):
            call()


@pytest.mark.parametrize("pools", [
    list(BUFFER.view(8, 20, 8, 8).unbind(0)),  # one after the other
    list(BUFFER.view(20, 8, 8, 8).unbind(1)),  # page by page
    list(BUFFER.view(20, 8, 8, 8).unbind(2)),  # token by token
    list(BUFFER.view(8, 8, 20, 8).permute(2, 1, 0, 3).unbind(2)),  # tokens ahead of pages
    list(BUFFER.view(8, 8, 20, 8).permute(2, 0, 1, 3).unbind(2)),
    [BUFFER.view(20, 8, 64)[..., 40:], BUFFER.view(20, 8, 64)[..., :33]],  # rows of unlike widths
    [BUFFER.view(20, 512)[:, :448].view(20, 8, 56), BUFFER.view(20, 512)[:, 448:].view(torch.float16).view(20, 8, 16)],
    [torch.zeros(20, 2, 8, 4)[:, i] for i in (0, 1)] + [BUFFER.view(40, 8, 32)[::2], BUFFER.view(40, 8, 32)[1::2]],
    [BUFFER[:20 * 16 * 16].view(20, 16, 16)[:, :8], BUFFER[:20 * 16 * 16].view(20, 16, 16)[:, 8:], torch.zeros(20, 8, 3)],
])
def test_pools_that_lie_apart_are_taken(pools):
    for call in pool_calls(pools):
        with pytest.raises(RuntimeError, match="runs on the GPU"):
            call()


def test_news_that_lie_in_a_pool_are_refused():
    pool, other = torch.zeros(20, 8, 4), torch.zeros(20, 8, 4)
    with pytest.raises(ValueError, match="news.1. and pools.0"):
        bg.write_tokens([pool, other], [torch.zeros(4, 2, 4), pool[:4, 3:5]], table())
    joint = torch.zeros(4, 2, 2, 4)
    for news in (joint.unbind(2), [joint[:, :, 0]] * 2, [joint[:, :, 0], torch.zeros(1, 1, 4).expand(4, 2, 4)]):
        with pytest.raises(RuntimeError, match="runs on the GPU"):
            bg.write_tokens([pool, other], list(news), table())


def test_states_that_meet_are_refused():
    parents = torch.zeros(2, 3, dtype=torch.int64)
    base = torch.zeros(100)
    state = base[:30].view(2, 3, 5)
    for states, which in (([state, state], "0. and states.1"), ([torch.zeros(2, 3), state, base[29:35].view(2, 3)], "1. and states.2"),
                          ([state, torch.zeros(2, 3, 0), base.view(torch.uint8)[119:125].view(2, 3)], "0. and states.2")):
        with pytest.raises(ValueError, match=which):
            bg.reorder_states(states, parents, inplace=True)
        with pytest.raises(RuntimeError, match="runs on the GPU"):
            bg.reorder_states(states, parents)  # only read
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        bg.reorder_states([base[30:36].view(2, 3), state, base[36:66].view(2, 3, 5)], parents, inplace=True)


PROBE = r"""
#include "regions.hpp"
#include <stdio.h>
#include <stdlib.h>
#include <map>
using namespace dbs_hip;
static uint32_t state = 12345;
static int draw(int n) { state = state * 1664525u + 1013904223u; return static_cast<int>((state >> 8) % n); }
int main() {
    int met = 0, none = 0;
    for (int round = 0; round < 200000; ++round) {
        // regions on a common grid, or of any strides
        const int n = 1 + draw(4), reads = draw(3);
        const int ts = 1 + draw(6), ps = draw(2) ? ts * (1 + draw(6)) : 1 + draw(20);
        std::vector<Region> w, r;
        for (int i = 0; i < n + reads; ++i) {
            Region x{static_cast<uintptr_t>(1000 + draw(60)), {1 + draw(4), 1 + draw(4)}, {draw(4) ? ps : draw(30), draw(4) ? ts : draw(8)}, 1 + draw(3)};
            if (draw(3) == 0) std::swap(x.stride[0], x.stride[1]);
            (i < n ? w : r).push_back(x);
        }
        const Meeting m = find_meeting(w, r);
        // byte by byte
        std::map<uintptr_t, int> owner;
        bool meet = false;
        for (int i = 0; i < n; ++i)
            for (int a = 0; a < w[i].n[0]; ++a)
                for (int b = 0; b < w[i].n[1]; ++b)
                    for (int c = 0; c < w[i].bytes; ++c) meet |= owner[w[i].base + a * w[i].stride[0] + b * w[i].stride[1] + c]++ > 0;
        for (const Region& x : r)
            for (int a = 0; a < x.n[0]; ++a)
                for (int b = 0; b < x.n[1]; ++b)
                    for (int c = 0; c < x.bytes; ++c) meet |= owner.count(x.base + a * x.stride[0] + b * x.stride[1] + c) > 0;
        const auto of = [](const std::vector<Region>& x) { return [&](int i) { return x[i]; }; };
        const bool apart = all_apart(n, of(w), reads, of(r));
        if (apart != (m.first < 0)) { printf("round %d: two answers\n", round); return 6; }
        if (m.first < 0 && meet) { printf("round %d: regions that meet are taken\n", round); return 1; }
        meet ? ++met : m.first < 0 ? ++none : 0;
    }
    if (met < 1000 || none < 1000) { printf("%d %d\n", met, none); return 2; }
    // what no address holds
    if (find_meeting({{16, {INT64_MAX, 2}, {INT64_MAX, 1}, 1}}, {}).first != 0) return 3;
    if (find_meeting({{UINTPTR_MAX - 3, {1, 1}, {0, 0}, 8}}, {}).first != 0) return 4;
    if (find_meeting({{16, {1, 1}, {0, 0}, 8}}, {{64, {INT64_MAX, 1}, {INT64_MAX, 1}, 1}}).first != 0) return 5;
    return 0;
}
"""


def test_regions_against_bytes(tmp_path):
    """Random grids: none that meet are taken for apart."""
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(PROBE)
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", f"-I{ROOT}/include", f"-I{ROOT}/beamgrad_amd/csrc", str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_c_entries_refuse_what_meets(tmp_path):
    """By a C program that launches nothing: the addresses are none of a device."""
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(r"""
#include <string.h>
#include "beamgrad_state.h"
int main(void) {
    static int32_t ints[64];
    static char memory[4096];
    void* base[2] = {memory, memory};
    int64_t row[2] = {16, 16}, page[2] = {64, 64}, token[2] = {16, 16}, strides[4] = {32, 16, 32, 16};
    BeamgradPools p = {base, row, page, token, 2, 4, 4, 0};
    BeamgradTable from = {ints, ints + 16, ints + 20}, to = {ints + 32, ints + 48, ints + 52};
    const void* news[2] = {memory + 2048, memory + 3200};
    if (beamgrad_fork_pages(&p, &from, ints, 0, 4, 4, &to, ints, 4096, 0) != 2) return 1;
    if (beamgrad_keep_tokens(&p, &from, ints, ints, ints, 4, 4, 1, &to, 0) != 2) return 2;
    if (beamgrad_write_tokens(&p, news, strides, ints, ints, 0, 4, 4, 2, 0) != 2) return 3;
    base[1] = memory + 1024;
    news[1] = memory + 1024 + 255;
    if (beamgrad_write_tokens(&p, news, strides, ints, ints, 0, 4, 4, 2, 0) != 2) return 4;
    const void* f[2] = {memory, memory};
    void* t[2] = {memory, memory};
    int64_t n[2] = {8, 8};
    if (beamgrad_reorder_states(f, t, n, 2, ints, 0, 2, 4, 0) != 2) return 5;      /* in place, twice */
    t[0] = memory + 1024, t[1] = memory + 1024 + 63;
    if (beamgrad_reorder_states(f, t, n, 2, ints, 0, 2, 4, 0) != 2) return 6;      /* written twice */
    t[1] = memory + 63;
    if (beamgrad_reorder_states(f, t, n, 2, ints, 0, 2, 4, 0) != 2) return 7;      /* read and written */
    if (beamgrad_reorder_states_backward(f, t, n, 2, 0, ints, 0, 2, 4, 0) != 2) return 8;
    return 0;
}
""")
    lib = os.path.dirname(_build.lib_path())
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), f"-L{lib}", "-ldbs_hip",
                    f"-Wl,-rpath,{lib}", f"-L{_build.ROCM}/lib", f"-Wl,-rpath,{_build.ROCM}/lib", "-lamdhip64", "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0
