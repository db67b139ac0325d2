# SPDX-License-Identifier: MIT
"""CPU checks of the operators of a model's state: what they refuse, and the
arithmetic that says where a token lies."""

import os
import subprocess

import pytest
import torch

import beamgrad_amd as bg
from beamgrad_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def table(S=4, P=5, n_pages=20):
    return bg.PageTable.empty(S, P, n_pages, device="cpu")


def attend(S=4, N=3, H=4, Hkv=2, D=16, page=8, dtype=torch.float32, **more):
    args = dict(q=torch.zeros(S, N, H, D, dtype=dtype), k=torch.zeros(20, page, Hkv, D, dtype=dtype),
                v=torch.zeros(20, page, Hkv, D, dtype=dtype), table=table(S))
    args.update(more)
    q, k, v, t = (args.pop(n) for n in ("q", "k", "v", "table"))
    return bg.tree_attention(q, k, v, t, **args)


def test_accepted_calls_need_the_gpu():
    pools = [torch.zeros(20, 8, 4)]
    ones = torch.ones(4, dtype=torch.int32)
    for call in (lambda: attend(), lambda: attend(beams=2, shared=torch.zeros(2, dtype=torch.int64), return_lse=True),
                 lambda: attend(parents=torch.zeros(4, 3, dtype=torch.int32), counts=ones, scale=0.5),
                 lambda: bg.fork_pages(pools, table(), ones), lambda: bg.extend_pages(table(), ones, 8),
                 lambda: bg.write_tokens(pools, [torch.zeros(4, 2, 4)], table(), ones),
                 lambda: bg.keep_tokens(pools, table(), ones, torch.zeros(4, 2, dtype=torch.int32), ones),
                 lambda: bg.reorder_states([torch.zeros(2, 3, 5)], torch.zeros(2, 3, dtype=torch.int64)),
                 lambda: bg.reorder_states([torch.zeros(2, 3, 5)], torch.zeros(2, 3, dtype=torch.int64), inplace=True)):
        with pytest.raises(RuntimeError, match="runs on the GPU"):
            call()


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(4, 3, 4)), "q must be a"),
    (dict(q=torch.zeros(4, 0, 4, 16)), "q must be a"),
    (dict(q=torch.zeros(4, 3, 4, 16, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (dict(k=torch.zeros(20, 8, 2, 16, dtype=torch.float16)), "one type"),
    (dict(v=torch.zeros(20, 8, 1, 16)), "of one shape"),
    (dict(q=torch.zeros(5, 3, 4, 16)), "5 sequences, the page table 4"),
    (dict(q=torch.zeros(4, 3, 3, 16)), "multiple of the cache's 2"),
    (dict(q=torch.zeros(4, 3, 4, 12), k=torch.zeros(20, 8, 2, 12), v=torch.zeros(20, 8, 2, 12)), "multiple of 8"),
    (dict(q=torch.zeros(4, 3, 4, 264), k=torch.zeros(20, 8, 2, 264), v=torch.zeros(20, 8, 2, 264)), "multiple of 8 up to 256"),
    (dict(q=torch.zeros(4, 3, 4, 24)), "width must be one"),
    (dict(counts=torch.ones(3, dtype=torch.int32)), "counts must be"),
    (dict(counts=torch.ones(4)), "counts must be"),
    (dict(parents=torch.zeros(4, 2, dtype=torch.int32)), "parents must be"),
    (dict(q=torch.zeros(4, 513, 4, 16), parents=torch.zeros(4, 513, dtype=torch.int32)), "at most 512"),
    (dict(beams=3), "beams must divide"),
    (dict(beams=0), "beams must divide"),
    (dict(beams=2, shared=torch.zeros(4, dtype=torch.int32)), "shared must be"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=-1.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(scale=1e300), "scale must be positive"),
    (dict(k=torch.zeros(20, 8, 16, 2).transpose(2, 3)), "rows must be contiguous"),
    (dict(k=torch.zeros(20 * 8 * 2 * 16 + 1)[1:].view(20, 8, 2, 16)), "multiples of 16 bytes"),
    (dict(v=torch.zeros(20, 8, 2, 17)[..., :16]), "multiples of 16 bytes"),
    (dict(table=bg.PageTable(torch.zeros(4, 5, dtype=torch.int64), *table()[1:])), "pages must be a contiguous int32"),
    (dict(table=bg.PageTable(torch.zeros(4, 10, dtype=torch.int32)[:, ::2], *table()[1:])), "pages must be a contiguous int32"),
    (dict(table=bg.PageTable(table()[0], torch.zeros(3, dtype=torch.int32), table()[2])), "lengths must be"),
    (dict(table=bg.PageTable(torch.zeros(1, 1, dtype=torch.int32).expand(4, 5), *table()[1:])), "pages must be a contiguous"),
])
def test_attention_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        attend(**change)


def test_types_and_gradients_are_refused():
    with pytest.raises(TypeError, match="PageTable"):
        attend(table=tuple(table()))
    with pytest.raises(TypeError, match="q must be a torch.Tensor"):
        attend(q=[1.0])
    with pytest.raises(RuntimeError, match="no gradient"):
        attend(q=torch.zeros(4, 3, 4, 16, requires_grad=True))
    pools = [torch.zeros(20, 8, 4, requires_grad=True)]
    ones = torch.ones(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no gradient"):
        bg.fork_pages(pools, table(), ones)
    with pytest.raises(RuntimeError, match="no gradient"):
        bg.write_tokens([pools[0].detach()], [torch.zeros(4, 2, 4, requires_grad=True)], table())
    with pytest.raises(RuntimeError, match="no gradient"):
        bg.reorder_states([torch.zeros(2, 3, requires_grad=True)], torch.zeros(2, 3, dtype=torch.int64), inplace=True)
    with pytest.raises(TypeError, match="float32, float16 and bfloat16"):
        bg.reorder_states([torch.zeros(2, 3, dtype=torch.float64, requires_grad=True)], torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(TypeError, match="a list in it"):
        bg.reorder_states([[0.0]], torch.zeros(2, 3, dtype=torch.int64))


@pytest.mark.parametrize("pools, parents, message", [
    ([], torch.ones(4, dtype=torch.int32), "at least one pool"),
    ([torch.zeros(20, 8)], torch.ones(4, dtype=torch.int32), "must be a"),
    ([torch.zeros(19, 8, 4)], torch.ones(4, dtype=torch.int32), "must have 20 pages"),
    ([torch.zeros(20, 8, 4), torch.zeros(20, 7, 4)], torch.ones(4, dtype=torch.int32), "pages of 8 tokens"),
    ([torch.zeros(20, 8, 4, 4).transpose(2, 3)], torch.ones(4, dtype=torch.int32), "row of pools"),
    ([torch.zeros(1, 8, 4).expand(20, 8, 4)], torch.ones(4, dtype=torch.int32), "overlap"),
    ([torch.zeros(20, 1, 4).expand(20, 8, 4)], torch.ones(4, dtype=torch.int32), "overlap"),
    ([torch.zeros(20, 8, 4)], torch.ones(4), "parents must be"),
    ([torch.zeros(20, 8, 4)], torch.ones(2, 2, dtype=torch.int32), "parents must be"),
])
def test_fork_refusals(pools, parents, message):
    with pytest.raises(ValueError, match=message):
        bg.fork_pages(pools, table(), parents)


def test_page_refusals():
    ones = torch.ones(4, dtype=torch.int32)
    pools = [torch.zeros(20, 8, 4)]
    with pytest.raises(ValueError, match="counts must be"):
        bg.extend_pages(table(), torch.ones(5, dtype=torch.int32), 8)
    with pytest.raises(ValueError, match="at least one token"):
        bg.extend_pages(table(), ones, 0)
    with pytest.raises(ValueError, match="fewer than 2"):
        bg.extend_pages(table(), ones, 1 << 29)
    with pytest.raises(ValueError, match="refs must be"):
        bg.extend_pages(table()._replace(refs=torch.zeros(20)), ones, 8)
    with pytest.raises(ValueError, match="as many"):
        bg.write_tokens(pools, [], table())
    with pytest.raises(ValueError, match="with the row of pools"):
        bg.write_tokens(pools, [torch.zeros(4, 2, 5)], table())
    with pytest.raises(ValueError, match="with the row of pools"):
        bg.write_tokens(pools, [torch.zeros(3, 2, 4)], table())
    with pytest.raises(ValueError, match="type and device"):
        bg.write_tokens(pools, [torch.zeros(4, 2, 4, dtype=torch.float16)], table())
    with pytest.raises(ValueError, match="counts must be"):
        bg.write_tokens(pools, [torch.zeros(4, 2, 4)], table(), ones[:2])
    with pytest.raises(ValueError, match="keep must be"):
        bg.keep_tokens(pools, table(), ones, torch.zeros(4, 0, dtype=torch.int32), ones)
    with pytest.raises(ValueError, match="keep must be"):
        bg.keep_tokens(pools, table(), ones, torch.zeros(3, 2, dtype=torch.int32), ones)
    with pytest.raises(ValueError, match="drafted must be"):
        bg.keep_tokens(pools, table(), ones.float(), torch.zeros(4, 2, dtype=torch.int32), ones)
    with pytest.raises(ValueError, match="kept must be"):
        bg.keep_tokens(pools, table(), ones, torch.zeros(4, 2, dtype=torch.int32), ones[:1])


@pytest.mark.parametrize("states, parents, inplace, message", [
    ([torch.zeros(2, 3)], torch.zeros(2, 3), False, "parents must be"),
    ([torch.zeros(2, 3)], torch.zeros(6, dtype=torch.int64), False, "parents must be"),
    ([torch.zeros(2, 4)], torch.zeros(2, 3, dtype=torch.int64), False, "must be .B, K"),
    ([torch.zeros(2)], torch.zeros(2, 3, dtype=torch.int64), False, "must be .B, K"),
    ([torch.zeros(2, 3), torch.zeros(2, 3, 8)[..., ::2]], torch.zeros(2, 3, dtype=torch.int64), True, "contiguous"),
    ([torch.zeros(2, 1).expand(2, 3)], torch.zeros(2, 3, dtype=torch.int64), True, "contiguous"),
    ([torch.zeros(1, 4097)], torch.zeros(1, 4097, dtype=torch.int64), False, "4096 beams"),
])
def test_reorder_refusals(states, parents, inplace, message):
    with pytest.raises(ValueError, match=message):
        bg.reorder_states(states, parents, inplace=inplace)


PROBE = r"""
#include "paged.hpp"
#include <stdio.h>
using namespace dbs_hip;
int main() {
    const uint32_t ds[] = {1, 2, 3, 5, 7, 8, 16, 20, 24, 64, 100, 1023, 1024, 1025, 65536, 1000003, 0x3fffffff, 0x40000000, 0x40000001, 0x7fffffff};
    for (uint32_t d : ds) {
        const Divider q = Divider::of(d);
        const auto check = [&](uint32_t n) { if (n < 0x80000000u && q.quotient(n) != n / d) { printf("%u / %u\n", n, d); return 1; } return 0; };
        for (uint32_t n = 0; n < 3000; ++n) if (check(n)) return 1;
        for (uint64_t k = 0; k < 0x80000000u; k += 1000003) {
            const uint32_t at = static_cast<uint32_t>(k / d * d);
            if (check(at) || check(at + d - 1) || check(at ? at - 1 : 0) || check(static_cast<uint32_t>(k))) return 1;
        }
        if (check(0x7fffffffu) || check(0x7ffffffeu)) return 1;
    }
    const PageSpan s{Divider::of(24), 10, 3};
    if (s.is_page(-1) || s.is_page(10) || s.is_page(0x7fffffff) || s.is_page(-0x7fffffff - 1) || !s.is_page(0) || !s.is_page(9)) return 2;
    if (s.length(-5) != 0 || s.length(72) != 72 || s.length(73) != 72 || s.length(0x7fffffff) != 72 || s.length(7) != 7) return 3;
    if (s.held(0) != 0 || s.held(1) != 1 || s.held(24) != 1 || s.held(25) != 2 || s.held(72) != 3) return 4;
    return 0;
}
"""


def test_where_a_token_lies(tmp_path):
    """Quotients without a division, page entries and lengths out of range."""
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(PROBE)
    subprocess.run(["g++", "-std=c++20", "-O1", "-w", "-D__HIP_PLATFORM_AMD__=1", f"-I{_build.ROCM}/include",
                    f"-I{ROOT}/beamgrad_amd/csrc", str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_c_entries_refuse(tmp_path):
    """Null pointers and sizes, by a C program that launches nothing."""
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(r"""
#include <string.h>
#include "beamgrad_state.h"
int main(void) {
    BeamgradAttention a; memset(&a, 0, sizeof a);
    if (beamgrad_tree_attention_workspace_size(0) != -1 || beamgrad_tree_attention_workspace_size(&a) != -1) return 1;
    a.data_type = 2; a.sequences = 4; a.tokens = 1; a.heads = 8; a.kv_heads = 2; a.head_dim = 64; a.beams = 2;
    a.page_tokens = 16; a.n_pages = 10; a.table_pages = 4; a.scale = 0.125f;
    if (beamgrad_tree_attention_workspace_size(&a) <= 0) return 2;
    if (beamgrad_tree_attention(&a, 0, 0, 0) != 2) return 3;
    BeamgradAttention b = a; b.heads = 7; if (beamgrad_tree_attention_workspace_size(&b) != -1) return 4;
    b = a; b.head_dim = 60; if (beamgrad_tree_attention_workspace_size(&b) != -1) return 5;
    b = a; b.k_strides[0] = 4; if (beamgrad_tree_attention_workspace_size(&b) != -1) return 6;
    b = a; b.beams = 3; if (beamgrad_tree_attention_workspace_size(&b) != -1) return 7;
    b = a; b.table_pages = 0x7fffffff; if (beamgrad_tree_attention_workspace_size(&b) != -1) return 8;
    b = a; b.reserved = 1; if (beamgrad_tree_attention_workspace_size(&b) != -1) return 9;
    BeamgradPools p; memset(&p, 0, sizeof p);
    BeamgradTable t; memset(&t, 0, sizeof t);
    if (beamgrad_fork_pages(&p, &t, 0, 0, 4, 4, &t, 0, 0, 0) != 2 || beamgrad_fork_pages(0, 0, 0, 0, 4, 4, 0, 0, 0, 0) != 2) return 10;
    if (beamgrad_extend_pages(&t, 0, 4, 4, 4, 4, &t, 0, 0, 0) != 2) return 11;
    if (beamgrad_write_tokens(&p, 0, 0, 0, 0, 0, 4, 4, 1, 0) != 2) return 12;
    if (beamgrad_keep_tokens(&p, &t, 0, 0, 0, 4, 4, 1, &t, 0) != 2) return 13;
    int x = 0; int64_t n = 4; const void* f = &x; void* g = &x;
    if (beamgrad_reorder_states(&f, &g, &n, 1, 0, 0, 1, 1, 0) != 2 || beamgrad_reorder_states(&f, &g, &n, 1, &x, 0, 1, 5000, 0) != 2) return 14;
    if (beamgrad_reorder_states_backward(&f, &g, &n, 1, 0, &x, 0, 1, 1, 0) != 2) return 15;
    if (beamgrad_fork_pages_workspace_size(0) != -1 || beamgrad_extend_pages_workspace_size(0) != -1) return 16;
    return 0;
}
""")
    lib = os.path.dirname(_build.lib_path())
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), f"-L{lib}", "-ldbs_hip",
                    f"-Wl,-rpath,{lib}", f"-L{_build.ROCM}/lib", f"-Wl,-rpath,{_build.ROCM}/lib", "-lamdhip64", "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0


def test_shapes_without_a_gpu():
    """Meta tensors pass through every operator."""
    meta = torch.device("meta")
    t = bg.PageTable.empty(4, 5, 20, device=meta)
    pool = torch.zeros(20, 8, 2, 16, device=meta)
    ones = torch.ones(4, dtype=torch.int32, device=meta)
    out, lse = bg.tree_attention(torch.zeros(4, 3, 4, 16, device=meta), pool, pool, t, return_lse=True)
    assert out.shape == (4, 3, 4, 16) and lse.shape == (4, 3, 4) and lse.dtype == torch.float32
    for new in (bg.fork_pages([pool], t, ones), bg.extend_pages(t, ones, 8),
                bg.keep_tokens([pool], t, ones, torch.zeros(4, 2, dtype=torch.int32, device=meta), ones)):
        assert [x.shape for x in new] == [x.shape for x in t] and all(x.dtype == torch.int32 for x in new)
    assert bg.write_tokens([pool], [torch.zeros(4, 3, 2, 16, device=meta)], t) is None
    parents = torch.zeros(2, 3, dtype=torch.int64, device=meta)
    states = [torch.zeros(2, 3, 7, device=meta, requires_grad=True)]
    assert bg.reorder_states(states, parents)[0].shape == (2, 3, 7)
