"""Argument checks of the serving operators (rotation with append, beam selection, reordering of states), which fail
before anything touches the device, and the host control plane's reordering."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20  # a fake, aligned address: validation fails before any device access


def _rope(kvb, **kw):
    a = kvb.RopeArgs()
    a.in_dtype = a.out_dtype = a.kv_dtype = kvb.BF16
    a.num_tokens, a.num_heads, a.kv_heads, a.head_dim, a.rot_dim, a.block_size, a.num_blocks = 3, 8, 2, 64, 64, 16, 4
    a.max_positions, a.eps = 100, 1e-6
    a.q = a.k = a.v = a.q_out = a.table = a.positions = a.k_cache = a.v_cache = a.slots = PTR
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(in_dtype=9), dict(out_dtype=3), dict(kv_dtype=0), dict(head_dim=40), dict(head_dim=272),
                                 dict(rot_dim=8), dict(rot_dim=80), dict(rot_dim=24), dict(num_heads=0), dict(kv_heads=0),
                                 dict(num_tokens=-1), dict(max_positions=0), dict(q=0), dict(k=0), dict(v=0), dict(q_out=0),
                                 dict(table=0), dict(positions=0), dict(slots=0), dict(k_cache=0), dict(num_blocks=0),
                                 dict(block_size=0), dict(q=PTR + 2), dict(k_cache=PTR + 8), dict(q_stride=100),
                                 dict(k_stride=132), dict(v_stride=4), dict(q_out_stride=516), dict(k_out=PTR + 4),
                                 dict(q_norm=PTR, eps=-1.0), dict(q_norm=PTR, eps=float("nan")), dict(q_norm=PTR + 2),
                                 dict(k_cache=0, v_cache=0, slots=0), dict(num_heads=1 << 21)])
def test_rope_refuses(kvb, bad):
    assert kvb.lib().kvp_rope_append(C.byref(_rope(kvb, **bad)), None) == kvb.KVP_EINVAL and kvb.last_error()


def test_rope_of_no_tokens_is_fine(kvb):
    a = _rope(kvb, num_tokens=0, q=0, k=0, v=0)
    assert kvb.lib().kvp_rope_append(C.byref(a), None) == kvb.KVP_OK
    assert kvb.lib().kvp_rope_append(None, None) == kvb.KVP_EINVAL


def _beam(kvb, **kw):
    a = kvb.BeamArgs()
    a.logits = a.scores = a.out_scores = a.out_parents = a.out_tokens = a.workspace = PTR
    a.logits_dtype, a.batch, a.beams, a.vocab, a.select, a.workspace_bytes = kvb.BF16, 2, 4, 1000, 8, 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(logits_dtype=5), dict(batch=-1), dict(beams=0), dict(beams=33), dict(select=0),
                                 dict(select=33), dict(vocab=0), dict(vocab=(1 << 26) + 1), dict(vocab=1), dict(row_stride=999),
                                 dict(logits=0), dict(scores=0), dict(out_tokens=0), dict(logits=PTR + 1),
                                 dict(workspace=PTR + 8), dict(batch=1 << 23)])
def test_beam_refuses(kvb, bad):
    assert kvb.lib().kvp_beam_select(C.byref(_beam(kvb, **bad)), None) == kvb.KVP_EINVAL and kvb.last_error()


def test_beam_workspace(kvb):
    need = kvb.lib().kvp_beam_workspace_size(C.byref(_beam(kvb)))
    assert 0 < need < 1 << 20
    small = _beam(kvb, workspace_bytes=need - 1)
    assert kvb.lib().kvp_beam_select(C.byref(small), None) == kvb.KVP_ENOSPACE
    assert kvb.lib().kvp_beam_workspace_size(C.byref(_beam(kvb, select=40))) == 0 and kvb.last_error()
    assert kvb.lib().kvp_beam_workspace_size(C.byref(_beam(kvb, batch=0))) == 0
    assert kvb.lib().kvp_beam_select(C.byref(_beam(kvb, batch=0)), None) == kvb.KVP_OK
    assert kvb.lib().kvp_beam_workspace_size(None) == 0 and kvb.lib().kvp_beam_select(None, None) == kvb.KVP_EINVAL


def _prefix(kvb, **kw):
    a = kvb.PrefixArgs()
    a.q = a.k_cache = a.v_cache = a.block_tables = a.seq_lens = a.prefix_blocks = a.group_starts = a.out = a.workspace = PTR
    a.q_dtype = a.kv_dtype = a.out_dtype = kvb.BF16
    a.num_seqs, a.num_groups, a.num_heads, a.kv_heads, a.head_dim, a.block_size, a.max_blocks = 6, 2, 8, 2, 64, 16, 10
    a.num_blocks, a.workspace_bytes = 40, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(q_dtype=7), dict(kv_dtype=-1), dict(out_dtype=3), dict(num_seqs=-1), dict(num_groups=-1),
                                 dict(num_groups=0), dict(num_groups=7), dict(num_blocks=0), dict(num_blocks=-5),
                                 dict(block_size=0), dict(max_blocks=0), dict(head_dim=48), dict(head_dim=0), dict(num_heads=7),
                                 dict(num_heads=0), dict(kv_heads=0), dict(num_heads=34), dict(q=0), dict(out=0),
                                 dict(k_cache=0), dict(v_cache=0), dict(block_tables=0), dict(seq_lens=0),
                                 dict(prefix_blocks=0), dict(group_starts=0), dict(k_cache=PTR + 8), dict(v_cache=PTR + 2),
                                 dict(workspace=PTR + 16), dict(num_blocks=1 << 27), dict(num_blocks=(1 << 60) + 1)])
def test_prefix_refuses(kvb, bad):
    assert kvb.lib().kvp_prefix_attention(C.byref(_prefix(kvb, **bad)), None) == kvb.KVP_EINVAL and kvb.last_error()


def test_prefix_workspace(kvb):
    L = kvb.lib()
    need = L.kvp_prefix_workspace_size(C.byref(_prefix(kvb)))
    assert 0 < need < 1 << 30
    for kw in (dict(workspace_bytes=need - 1), dict(workspace=0)):
        assert L.kvp_prefix_attention(C.byref(_prefix(kvb, **kw)), None) == kvb.KVP_ENOSPACE
    assert L.kvp_prefix_workspace_size(C.byref(_prefix(kvb, head_dim=48))) == 0 and kvb.last_error()
    empty = _prefix(kvb, num_seqs=0, num_groups=0, q=0, out=0, workspace=0, workspace_bytes=0)
    assert L.kvp_prefix_workspace_size(C.byref(empty)) == 0 and not kvb.last_error()
    assert L.kvp_prefix_attention(C.byref(empty), None) == kvb.KVP_OK
    assert L.kvp_prefix_workspace_size(None) == 0 and L.kvp_prefix_attention(None, None) == kvb.KVP_EINVAL


def test_prefix_groups_from_tables(kvb):
    groups = lambda tables, lens, B=4: tuple(x.tolist() for x in kvb.shared_prefix_groups(np.array(tables), lens, B))
    assert groups(np.zeros((0, 3), np.int32), []) == ([], [0])
    assert groups([[5, 6, 7]], [12]) == ([0], [0, 1])  # alone: nothing is shared
    assert groups([[5, 6, 7], [5, 6, 8]], [12, 9]) == ([2, 2], [0, 2])
    assert groups([[5, 6, 7], [5, 6, 7]], [12, 12]) == ([3, 3], [0, 2])
    assert groups([[5, 6, 7], [5, 6, 7]], [12, 11]) == ([2, 2], [0, 2])  # only full blocks
    assert groups([[5, 6, 7], [5, 6, 7]], [12, 3]) == ([0, 0], [0, 1, 2])  # no full block
    # neighbours only; the run takes what all of it shares
    assert groups([[1, 2, 3], [1, 2, 4], [1, 9, 0], [8, 2, 3], [1, 2, 3], [0, 0, 0]], [12, 12, 6, 9, 12, 0]) == (
        [1, 1, 1, 0, 0, 0], [0, 3, 4, 5, 6])
    for tables, lens in (([[1, 2]], [12]), ([[1, 2]], [3, 4]), ([1, 2], [4, 4])):
        with pytest.raises(ValueError):
            kvb.shared_prefix_groups(np.array(tables), lens, 4)


def test_struct_layouts_match_the_header(kvb, tmp_path):
    structs = {"kvp_rope_args": kvb.RopeArgs, "kvp_beam_args": kvb.BeamArgs}
    if hasattr(kvb, "PrefixArgs"):
        structs["kvp_prefix_args"] = kvb.PrefixArgs
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "kvp_b200.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        s, f, v = ln.split()
        want = C.sizeof(structs[s]) if f == "sizeof" else getattr(structs[s], f).offset
        assert int(v) == want, (s, f)


# ------------------------------------------------------------------------------------------------ reordering of states
class Plain:
    """Block tables as plain lists: reordering is a permutation of their contents."""

    def __init__(self, mgr, rids):
        self.mgr, self.rids = mgr, rids
        self.read()

    def read(self):
        self.tables = [self.mgr.block_table(r) for r in self.rids]
        self.lens = [self.mgr.num_tokens(r) for r in self.rids]

    def reorder(self, parents):
        tables, lens = [self.tables[p] for p in parents], [self.lens[p] for p in parents]
        self.mgr.reorder(self.rids, parents)
        assert self.mgr.validate() == ""
        self.read()
        assert self.tables == tables and self.lens == lens


def test_reorder_random_walk(kvb):
    r = np.random.default_rng(3)
    mgr = kvb.KVManager(200, 4)
    rids = [10, 3, 77, 5]
    assert mgr.admit(10, 9)
    for x in rids[1:]:
        assert mgr.fork(x, 10)
    assert mgr.admit(1000, 30)  # a bystander
    other = mgr.block_table(1000)
    p = Plain(mgr, rids)
    for step in range(120):
        done, slots, pairs = mgr.append_batch(rids)
        assert done == 4 and len(set(slots.tolist())) == 4
        # no copy of a step reads what another one writes
        assert not set(pairs[:, 1].tolist()) & set(pairs[:, 0].tolist())
        p.read()
        p.reorder(r.integers(0, 4, 4).tolist())
        assert mgr.block_table(1000) == other
    assert mgr.num_tokens(10) == 129
    for x in rids + [1000]:
        mgr.free(x)
    assert mgr.free_blocks() == 200 and mgr.validate() == ""


def test_reorder_of_different_lengths_and_a_full_pool(kvb):
    """States of different lengths change hands; a pool without a free block is no obstacle."""
    mgr = kvb.KVManager(6, 4)
    assert mgr.admit(0, 15) and mgr.admit(1, 2) and mgr.admit(2, 1) and mgr.free_blocks() == 0
    p = Plain(mgr, [0, 1, 2])
    p.reorder([1, 0, 0])
    assert mgr.free_blocks() == 1 and [mgr.num_tokens(r) for r in (0, 1, 2)] == [2, 15, 15]
    p.reorder([2, 2, 2])
    assert mgr.free_blocks() == 2 and mgr.stats()["blocks_saved"] == 8
    p.reorder([0, 1, 2])
    mgr.reorder([], [])
    assert mgr.validate() == ""


def test_reorder_keeps_cached_prefixes(kvb):
    mgr = kvb.KVManager(20, 4)
    assert mgr.admit(0, 9) and mgr.cache_prefix(5, 0, 8) and mgr.admit(1, 5)
    mgr.reorder([0, 1], [1, 1])
    assert mgr.cached_prefix_tokens(5) == 8 and mgr.validate() == ""
    assert mgr.admit_with_cached_prefix(2, 5, 8, 12) and mgr.validate() == ""


def test_reorder_refuses_and_changes_nothing(kvb):
    mgr = kvb.KVManager(20, 4)
    assert mgr.admit(0, 9) and mgr.admit(1, 5)
    before = [mgr.block_table(r) for r in (0, 1)], mgr.stats()
    for rids, parents, err in (([0, 1], [0, 2], ValueError), ([0, 1], [-1, 0], ValueError), ([0, 0], [0, 1], ValueError),
                               ([0, 9], [0, 1], RuntimeError), ([0, 1], [0], ValueError)):
        with pytest.raises(err):
            mgr.reorder(rids, parents)
    assert before == ([mgr.block_table(r) for r in (0, 1)], mgr.stats()) and mgr.validate() == ""
    assert kvb.lib().kvp_mgr_reorder(None, None, None, 0) == kvb.KVP_EINVAL
    assert kvb.lib().kvp_mgr_reorder(mgr.handle, None, None, -1) == kvb.KVP_EINVAL


@pytest.mark.parametrize("shape,strides", [((4, 8, 64), (0, 64, 1)), ((2, 8, 64), (0, 64, 1)), ((4, 8, 64), (256, 64, 1)),
                                           ((4, 1, 64), (0, 64, 1)), ((4, 1, 64), (32, 64, 1))])
def test_rows_that_several_tokens_share_are_refused(kvb, shape, strides):
    """One row expanded over the tokens, or rows that run into each other: below, a stride of 0 stands for contiguous rows,
    which the storage does not hold."""
    import torch
    with pytest.raises(ValueError):
        kvb._token_stride(torch.zeros(4096).as_strided(shape, strides), "q", torch.Size(shape))


def test_strides_that_are_fine(kvb):
    import torch
    stride = lambda t: kvb._token_stride(t, "q", t.shape)  # noqa: E731
    assert stride(torch.zeros(4, 8, 64)) == 512 and stride(torch.zeros(4, 1024)[:, 256:768].view(4, 8, 64)) == 1024
    assert stride(torch.zeros(8, 64).expand(1, 8, 64)) == 512 and stride(torch.zeros(0, 8, 64)) == 512


def test_prefix_table_rows_near_32_bits(kvb):
    """A table row of nearly 2^31 tokens, whose last tiles' places would pass 32 bits, goes the way of longer ones: it needs
    the same workspace."""
    size = lambda blocks: kvb.lib().kvp_prefix_workspace_size(C.byref(_prefix(kvb, num_seqs=2000, max_blocks=blocks)))  # noqa: E731
    longer = size(1 << 27)
    assert 0 < longer < size((1 << 27) - 64) == size(10)
    for blocks in ((1 << 27) - 1, (1 << 27) - 20, (1 << 27) - 63):
        assert size(blocks) == longer


@pytest.mark.parametrize("D,g", [(32, 16), (64, 16), (128, 8), (256, 8), (96, 4)])
@pytest.mark.parametrize("B", [5, 16, 130])
@pytest.mark.parametrize("kv", ["BF16", "F16"])
def test_prefix_workspace_covers_any_alignment(kvb, D, g, B, kv):
    """A size asked for without buffers serves any of them: queries or outputs off a 16-byte boundary go another way."""
    for q in ("BF16", "F32"):
        for kvh in (1, 2, 8):
            size = lambda **kw: kvb.lib().kvp_prefix_workspace_size(C.byref(_prefix(  # noqa: E731
                kvb, head_dim=D, kv_heads=kvh, num_heads=kvh * g, block_size=B, kv_dtype=getattr(kvb, kv),
                q_dtype=getattr(kvb, q), **kw)))
            need = size()
            assert need == size(q=0, out=0)
            if need == 0:  # a shape that the decode attention does not take
                assert "shared memory" in kvb.last_error()
                continue
            # (a call off the boundary shares nothing and may need less)
            assert need >= max(size(q=PTR + 2), size(out=PTR + 4), size(q=PTR + 2, out=PTR + 4)) > 0


def test_sizes_beyond_32_bits_are_refused(kvb):
    """ctypes cuts a number to a field's 32 bits: select = 2^32 + 3 would have become 3."""
    assert kvb._i32(2 ** 31 - 1, "x") == 2 ** 31 - 1 and kvb._i32(-1, "x") == -1
    for x in (2 ** 31, 2 ** 32 + 3, -2 ** 31 - 1):
        with pytest.raises(ValueError):
            kvb._i32(x, "x")


def test_status_words_of_other_types_are_refused(kvb):
    import torch
    for bad in (torch.zeros(1, dtype=torch.uint8), torch.zeros(1), torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="status"):
            kvb._status_word(bad)


def test_when_a_step_goes_by_groups(kvb):
    """The engine's rule between the shared-prefix attention and the decode attention, on both sides of it."""
    import importlib
    pays = importlib.import_module("paged-kv-cache-manager_b200.model")._sharing_pays

    def step(groups, block=16, kv_heads=8, dim=128):  # (shared blocks, own tokens of each member)
        prefix, starts, lens = [], [0], []
        for blocks, own in groups:
            prefix += [blocks] * len(own)
            lens += [blocks * block + x for x in own]
            starts.append(len(lens))
        return pays(np.array(prefix, np.int32), np.array(starts, np.int32), lens, block, kv_heads, dim, 148)

    for yes in ([(128, [100] * 256)], [(1024, [8192] * 16)], [(1, [100] * 16)], [(128, [1000] * 2)], [(5, [1, 2, 3])],
                [(0, [50]), (9, [3, 4])], [(128, [100] * 255 + [3000])], [(256, [4000] * 64)]):
        assert step(yes), yes
    for no in ([(1, [100] * 255 + [30000])], [(1, [30000, 30000])], [(1024, [8192] * 4)], [(16, [100] * 128 + [4000])],
               [(0, [30000]), (9, [3, 4])], [(1, [8192] * 64)]):
        assert not step(no), no
