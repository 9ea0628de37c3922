"""Decode attention of groups that share leading blocks (kvp_prefix_attention) against softmax attention of each
sequence over its whole context in 64 bits.

Tolerance of an output element, with weights p_i (sum 1), values v_i, n context tokens, u = eps / 2 of the pools' type
and A = sum p_i |v_i|:
  * the output's rounding: (eps / 2 of its type) |out|;
  * every weight of the shared part is rounded to the pools' type before the product: at most u A; fp16 weights below
    2^-14 of the (at most 1) largest have an absolute error of 2^-25 instead, in all at most n 2^-25 max |v|;
  * a score is a sum of head_dim products in fp32: off by at most (head_dim + 4) 2^-24 sum |q_d k_d| scale =: e; that
    changes a weight and the sum of all by a factor of at most 1 + 2 e each: 4 e A.  The exponentials (2^-22 each) and
    their arguments (rounded sums of at most a few hundred: 2^-16 in all) add less than 2^-15 A;
  * the sums over tokens in fp32: n 2^-24 A, for numerator and sum: 2 n 2^-24 A."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


class Batch:
    """Groups of (members, shared blocks) with own tokens from `own(r)`, blocks in random places of a pool whose unused
    slots are NaN."""

    def __init__(self, groups, own, nh, kvh, D, B, qt="bf16", kvt="bf16", seed=0, spread=1.0):
        import torch
        r = np.random.default_rng(seed)
        self.nh, self.kvh, self.D, self.B = nh, kvh, D, B
        lens, tables, prefix, starts, used = [], [], [], [0], 0
        shared_at = []
        for members, blocks in groups:
            shared = list(range(used, used + blocks))
            used += blocks
            for _ in range(members):
                extra = int(own(r))
                if blocks == 0:
                    extra = max(extra, 1)
                nb = -(-extra // B)
                tables.append(shared + list(range(used, used + nb)))
                used += nb
                lens.append(blocks * B + extra)
                prefix.append(blocks)
            starts.append(starts[-1] + members)
        nb = used + 3
        perm = r.permutation(nb)
        width = max(len(t) for t in tables) + 2
        dense = np.zeros((len(tables), width), dtype=np.int32)
        for i, t in enumerate(tables):
            dense[i, :len(t)] = perm[t]
        slots = np.zeros((nb, B), dtype=bool)
        for i, t in enumerate(tables):
            for j, b in enumerate(t):
                slots[perm[b], :min(B, lens[i] - j * B)] = True
        g = torch.Generator(device="cuda").manual_seed(seed)
        mk = lambda: torch.randn((nb, B, kvh, D), generator=g, device="cuda")  # noqa: E731
        hole = ~torch.from_numpy(slots).cuda()[:, :, None, None]
        self.k = mk().masked_fill(hole, math.nan).to(_dt(kvt))
        self.v = mk().masked_fill(hole, math.nan).to(_dt(kvt))
        n = len(tables)
        self.q = (spread * torch.randn((n, nh, D), generator=g, device="cuda")).to(_dt(qt))
        dev = lambda a: torch.from_numpy(np.asarray(a, dtype=np.int32)).cuda()  # noqa: E731
        self.tables, self.lens, self.prefix, self.starts = dev(dense), dev(lens), dev(prefix), dev(starts)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def args(self):
        return (self.q, self.k, self.v, self.tables, self.lens, self.prefix, self.starts, self.nh, self.kvh)

    def run(self, kvb, **kw):
        return kvb.shared_prefix_attention(*self.args(), status=self.status, **kw)

    def reference(self, scale=None):
        """out, A and the largest e and |v| of every row, in 64 bits."""
        import torch
        n, nh, D = self.q.shape
        out, mag, err, top = (torch.zeros((n, nh, w), dtype=torch.float64, device="cuda") for w in (D, D, 1, 1))
        kf, vf = self.k.view(-1, self.kvh, D), self.v.view(-1, self.kvh, D)
        per, scale = nh // self.kvh, scale or D ** -0.5
        for i, n_i in enumerate(self.lens.tolist()):
            at = torch.arange(n_i, device="cuda")
            slot = self.tables[i].long()[at // self.B] * self.B + at % self.B
            k, v = (x[slot].double().repeat_interleave(per, 1) for x in (kf, vf))
            q = self.q[i].double()
            w = torch.softmax(torch.einsum("hd,thd->ht", q, k) * scale, -1)
            out[i] = torch.einsum("ht,thd->hd", w, v)
            mag[i] = torch.einsum("ht,thd->hd", w, v.abs())
            err[i] = (torch.einsum("hd,thd->ht", q.abs(), k.abs()).amax(-1) * scale * (D + 4) * 2.0 ** -24)[:, None]
            top[i] = v.abs().amax((0, 2))[:, None]
        return out, mag, err, top

    def check(self, got, scale=None):
        import torch
        want, mag, err, top = self.reference(scale)
        n = self.lens.double()[:, None, None]
        u = torch.finfo(self.k.dtype).eps / 2
        tol = want.abs() * (torch.finfo(got.dtype).eps / 2) + (u + 4 * err + 2.0 ** -15 + 2 * n * 2.0 ** -24) * mag
        if self.k.dtype == torch.float16 or got.dtype == torch.float16:
            tol = tol + n * 2.0 ** -25 * top
        bad = (got.double() - want).abs() - tol
        assert bool(torch.isfinite(got).all()), "not finite"
        assert float(bad.max()) <= 0, (float(bad.max()), float((got.double() - want).abs().max()))
        assert int(self.status.item()) == 0


few = lambda r: r.integers(0, 40)  # noqa: E731
mixed = lambda r: r.choice([0, 1, 15, 16, 17, 100, 333])  # noqa: E731

SHARING = [
    # groups, own tokens, heads, kv heads, dim, block, type
    ([(4, 8)], few, 32, 8, 128, 16, "bf16"),
    ([(1, 1)], few, 1, 1, 64, 8, "fp16"),
    ([(2, 8)], few, 4, 4, 64, 16, "bf16"),
    ([(3, 9)], mixed, 14, 2, 64, 16, "fp16"),              # seven heads per kv head: 126-row tiles
    ([(33, 20)], mixed, 32, 8, 128, 16, "bf16"),            # just over one row tile
    ([(65, 33)], few, 32, 8, 128, 16, "fp16"),              # just over two: a second pair with one tile
    ([(200, 40)], few, 8, 8, 64, 16, "bf16"),               # one head per kv head
    ([(40, 30)], few, 16, 1, 128, 16, "bf16"),              # sixteen heads on one kv head
    ([(5, 3), (1, 0), (7, 11), (1, 4), (2, 0), (90, 17)], mixed, 32, 4, 64, 16, "fp16"),
    ([(3, 37), (30, 5)], few, 8, 2, 128, 8, "bf16"),
    ([(9, 3), (4, 1)], mixed, 8, 2, 64, 128, "fp16"),
    ([(9, 3)], mixed, 8, 2, 128, 256, "bf16"),
    ([(6, 5)], mixed, 8, 2, 128, 24, "bf16"),               # 24 tokens a block: runs of 8
    ([(6, 4)], mixed, 8, 2, 64, 40, "fp16"),
    ([(16, 300)], few, 32, 8, 128, 16, "bf16"),             # many key tiles per CTA
    ([(130, 260)], few, 32, 8, 128, 16, "bf16"),
    ([(2, 2)] * 400, few, 8, 2, 64, 16, "bf16"),            # more groups than the kernel has threads
]


@pytest.mark.parametrize("case", range(len(SHARING)))
def test_sharing_kernel(kvb, cuda, case):
    groups, own, nh, kvh, D, B, t = SHARING[case]
    b = Batch(groups, own, nh, kvh, D, B, t, t, seed=case)
    b.check(b.run(kvb))


@pytest.mark.parametrize("nh,kvh,D,B,qt,kvt,out", [(8, 2, 32, 16, "bf16", "bf16", "bf16"), (8, 2, 96, 16, "fp16", "fp16", "fp32"),
                                                   (8, 2, 256, 16, "bf16", "bf16", "bf16"), (8, 2, 64, 5, "bf16", "bf16", "bf16"),
                                                   (8, 2, 128, 1, "fp16", "fp16", "fp16"), (8, 2, 64, 16, "fp32", "fp16", "fp32"),
                                                   (8, 2, 64, 16, "fp32", "fp32", "fp32"), (8, 2, 64, 16, "bf16", "fp16", "bf16")])
def test_whole_context_path(kvb, cuda, nh, kvh, D, B, qt, kvt, out):
    """Shapes that the sharing kernel does not take have the same answers."""
    b = Batch([(4, 6), (3, 0), (5, 2)], mixed, nh, kvh, D, B, qt, kvt, seed=D + B)
    # a context of no own tokens is at least its shared blocks long, so every length is positive
    b.check(b.run(kvb, out_dtype=_dt(out)))


@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
def test_output_types_and_scale(kvb, cuda, out):
    b = Batch([(10, 20), (40, 3)], mixed, 16, 4, 128, 16, seed=5)
    b.check(b.run(kvb, out_dtype=_dt(out), scale=0.2), scale=0.2)


@pytest.mark.parametrize("spread", [8.0, 30.0])
def test_peaked_scores(kvb, cuda, spread):
    """Large scores: a few keys carry the weight, and the running maximum moves far between key tiles."""
    for D, t in ((128, "bf16"), (64, "fp16")):
        b = Batch([(40, 60), (3, 70)], mixed, 8, 2, D, 16, t, t, seed=3, spread=spread)
        b.check(b.run(kvb))


def test_rising_and_falling_scores(kvb, cuda):
    """Keys that grow (then shrink) along the context: every key tile rescales (none does)."""
    import torch
    for falling in (False, True):
        b = Batch([(40, 64)], few, 8, 2, 64, 16, seed=4)
        n = 64 * 16
        ramp = torch.linspace(40 if falling else -40, -40 if falling else 40, n, device="cuda")
        slot = (b.tables[0, :64].long()[:, None] * 16 + torch.arange(16, device="cuda")).flatten()
        q = b.q.float()
        b.q = (q / q.norm(dim=-1, keepdim=True)).to(b.q.dtype)
        mean = b.q.float().view(40, 2, 4, 64)[0, :, 0]
        flat = b.k.view(-1, 2, 64)
        flat[slot] = (ramp[:, None, None] * mean).to(flat.dtype)
        b.check(b.run(kvb, scale=1.0), scale=1.0)


def test_equals_paged_attention(kvb, cuda):
    """The same batch through the decode attention: both are inside the tolerance, and alike without sharing."""
    import torch
    b = Batch([(6, 12), (2, 30)], mixed, 32, 8, 128, 16, seed=8)
    b.check(kvb.paged_attention(b.q, b.k, b.v, b.tables, b.lens, 32, 8))
    b = Batch([(6, 0), (1, 0)], mixed, 32, 8, 128, 16, seed=8)
    got = b.run(kvb, out_dtype=torch.float32)
    b.check(got)
    # Without sharing both keep a weight as two 16-bit numbers, which are off by at most (eps / 2)^2 = 2^-16 of it, beside
    # the scores', exponentials' and sums' fp32 errors of the module's account; each may be off by as much.
    _, mag, err, _ = b.reference()
    each = (2.0 ** -16 + 4 * err + 2.0 ** -15 + 2 * b.lens.double()[:, None, None] * 2.0 ** -24) * mag
    other = kvb.paged_attention(b.q, b.k, b.v, b.tables, b.lens, 32, 8, out_dtype=torch.float32)
    assert float(((got - other).double().abs() - 2 * each).max()) <= 0


def test_same_answer_every_time_and_with_dirty_workspace(kvb, cuda):
    import torch
    b = Batch([(70, 50), (9, 31)], mixed, 32, 8, 128, 16, seed=9)
    need = kvb.shared_prefix_workspace_bytes(b.q, b.k, b.tables, b.starts, 32, 8)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    first = b.run(kvb)
    for _ in range(5):
        assert torch.equal(b.run(kvb, workspace=ws), first)
    # a smaller batch of the same heads in the same workspace, then the first one again
    c = Batch([(3, 4)], few, 32, 8, 128, 16, seed=10)
    c.check(c.run(kvb, workspace=ws))
    assert torch.equal(b.run(kvb, workspace=ws), first)


def test_stream_and_graph(kvb, cuda):
    """Another stream; a captured call replayed on changed queries, lengths and groups; two graphs in turn on one
    workspace."""
    import torch
    b, c = (Batch([(20, 18), (5, 7)], mixed, 8, 2, 64, 16, seed=s) for s in (1, 2))
    want_b, want_c = b.run(kvb), c.run(kvb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = b.run(kvb, stream=side)
    side.synchronize()
    assert torch.equal(got, want_b)
    ws = torch.empty(kvb.shared_prefix_workspace_bytes(b.q, b.k, b.tables, b.starts, 8, 2), dtype=torch.uint8, device="cuda")
    graphs = []
    for x in (b, c):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(x.q)
        with torch.cuda.graph(g):
            x.run(kvb, out=out, workspace=ws)
        graphs.append((g, out))
    for g, _ in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want_b) and torch.equal(graphs[1][1], want_c)
    # other queries, one group cut in two and shorter contexts, all read on the device
    b.q.copy_(c.q)
    b.lens[0] = int(b.prefix[0]) * 16
    b.prefix[20:] = 6
    graphs[0][0].replay()
    torch.cuda.synchronize()
    b.check(graphs[0][1])


def test_bad_groups_lengths_and_blocks(kvb, cuda):
    """What only the device can see: the sequences concerned get zeros and a status bit, the others their answers."""
    import torch
    base = lambda: Batch([(4, 6), (3, 2), (5, 9)], lambda r: r.integers(1, 30), 8, 2, 64, 16, seed=6)  # noqa: E731
    good = base().run(kvb)
    for change, rows in ((lambda b: b.lens.__setitem__(5, 0), [5]), (lambda b: b.lens.__setitem__(5, -7), [5]),
                         (lambda b: b.lens.__setitem__(5, 1 << 20), [5]), (lambda b: b.lens.__setitem__(5, 31), [5]),
                         (lambda b: b.prefix.__setitem__(5, 1), [5]), (lambda b: b.prefix.__setitem__(4, -1), [4, 5, 6]),
                         (lambda b: b.prefix.__setitem__(4, 1 << 30), [4, 5, 6]),
                         (lambda b: b.prefix.__setitem__(6, 1 << 30), [6]),
                         (lambda b: b.starts.__setitem__(2, 99), None), (lambda b: b.starts.__setitem__(1, -3), None),
                         (lambda b: b.starts.__setitem__(0, 2), None), (lambda b: b.starts.__setitem__(3, 11), [11])):
        b = base()
        change(b)
        got = b.run(kvb)
        torch.cuda.synchronize()
        assert int(b.status.item()) == kvb.KVP_STATUS_BAD_LEN
        zero = [i for i in range(12) if bool((got[i] == 0).all())]
        if rows is not None:
            assert zero == rows
            keep = [i for i in range(12) if i not in rows]
            torch.testing.assert_close(got[keep].float(), good[keep].float(), rtol=2e-2, atol=2e-2)
    b = base()
    b.tables[4:7, 1] = 1 << 20  # a shared block outside the pool: its tokens count as zero keys and values
    b.run(kvb)
    torch.cuda.synchronize()
    assert int(b.status.item()) == kvb.KVP_STATUS_BAD_BLOCK


def test_groups_from_tables(kvb, cuda):
    """A manager's forks and prefix admissions, through shared_prefix_groups, against the decode attention."""
    import torch
    mgr = kvb.KVManager(200, 16)
    assert mgr.admit(0, 100) and mgr.fork(1, 0) and mgr.fork(2, 0) and mgr.admit(3, 50) and mgr.admit_with_prefix(4, 3, 40, 77)
    assert mgr.admit(5, 9)
    rids = [0, 1, 2, 3, 4, 5]
    for _ in range(20):
        assert mgr.append_batch(rids)[0] == 6
    tables, lens = mgr.dense_tables(rids, 12)
    prefix, starts = kvb.shared_prefix_groups(tables, lens, 16)
    assert prefix.tolist() == [6, 6, 6, 2, 2, 0] and starts.tolist() == [0, 3, 5, 6]
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((200, 16, 2, 64), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((6, 8, 64), generator=g, device="cuda").half()
    t, n, p, s = (torch.from_numpy(x).cuda() for x in (tables, lens, prefix, starts))
    got = kvb.shared_prefix_attention(q, k, v, t, n, p, s, 8, 2)
    torch.testing.assert_close(got, kvb.paged_attention(q, k, v, t, n, 8, 2), rtol=2e-3, atol=2e-3)


def test_empty_batch_and_refusals(kvb, cuda):
    import torch
    b = Batch([(3, 4)], few, 8, 2, 64, 16, seed=1)
    run = lambda **kw: kvb.shared_prefix_attention(*{**dict(zip(("q", "k", "v", "t", "n", "p", "s", "nh", "kvh"), b.args())), **kw}.values())  # noqa: E731
    for bad in (dict(q=b.q[:, :4]), dict(q=b.q.cpu()), dict(t=b.tables.long()), dict(t=b.tables[:2]), dict(n=b.lens[:2]),
                dict(p=b.prefix[:1]), dict(s=b.starts[:1]), dict(s=torch.zeros(5, dtype=torch.int32, device="cuda")),
                dict(v=b.v.float()), dict(q=b.q.transpose(0, 1)), dict(kvh=4), dict(nh=9)):
        with pytest.raises(ValueError):
            run(**bad)
    with pytest.raises(kvb.KVPError):
        b.run(kvb, workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    none = kvb.shared_prefix_attention(b.q[:0], b.k, b.v, b.tables[:0], b.lens[:0], b.prefix[:0], b.starts[:1], 8, 2)
    assert none.shape == (0, 8, 64)


@pytest.mark.parametrize("groups,own,nh,kvh,D,t", [([(290, 3), (15, 0)], mixed, 16, 8, 128, "bf16"),  # a warp per (sequence, kv head)
                                                   ([(310, 2)], few, 32, 8, 64, "fp16"),
                                                   ([(80, 4)], mixed, 8, 8, 128, "fp16"),              # four warps
                                                   ([(9, 1), (30, 6)], lambda r: r.integers(500, 900), 16, 1, 64, "bf16"),
                                                   ([(2, 3)] * 32, few, 8, 2, 64, "fp16"),            # found by a warp alone
                                                   ([(2, 3)] * 33, few, 8, 2, 64, "fp16"),            # and by the CTA
                                                   ([(1, 0)] * 40, mixed, 8, 2, 128, "bf16")])         # nothing is shared
def test_splits_of_the_own_parts(kvb, cuda, groups, own, nh, kvh, D, t):
    b = Batch(groups, own, nh, kvh, D, 16, t, t, seed=len(groups) + nh)
    b.check(b.run(kvb))


def test_calls_behind_each_other(kvb, cuda):
    """Every kernel may start before the one ahead has ended: calls on one workspace, whose queries, lengths and pools are
    overwritten by kernels in between and whose output is read by the next, give what they give one at a time."""
    import torch
    b = Batch([(40, 6), (3, 9)], lambda r: r.integers(20, 200), 16, 4, 128, 16, seed=31)
    ws = torch.empty(kvb.shared_prefix_workspace_bytes(b.q, b.k, b.tables, b.starts, 16, 4), dtype=torch.uint8, device="cuda")
    qs = [torch.randn_like(b.q, dtype=torch.float32).to(b.q.dtype) for _ in range(6)]
    lens, k = b.lens.clone(), b.k.clone()

    def step(i):
        b.lens.copy_(lens - i)
        b.k.copy_(k).mul_(1.0 + i / 8)
        b.q.copy_(qs[i])
        x = b.run(kvb, workspace=ws)
        return kvb.shared_prefix_attention(x, *b.args()[1:], workspace=ws, status=b.status)

    alone = []
    for i in range(6):
        alone.append(step(i))
        torch.cuda.synchronize()
    for _ in range(5):
        behind = [step(i) for i in range(6)]
        torch.cuda.synchronize()
        for x, y in zip(alone, behind):
            assert torch.equal(x, y)
    assert int(b.status.item()) == 0


def test_pool_behind_32_bit_offsets(kvb, cuda):
    """The same blocks at the end of pools of more than 2^32 elements: the same bits."""
    import torch
    b = Batch([(20, 12), (4, 3)], mixed, 32, 8, 128, 16, seed=12)
    want = b.run(kvb)
    nb = b.k.shape[0]
    many = (1 << 32) // (16 * 8 * 128) + 1000
    big = [torch.empty((many, 16, 8, 128), dtype=b.k.dtype, device="cuda") for _ in range(2)]
    for x, y in zip(big, (b.k, b.v)):
        x[-nb:].copy_(y)
    got = kvb.shared_prefix_attention(b.q, *big, b.tables + (many - nb), b.lens, b.prefix, b.starts, 32, 8, status=b.status)
    assert torch.equal(got, want) and int(b.status.item()) == 0


@pytest.mark.parametrize("groups,nh,kvh,D,B,t", [([(70, 60), (3, 9)], 8, 2, 128, 5, "bf16"), ([(9, 200)], 32, 8, 64, 1, "fp16"),
                                                 ([(40, 7)], 16, 4, 128, 33, "fp16"), ([(6, 3), (2, 0), (80, 2)], 32, 4, 64, 100, "bf16"),
                                                 ([(5, 40)], 8, 2, 128, 12, "bf16"), ([(7, 30)], 14, 2, 64, 7, "fp16"),
                                                 ([(20, 2)], 8, 2, 64, 127, "bf16"), ([(20, 2)], 8, 2, 64, 130, "bf16")])
def test_blocks_of_odd_sizes(kvb, cuda, groups, nh, kvh, D, B, t):
    """Tiles of as many whole blocks as fit 128 keys (none of 130 tokens)."""
    b = Batch(groups, mixed, nh, kvh, D, B, t, t, seed=B)
    b.check(b.run(kvb))


@pytest.mark.parametrize("groups,nh,kvh,D", [([(100, 500)] + [(2, 1)] * 40, 32, 8, 128), ([(2, 1)] * 300, 8, 8, 64),
                                             ([(3, 8), (2, 9), (2, 1), (2, 1), (4, 17), (2, 2)] * 30, 16, 8, 64)])
def test_groups_of_one_key_tile(kvb, cuda, groups, nh, kvh, D):
    """CTAs with stretch after stretch of a single key tile (and of one, two and three in turn), behind a long one: one
    warpgroup has nothing to do in most of them and falls behind the other by as much as it likes."""
    import torch
    b = Batch(groups, few, nh, kvh, D, 16, seed=len(groups))
    first = b.run(kvb)
    b.check(first)
    for _ in range(20):
        assert torch.equal(b.run(kvb), first)
    assert int(b.status.item()) == 0


def _check_close(b, got, scale=None, lift=0):
    """The module's account with weights kept as two 16-bit numbers, a part and the rest: off by at most u^2, and in fp16 by
    2^-25 of the largest where the rest lies below the type's smallest steps (2^-25 - lift, where the largest weight is
    represented by 2^lift)."""
    import torch
    want, mag, err, top = b.reference(scale)
    n = b.lens.double()[:, None, None]
    u = torch.finfo(b.k.dtype).eps / 2
    tol = want.abs() * (torch.finfo(got.dtype).eps / 2) + (u * u + 4 * err + 2.0 ** -15 + 2 * n * 2.0 ** -24) * mag
    if b.k.dtype == torch.float16:
        tol = tol + n * 2.0 ** (-25 - lift) * top
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # the output's smallest step
    assert bool(torch.isfinite(got).all()) and int(b.status.item()) == 0
    assert float(((got.double() - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("groups,nh,kvh,D,t", [([(4, 8)], 32, 8, 128, "bf16"), ([(40, 30), (3, 1)], 32, 8, 128, "bf16"),
                                               ([(70, 20)], 8, 2, 64, "bf16"), ([(40, 30)], 16, 4, 64, "fp16"),
                                               ([(9, 12), (65, 9)], 32, 8, 128, "fp16")])
@pytest.mark.parametrize("out", ["same", "fp32"])
@pytest.mark.parametrize("spread", [1.0, 4.0])
def test_weights_of_shared_keys_keep_their_bits(kvb, cuda, groups, nh, kvh, D, t, out, spread):
    """Shared keys' weights are as exact as those of own ones and of the decode attention: an fp32 output shows it."""
    b = Batch(groups, lambda r: r.integers(0, 3), nh, kvh, D, 16, t, t, seed=nh + D, spread=spread)
    _check_close(b, b.run(kvb, out_dtype=_dt(t if out == "same" else out)))


@pytest.mark.parametrize("t", ["fp16", "bf16"])
@pytest.mark.parametrize("shared,n,nh,kvh", [(True, 1 << 17, 4, 1), (False, 1 << 17, 4, 1), (True, 1 << 15, 148, 148)])
@pytest.mark.parametrize("first", [True, False])
def test_long_flat_tail_below_one_key(kvb, cuda, t, shared, n, nh, kvh, first):
    """One key (the first, or a late one) and n - 1 others of 2^-25.5 of its weight: in fp16 numbers of the weights
    themselves all of these are zero, though they make up to 0.3% of the output.  148 heads: a head per CTA."""
    import torch
    b = Batch([(2, n // 16)] if shared else [(2, 0)], (lambda r: 0) if shared else (lambda r: n), nh, kvh, 64, 16, t, t)
    b.q.zero_()[..., 0] = 1
    slot = b.tables[:, :n // 16].long()[..., None] * 16 + torch.arange(16, device="cuda")
    at = slot.flatten(1)[:, 0 if first else n - 1000]
    k, v = b.k.view(-1, kvh, 64), b.v.view(-1, kvh, 64)
    k.zero_()[..., 0] = -17.67
    v.fill_(1)
    k[at, :, 0], v[at] = 0, 0
    _check_close(b, b.run(kvb, out_dtype=torch.float32, scale=1.0), scale=1.0, lift=12)


def test_large_values_behind_rising_scores(kvb, cuda):
    """Scores that rise by 2^39 behind the first key tiles, over values near 2^100: the weights' reference has to follow, or
    weight times value passes fp32's range.  148 heads: a head's eight key tiles for each CTA."""
    import torch
    b = Batch([(2, 64)], few, 148, 148, 64, 16, seed=4)
    b.v.mul_(2.0 ** 100)
    b.q.mul_(0.01)
    b.q[..., 0] = 1
    slot = (b.tables[0, :64].long()[:, None] * 16 + torch.arange(16, device="cuda")).flatten()
    b.k.view(-1, 148, 64)[slot, :, 0] = torch.where(torch.arange(1024, device="cuda") < 256, 0.0, 27.0).to(b.k.dtype)[:, None]
    b.check(b.run(kvb, scale=1.0), scale=1.0)


@pytest.mark.parametrize("D,t", [(64, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("where", ["one", "tile", "prefix", "own"])
def test_nan_keys_show(kvb, cuda, where, D, t):
    """NaN keys inside the context -- one, a tile's, all shared ones, all own ones of a sequence -- make the outputs of their kv
    head NaN, as softmax does and the decode attention does; the other head, and other sequences, keep their answers."""
    import torch
    base = lambda: Batch([(5, 30), (3, 9)], lambda r: r.integers(1, 60), 8, 2, D, 16, t, t, seed=21)  # noqa: E731
    good, b = base().run(kvb), base()
    blocks = {"one": b.tables[0, 7:8], "tile": b.tables[0, 8:16], "prefix": b.tables[0, :30], "own": b.tables[2, 30:]}[where].long()
    rows = [2] if where == "own" else list(range(5))
    if where == "own":
        blocks = blocks[:-(-(int(b.lens[2]) - 480) // 16)]
    b.k[blocks[:, None], torch.arange(1 if where == "one" else 16, device="cuda")[None], 1] = math.nan
    got, whole = b.run(kvb), kvb.paged_attention(b.q, b.k, b.v, b.tables, b.lens, 8, 2)
    hit = torch.zeros((8, 8), dtype=torch.bool, device="cuda")
    hit[rows, 4:] = True
    for x in (got, whole):
        assert bool(x[hit].isnan().all()) and bool(torch.isfinite(x[~hit]).all())
    assert torch.equal(got[~hit], good[~hit])


def test_infinite_scores_of_some_keys(kvb, cuda):
    """Scores of -inf weigh nothing, in part or all of what is shared."""
    import torch
    for blocks in (slice(3, 4), slice(0, 30)):
        b = Batch([(5, 30)], lambda r: r.integers(1, 60), 8, 2, 64, 16, seed=22)
        b.q[..., 0] = 1
        b.k[b.tables[0, blocks].long(), :, :, 0] = -math.inf
        got = b.run(kvb)
        keep = [i for i in range(30) if not blocks.start <= i < blocks.stop]
        c = Batch([(5, 30)], lambda r: r.integers(1, 60), 8, 2, 64, 16, seed=22)
        c.q[..., 0] = 1
        n = 16 * (blocks.stop - blocks.start)
        c.tables = torch.cat([c.tables[:, keep], c.tables[:, 30:]], 1).contiguous()
        c.lens, c.prefix = c.lens - n, c.prefix - n // 16
        c.check(got)
        assert int(b.status.item()) == 0


@pytest.mark.parametrize("nh,kvh,D,B,t", [(8, 2, 64, 130, "bf16"), (8, 2, 128, 250, "fp16"), (32, 2, 64, 129, "fp16"),
                                          (8, 2, 32, 130, "bf16")])
def test_blocks_that_do_not_fit_a_tile(kvb, cuda, nh, kvh, D, B, t):
    """Block sizes above 128 without runs of 8: whole contexts, the same answers."""
    b = Batch([(4, 3), (3, 0), (5, 2)], mixed, nh, kvh, D, B, t, t, seed=D + B)
    b.check(b.run(kvb))


@pytest.mark.parametrize("nh,kvh,D,t", [(16, 1, 64, "bf16"), (32, 8, 128, "fp16"), (16, 2, 128, "bf16")])
@pytest.mark.parametrize("off", ["q", "out", "both"])
def test_queries_and_outputs_off_16_bytes(kvb, cuda, nh, kvh, D, t, off):
    """They go the way of the decode attention, in a workspace of the size that was asked for without them."""
    import torch
    b = Batch([(6, 9), (2, 0)], mixed, nh, kvh, D, 16, t, t, seed=nh)
    ws = torch.empty(kvb.shared_prefix_workspace_bytes(b.q, b.k, b.tables, b.starts, nh, kvh), dtype=torch.uint8, device="cuda")
    moved = lambda x: torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)  # noqa: E731
    out = torch.zeros_like(b.q)
    if off != "out":
        b.q = moved(b.q)
    if off != "q":
        out = moved(out)
    assert kvb.shared_prefix_attention(*b.args(), out=out, workspace=ws, status=b.status) is out
    b.check(out)


@pytest.mark.parametrize("groups,own,nh,kvh,D,t", [([(2, 1)], lambda r: 30000 + int(r.integers(0, 9)), 32, 8, 128, "bf16"),
                                                   ([(64, 5)], lambda r: 7001 if r.random() < 0.1 else int(r.integers(0, 100)),
                                                    8, 2, 64, "fp16"),
                                                   ([(3, 40), (1, 0)], lambda r: int(10 ** r.uniform(0, 4)), 16, 1, 128, "bf16")])
def test_long_and_uneven_own_parts(kvb, cuda, groups, own, nh, kvh, D, t):
    """Own contexts of thousands of tokens, and of lengths that are orders of magnitude apart."""
    b = Batch(groups, own, nh, kvh, D, 16, t, t, seed=51)
    assert int(b.lens.max()) > 5000
    _check_close(b, b.run(kvb), lift=12)


@pytest.mark.parametrize("groups,change", [([(4, 6), (3, 2), (5, 9)], {1: 8, 2: 4}), ([(4, 6), (3, 6), (5, 6)], {1: 12, 2: 0}),
                                           ([(4, 6), (3, 2), (5, 9)], {1: 99}), ([(2, 3)] * 40, {20: 10}),
                                           ([(2, 3)] * 40, {1: 80, 2: 0, 3: 80, 4: 0}), ([(2, 2)] * 400, {398: 12})])
def test_groups_that_overlap(kvb, cuda, groups, change):
    """A group that starts before the one ahead puts sequences into two groups, whose partial results would mix with those
    of others: all get zeros and the status bit; the next call in the same workspace is as ever."""
    import torch
    b = Batch(groups, few, 8, 2, 64, 16, seed=61)
    ws = torch.empty(kvb.shared_prefix_workspace_bytes(b.q, b.k, b.tables, b.starts, 8, 2), dtype=torch.uint8, device="cuda")
    good, starts = b.run(kvb, workspace=ws), b.starts.clone()
    for i, v in change.items():
        b.starts[i] = v
    got = b.run(kvb, workspace=ws)
    torch.cuda.synchronize()
    assert int(b.status.item()) == kvb.KVP_STATUS_BAD_LEN and bool((got == 0).all())
    b.starts.copy_(starts)
    b.status.zero_()
    assert torch.equal(b.run(kvb, workspace=ws), good)
    b.check(good)
