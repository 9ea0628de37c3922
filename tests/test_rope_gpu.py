"""Rotation, head norms and append in one pass (kvp_rope_append) against the formulas in 64 bits.

Tolerance of a rotated element, from the arithmetic: the kernel computes in fp32 what the formula computes in 64 bits
from the same inputs and the same fp32 table.  A normed element carries at most: half an ulp for each of the square
sum's terms and additions (non-negative terms: a relative error of at most (dim / 2 + 6) half-ulps, halved by the root
and bounded here by dim / 2), the root, the quotient and two products, 8 more.  The rotation adds two products and a
sum, 3 half-ulps of |x0| + |x1|.  Half an ulp of fp32 is 2^-24 relative, so the error before the last rounding is at most
(dim / 2 + 16) 2^-24 (|x0| + |x1|); the rounding to the output's type adds half a step of the result, eps / 2 relative,
and for fp16 results below 2^-14 an absolute 2^-25.  Values are copied bit for bit."""
import math

import pytest

pytestmark = pytest.mark.gpu

DT = {"bf16": "bfloat16", "fp16": "float16", "fp32": "float32"}


def _dt(name):
    import torch
    return getattr(torch, DT[name])


def _formula(x, table, pos, rot, norm, eps, interleaved):
    """The formula in 64 bits, and |x0| + |x1| of each element's pair."""
    import torch
    x = x.double()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    half = rot // 2
    row = table.double()[pos.long()][:, None]
    c, s = row[..., :half], row[..., half:]
    y, mag = x.clone(), x.abs()
    ia = torch.arange(0, rot, 2, device=x.device) if interleaved else torch.arange(half, device=x.device)
    ib = ia + 1 if interleaved else ia + half
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


def _close(got, want, mag, dim, what):
    import torch
    tol = want.abs() * (torch.finfo(got.dtype).eps / 2) + (dim / 2 + 16) * 2.0 ** -24 * mag
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = (got.double() - want).abs() - tol
    assert bool(torch.isfinite(got).all()) and float(err.max()) <= 0, (what, float(err.max()))


def _inputs(n, nh, kvh, D, dtype, seed, norm, fused, far=300):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if fused:
        qkv = r(n, (nh + 2 * kvh) * D).to(dtype)
        q, k, v = (t.view(n, -1, D) for t in qkv.split([nh * D, kvh * D, kvh * D], 1))
    else:
        q, k, v = r(n, nh, D).to(dtype), r(n, kvh, D).to(dtype), r(n, kvh, D).to(dtype)
    pos = torch.randint(0, far, (n,), generator=g, device="cuda", dtype=torch.int32)
    w = [(1 + 0.3 * r(D)).to(dtype) for _ in range(2)] if norm else [None, None]
    return q, k, v, pos, w, g


CASES = [
    # n, heads, kv heads, dim, rot, in, pool, out, norm, interleaved, block
    (1, 32, 8, 128, 128, "bf16", "bf16", "bf16", False, False, 16),
    (1, 1, 1, 16, 16, "fp16", "fp16", "fp16", True, True, 1),
    (3, 14, 2, 64, 64, "fp16", "fp16", "fp16", False, False, 16),
    (17, 32, 4, 64, 32, "bf16", "bf16", "bf16", True, True, 5),
    (64, 8, 8, 64, 48, "bf16", "fp16", "fp32", True, False, 3),
    (5, 7, 7, 96, 96, "fp32", "bf16", "fp32", True, False, 16),
    (5, 6, 3, 80, 32, "fp32", "fp16", "bf16", False, True, 7),
    (33, 4, 1, 256, 256, "bf16", "bf16", "fp16", True, False, 32),
    (9, 5, 1, 256, 16, "fp16", "bf16", "fp16", True, True, 32),
    (2501, 14, 2, 64, 64, "fp16", "fp16", "fp16", True, False, 16),
    (4999, 32, 8, 128, 128, "bf16", "bf16", "bf16", False, False, 16),
]


@pytest.mark.parametrize("n,nh,kvh,D,rot,din,dkv,dout,norm,inter,B", CASES)
@pytest.mark.parametrize("fused", [False, True])
def test_rope_append_against_the_formula(kvb, cuda, n, nh, kvh, D, rot, din, dkv, dout, norm, inter, B, fused):
    import torch
    q, k, v, pos, (qw, kw), g = _inputs(n, nh, kvh, D, _dt(din), n * 7 + D, norm, fused)
    table = kvb.rope_table(300, rot, base=10000.0)
    nb = -(-2 * n // B) + 2
    pools = [torch.full((nb, B, kvh, D), math.nan, device="cuda", dtype=_dt(dkv)) for _ in range(2)]
    slots = torch.randperm(nb * B, generator=g, device="cuda")[:n].to(torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = torch.empty((n, nh, D), dtype=_dt(dout), device="cuda")
    k_out = torch.empty((n, kvh, D), dtype=_dt(dout), device="cuda")
    got = kvb.rope_append(q, k, v, pos, table, *pools, slots, q_out=q_out, k_out=k_out, q_norm=qw, k_norm=kw, eps=1e-5,
                          interleaved=inter, status=status)
    assert got is q_out and int(status.item()) == 0
    wq, mq = _formula(q, table, pos, rot, qw, 1e-5, inter)
    wk, mk = _formula(k, table, pos, rot, kw, 1e-5, inter)
    _close(q_out, wq, mq, D, "q")
    _close(k_out, wk, mk, D, "k_out")
    flat = [p.view(nb * B, kvh, D) for p in pools]
    _close(flat[0][slots.long()], wk, mk, D, "k cache")
    assert torch.equal(flat[1][slots.long()], v.to(_dt(dkv)))
    rest = torch.ones(nb * B, dtype=torch.bool, device="cuda")
    rest[slots.long()] = False
    assert all(bool(f[rest].isnan().all()) for f in flat)  # nothing else is written


@pytest.mark.parametrize("n", [1, 40, 3001])
def test_without_a_cache_and_in_place(kvb, cuda, n):
    """qk_norm_rope equals the append form bit for bit, and so does the rotation in place inside the fused rows."""
    import torch
    q, k, v, pos, (qw, kw), g = _inputs(n, 12, 4, 128, torch.bfloat16, 5, True, True)
    table = kvb.rope_table(300, 64, base=500000.0)
    a, b = kvb.qk_norm_rope(q, k, pos, table, q_norm=qw, k_norm=kw)
    pools = [torch.zeros((n, 1, 4, 128), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    c = kvb.rope_append(q, k, v, pos, table, *pools, slots, q_norm=qw, k_norm=kw)
    assert torch.equal(a, c) and torch.equal(pools[0].view(n, 4, 128)[slots.long()], b)
    keep = v.clone()
    kvb.qk_norm_rope(q, k, pos, table, q_out=q, k_out=k, q_norm=qw, k_norm=kw)
    assert torch.equal(a, q) and torch.equal(b, k) and torch.equal(v, keep)


def test_padded_uncached_and_bad_rows(kvb, cuda):
    """Padding (negative position) is left alone; a negative slot is rotated, not cached; a slot or a position out of
    range is reported and skipped."""
    import torch
    n, nh, kvh, D, B, nb = 8, 4, 2, 64, 4, 6
    q, k, v, pos, _, _ = _inputs(n, nh, kvh, D, torch.bfloat16, 3, False, False, far=50)
    table = kvb.rope_table(50, D)
    slots = torch.tensor([0, 5, -1, 7, nb * B, 9, 11, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    for bad_pos, want in ((None, kvb.KVP_STATUS_BAD_BLOCK), (50, kvb.KVP_STATUS_BAD_BLOCK | kvb.KVP_STATUS_BAD_POSITION)):
        p = pos.clone()
        p[6] = -1
        if bad_pos:
            p[3] = bad_pos
        pools = [torch.full((nb, B, kvh, D), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((n, nh, D), 7.0, device="cuda", dtype=torch.bfloat16)
        kvb.rope_append(q, k, v, p, table, *pools, slots, q_out=out, status=status)
        skipped = [6] + ([3] if bad_pos else [])
        rows = [i for i in range(n) if i not in skipped]
        wq, mq = _formula(q, table, p.clamp(0, 49), D, None, 0, False)
        _close(out[rows], wq[rows], mq[rows], D, "q")
        assert bool((out[skipped] == 7).all())
        written = {int(slots[i]) for i in rows if 0 <= int(slots[i]) < nb * B}
        flat = pools[1].view(nb * B, kvh, D)
        for s in range(nb * B):
            i = [j for j in rows if int(slots[j]) == s]
            assert torch.equal(flat[s], v[i[0]]) if s in written else bool((flat[s] == 7).all())
        assert int(status.item()) == want


def test_far_positions_and_long_offsets(kvb, cuda):
    """Positions at the end of a long table; a slot whose element offset passes 2^31."""
    import torch
    n, nh, kvh, D, B = 4, 2, 8, 128, 16
    far = 1 << 20
    table = kvb.rope_table(far, D, base=500000.0)
    want = (far - 1) * torch.tensor(500000.0, dtype=torch.float64) ** -(torch.arange(0, D, 2, dtype=torch.float64) / D)
    assert float((table[-1].double().cpu() - torch.cat([want.cos(), want.sin()])).abs().max()) < 2.0 ** -24 + 1e-9
    nb = (2 ** 31 + 2 ** 22) // (B * kvh * D)  # 4.3 GB a pool
    pools = [torch.empty((nb, B, kvh, D), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    q, k, v, pos, _, _ = _inputs(n, nh, kvh, D, torch.bfloat16, 9, False, False)
    pos += far - 300
    slots = torch.tensor([nb * B - 1, 0, nb * B - 17, 5], dtype=torch.int32, device="cuda")
    kvb.rope_append(q, k, v, pos, table, *pools, slots)
    wk, mk = _formula(k, table, pos, D, None, 0, False)
    at = [(int(s) // B, int(s) % B) for s in slots]
    _close(torch.stack([pools[0][b, o] for b, o in at]), wk, mk, D, "k cache")
    assert torch.equal(torch.stack([pools[1][b, o] for b, o in at]), v)


def test_llama3_shape_matches_the_model_library(kvb, cuda):
    """The half-split rotation is the one of the model library's rotary embedding (its cos/sin in fp32)."""
    import torch
    from transformers.models.llama.modeling_llama import apply_rotary_pos_emb
    n, nh, kvh, D = 6, 4, 2, 64
    q, k, _, pos, _, _ = _inputs(n, nh, kvh, D, torch.float32, 1, False, False)
    table = kvb.rope_table(300, D)
    c, s = table[pos.long()].chunk(2, 1)
    cos, sin = torch.cat([c, c], 1)[None], torch.cat([s, s], 1)[None]
    hq, hk = apply_rotary_pos_emb(q.transpose(0, 1)[None], k.transpose(0, 1)[None], cos, sin)
    gq, gk = kvb.qk_norm_rope(q, k, pos, table)
    torch.testing.assert_close(gq, hq[0].transpose(0, 1), rtol=2e-6, atol=2e-6)
    torch.testing.assert_close(gk, hk[0].transpose(0, 1), rtol=2e-6, atol=2e-6)


def test_side_stream_graph_and_empty(kvb, cuda):
    import torch
    q, k, v, pos, _, _ = _inputs(20, 8, 2, 64, torch.float16, 4, False, True)
    table = kvb.rope_table(300, 64)
    pools = [torch.zeros((20, 1, 2, 64), device="cuda", dtype=torch.float16) for _ in range(2)]
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    want = kvb.rope_append(q, k, v, pos, table, *pools, slots)
    ref = [p.clone() for p in pools]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kvb.rope_append(q, k, v, pos, table, *pools, slots, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.full_like(want, 7.0)
    with torch.cuda.graph(graph):
        kvb.rope_append(q, k, v, pos, table, *pools, slots, q_out=out)
    for p in pools:
        p.zero_()
    pos2 = pos.clone()
    pos.add_(1)  # the graph reads its inputs again
    graph.replay()
    torch.cuda.synchronize()
    inside = pos2 + 1 < 300  # one of the positions moves past the table: its row is skipped
    again = kvb.rope_append(q, k, v, pos2 + 1, table, *[p.clone() for p in pools], slots)
    assert int(inside.sum()) == 19 and torch.equal(out[inside], again[inside]) and bool((out[~inside] == 7).all())
    assert torch.equal(pools[1][inside], ref[1][inside]) and not torch.equal(pools[0], ref[0])
    empty = kvb.rope_append(q[:0], k[:0], v[:0], pos[:0], table, *pools, slots[:0])
    assert empty.shape == (0, 8, 64)


def test_refusals(kvb, cuda):
    import torch
    q, k, v, pos, _, _ = _inputs(4, 8, 2, 64, torch.bfloat16, 4, False, False)
    table = kvb.rope_table(300, 64)
    pools = [torch.zeros((4, 1, 2, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    call = lambda **kw: kvb.rope_append(**{**dict(q=q, k=k, v=v, positions=pos, table=table, k_cache=pools[0],  # noqa: E731
                                                  v_cache=pools[1], slots=slots), **kw})
    off = torch.zeros(4 * 8 * 64 + 8, device="cuda", dtype=torch.bfloat16)[1:4 * 8 * 64 + 1].view(4, 8, 64)
    for bad in (dict(q=q.transpose(0, 1)), dict(k=k.float()), dict(positions=pos.long()), dict(positions=pos[:3]),
                dict(slots=slots[:2]), dict(v=v[:, :1]), dict(table=table.half()), dict(table=table[:, :24].contiguous()),
                dict(table=kvb.rope_table(9, 80)), dict(q=q.cpu()), dict(k_cache=pools[0][:, :, :1]), dict(q=off),
                dict(q_norm=torch.ones(64, device="cuda")), dict(q_norm=torch.ones(32, device="cuda").bfloat16()),
                dict(q_out=torch.empty(4, 8, 32, device="cuda")), dict(v=None), dict(slots=None), dict(eps=-1.0, q_norm=torch.ones(
                    64, device="cuda").bfloat16())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError):
        kvb.qk_norm_rope(q, k, pos, table, k_out=torch.empty(4, 2, 64, device="cuda"))


def test_slots_behind_32_bit_offsets(kvb, cuda):
    """Slots at the end of pools of more than 2^32 elements hold what the same call stores in a small pool."""
    import torch
    n, B, kvh, D = 40, 16, 8, 128
    q, k, v = (torch.randn(n, h, D, device="cuda", dtype=torch.bfloat16) for h in (32, kvh, kvh))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    table = kvb.rope_table(n, D)
    slots = torch.randperm(3 * B, device="cuda")[:n].int()
    many = (1 << 32) // (B * kvh * D) + 100
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    small = [torch.zeros(3, B, kvh, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    big = [torch.empty(many, B, kvh, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    for x in big:
        x[-3:].zero_()
    a = kvb.rope_append(q, k, v, pos, table, *small, slots, status=status)
    b = kvb.rope_append(q, k, v, pos, table, *big, slots + (many - 3) * B, status=status)
    assert torch.equal(a, b) and int(status.item()) == 0
    for x, y in zip(small, big):
        assert torch.equal(x, y[-3:])


def test_rows_that_several_tokens_share_are_refused(kvb, cuda):
    """Inputs and outputs that are expanded over the tokens hold one row, not as many as there are tokens."""
    import torch
    q, k, v, pos, _, _ = _inputs(4, 8, 2, 64, torch.bfloat16, 4, False, False)
    table = kvb.rope_table(300, 64)
    pools = [torch.zeros((4, 1, 2, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    one = lambda t: t[:1].clone().expand(4, -1, -1)  # noqa: E731
    for bad in (dict(q=one(q)), dict(k=one(k)), dict(v=one(v)), dict(q_out=one(q)), dict(k_out=one(k))):
        with pytest.raises(ValueError, match="overlap"):
            kvb.rope_append(**{**dict(q=q, k=k, v=v, positions=pos, table=table, k_cache=pools[0], v_cache=pools[1],
                                      slots=slots), **bad})
    for bad in (dict(q=one(q)), dict(k=one(k)), dict(q_out=one(q)), dict(k_out=one(k))):
        with pytest.raises(ValueError, match="overlap"):
            kvb.qk_norm_rope(**{**dict(q=q, k=k, positions=pos, table=table), **bad})
