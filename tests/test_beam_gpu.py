"""Beam selection (kvp_beam_select) against the definition in 64 bits.

Parents and tokens must be equal.  That is decidable: where two continuations of different beams are nearer than the
bound below, the order of the kernel's values is not determined by the formula, so the inputs (fixed seeds) are checked
on the host to have no such pair among the chosen and the next; equal values of one beam are real ties, which go to the
lower token.

Bound of a score: its last rounding is half an ulp, 2^-24 relative.  The sum of exponentials is taken in fp32: each
exponential is off by at most 2 + 1.16 |d| ulps of 2^-23 for an argument d <= 0 (the documented error of the intrinsic),
weighted by its value e^d: at most 3 ulps of the largest term for any d; an addition adds half an ulp, and a lane adds at
most 16 times the steps of its segment plus a rescaling, the warp five more.  So the sum's relative error, which is
the logarithm's absolute one, is at most (16 + 34 steps) 2^-24.  A segment has as many steps of 512 tokens as the row's
steps over the segments it is cut into, at most 32, for about 28 warps on each of 148 processors."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _steps(batch, beams, vocab, select):
    total = -(-(vocab + 7) // 512)
    segments = min((148 * 28 // (batch * beams) + 3) // 4 * 4, 32, total)
    return -(-total // max(1, segments))


def _bound(steps, values):
    return (16 + 34 * steps) * 2.0 ** -24 + np.abs(np.where(np.isfinite(values), values, 0)) * 2.0 ** -24


def _definition(logits, scores, select):
    """numpy, 64 bits: values, parents, tokens."""
    batch, beams = scores.shape
    x = logits.astype(np.float64).reshape(batch, beams, -1)
    x = np.where(x < np.inf, x, -np.inf)  # NaN and +inf are banned
    s = np.where(np.isfinite(scores), scores, -np.inf).astype(np.float64)
    top = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        lse = np.where(np.isfinite(top), top + np.log(np.exp(x - np.where(np.isfinite(top), top, 0)).sum(-1, keepdims=True)), 0)
    v = (s[..., None] + (x - lse)).reshape(batch, -1)
    order = np.argsort(-v, axis=1, kind="stable")
    at = order[:, :select]
    vocab = x.shape[-1]
    vals = np.take_along_axis(v, order[:, :select + 1], 1)
    beam = order[:, :select + 1] // vocab
    with np.errstate(invalid="ignore"):
        gap = vals[:, :-1] - vals[:, 1:]
    steps = _steps(batch, beams, vocab, select)
    near = (beam[:, :-1] != beam[:, 1:]) & np.isfinite(vals[:, 1:]) & (gap < 2 * _bound(steps, vals[:, 1:]))
    assert not near.any(), "the case has two continuations that the formula does not order"
    return np.take_along_axis(v, at, 1), at // vocab, at % vocab


def _check(kvb, logits, scores, select, **kw):
    import torch
    got = kvb.beam_select(logits, scores, select, **kw)
    want = _definition(logits.float().cpu().numpy(), scores.cpu().numpy(), select)
    steps = _steps(*scores.shape, logits.shape[1], select)
    g = got[0].cpu().numpy().astype(np.float64)
    fin = np.isfinite(want[0])
    assert np.array_equal(fin, np.isfinite(g)) and bool((g[~fin] == -np.inf).all())
    assert np.all(np.abs(g[fin] - want[0][fin]) <= _bound(steps, want[0])[fin]), float(np.abs(g[fin] - want[0][fin]).max())
    assert np.array_equal(got[1].cpu().numpy(), want[1]) and np.array_equal(got[2].cpu().numpy(), want[2])
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int32
    return got


def _make(batch, beams, vocab, dtype, seed, banned=0.0, spread=2.5):
    import torch
    r = np.random.default_rng(seed)
    x = (spread * r.standard_normal((batch * beams, vocab))).astype(np.float32)
    x[r.random(x.shape) < banned] = -np.inf
    s = (-5 * r.random((batch, beams))).astype(np.float32)
    return torch.from_numpy(x).to(dtype).cuda(), torch.from_numpy(s).cuda()


@pytest.mark.parametrize("batch,beams,vocab,select", [(1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 5, 15), (1, 4, 1000, 8), (3, 5, 1023, 10),
                                                      (2, 2, 1025, 4), (17, 5, 4099, 10), (1, 32, 700, 32), (3, 8, 32000, 16),
                                                      (1, 1, 151643, 32), (1, 8, 70001, 16), (300, 2, 515, 3)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_against_the_definition(kvb, cuda, batch, beams, vocab, select, dtype):
    import torch
    logits, scores = _make(batch, beams, vocab, getattr(torch, dtype), batch + vocab)
    _check(kvb, logits, scores, select)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("banned", [0.5, 0.999, 1.0])
def test_banned_tokens(kvb, cuda, dtype, banned):
    """Most or all tokens banned: continuations of value -inf fill up in order of beam and token."""
    import torch
    logits, scores = _make(4, 3, 3001, getattr(torch, dtype), 7, banned)
    logits[4] = -math.inf  # a row that its mask leaves empty
    logits[5, 10:] = -math.inf
    _check(kvb, logits, scores, 20)


def test_lowest_value_masks(kvb, cuda):
    """Masks of the type's lowest value instead of -inf are ordinary, very unlikely tokens."""
    import torch
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits, scores = _make(2, 2, 2000, dtype, 3)
        logits[0, 3:] = torch.finfo(dtype).min
        logits[1] = torch.finfo(dtype).min
        scores[1, 1] = -50
        _check(kvb, logits, scores, 6)


def test_first_step_and_unused_beams(kvb, cuda):
    import torch
    logits, scores = _make(3, 4, 9000, torch.bfloat16, 11)
    scores[:, 1:] = -math.inf
    got = _check(kvb, logits, scores, 8)
    assert bool((got[1] == 0).all())
    scores[1] = -math.inf  # a request without a live beam
    _check(kvb, logits, scores, 8)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_ties_go_to_the_lower_beam_and_token(kvb, cuda, dtype):
    """Equal logits everywhere, equal rows, and few distinct values."""
    import torch
    dt = getattr(torch, dtype)
    for vocab in (40, 2048, 5000):
        x = torch.zeros((4, vocab), device="cuda", dtype=dt)
        s = torch.zeros((2, 2), device="cuda")
        got = kvb.beam_select(x, s, 9)
        assert got[1].tolist() == [[0] * 9] * 2 and got[2].tolist() == [list(range(9))] * 2
    r = np.random.default_rng(5)
    x = torch.from_numpy(r.integers(0, 4, (6, 5003)).astype(np.float32)).to(dt).cuda()
    s = torch.tensor([[-1.0, -1.5, -0.75], [-2.0, -0.25, -9.0]], device="cuda")
    _check(kvb, x, s, 32)
    x[1] = x[0]  # the same row under two beams of one score: the lower beam first
    s[0] = torch.tensor([-1.0, -1.0, -5.0])
    v, p, t = kvb.beam_select(x, s, 32)
    first = (x[0] == 3).nonzero()[:32, 0].tolist()
    assert p[0].tolist().count(0) == 32 and t[0].tolist() == first
    # +0 and -0 are one value
    z = torch.zeros((1, 300), device="cuda", dtype=dt)
    z[0, ::2] = -0.0
    assert kvb.beam_select(z, torch.zeros((1, 1), device="cuda"), 5)[2].tolist() == [[0, 1, 2, 3, 4]]


def test_nan_and_infinity_are_reported_and_banned(kvb, cuda):
    import torch
    logits, scores = _make(2, 3, 4000, torch.float32, 21)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check(kvb, logits, scores, 6, status=status)
    assert int(status.item()) == 0
    for at, value in ((3, math.nan), (3999, math.inf), (2047, math.nan)):
        bad = logits.clone()
        bad[2, at] = value
        bad[2, at - 1] = math.inf
        status.zero_()
        _check(kvb, bad, scores, 6, status=status)
        assert int(status.item()) == kvb.KVP_STATUS_BAD_VALUE
    for value in (math.nan, math.inf):
        bad = scores.clone()
        bad[1, 0] = value
        status.zero_()
        _check(kvb, logits, bad, 6, status=status)
        assert int(status.item()) == kvb.KVP_STATUS_BAD_VALUE


def test_large_values(kvb, cuda):
    import torch
    logits, scores = _make(1, 2, 3000, torch.float32, 2, spread=1e4)
    _check(kvb, logits, scores, 4)
    logits[0, :8] = 3e38  # the finiteness check must not trip over a sum
    logits[0, 8:16] = -3e38
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check(kvb, logits, scores, 4, status=status)
    assert int(status.item()) == 0


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_strided_and_unaligned_rows(kvb, cuda, dtype):
    """Rows of a wider buffer from an odd column; what lies around them is NaN and is not read as a logit."""
    import torch
    dt = getattr(torch, dtype)
    logits, scores = _make(2, 2, 2500, dt, 8)
    for left, right in ((1, 0), (3, 4), (5, 1), (8, 3)):
        wide = torch.full((4, left + 2500 + right), math.nan, device="cuda", dtype=dt)
        wide[:, left:left + 2500] = logits
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        _check(kvb, wide[:, left:left + 2500], scores, 7, status=status)
        assert int(status.item()) == 0


def test_stream_graph_workspace(kvb, cuda):
    """Another stream, a kept workspace full of garbage, a captured graph replayed on new inputs, and two graphs that
    share the workspace, one after the other."""
    import torch
    a, sa = _make(3, 4, 20000, torch.bfloat16, 1)
    b, sb = _make(3, 4, 20000, torch.bfloat16, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kvb.beam_select(a, sa, 8, stream=side)
    side.synchronize()
    want_a, want_b = _check(kvb, a, sa, 8), _check(kvb, b, sb, 8)
    assert all(torch.equal(x, y) for x, y in zip(got, want_a))
    ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
    assert all(torch.equal(x, y) for x, y in zip(kvb.beam_select(a, sa, 8, workspace=ws), want_a))
    graphs = []
    for x, s in ((a.clone(), sa), (b, sb)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kvb.beam_select(x, s, 8, workspace=ws)
        graphs.append((g, out, x))
    for g, _, _ in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], want_a))
    assert all(torch.equal(x, y) for x, y in zip(graphs[1][1], want_b))
    graphs[0][2].copy_(b)
    sa.copy_(sb)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], want_b))


def test_same_answer_every_time(kvb, cuda):
    """No atomics decide anything: repeated calls agree to the bit."""
    import torch
    x, s = _make(5, 8, 30011, torch.float16, 4)
    first = kvb.beam_select(x, s, 16)
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(kvb.beam_select(x, s, 16), first))


def test_refusals_and_empty(kvb, cuda):
    import torch
    x, s = _make(2, 4, 100, torch.float32, 1)
    for bad in (lambda: kvb.beam_select(x, s, 0), lambda: kvb.beam_select(x, s, 33), lambda: kvb.beam_select(x, s.double(), 4),
                lambda: kvb.beam_select(x[:7], s, 4), lambda: kvb.beam_select(x.t(), s, 4), lambda: kvb.beam_select(x.long(), s, 4),
                lambda: kvb.beam_select(x.cpu(), s, 4), lambda: kvb.beam_select(x.expand(8, 100)[:1].expand(8, 100), s, 4),
                lambda: kvb.beam_select(x[:, :2].contiguous(), s, 9)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(kvb.KVPError):
        kvb.beam_select(x, s, 4, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    out = kvb.beam_select(x[:0], s[:0], 4)
    assert [tuple(t.shape) for t in out] == [(0, 4)] * 3


def test_numbers_that_pass_32_bits(kvb, cuda):
    import torch
    x, s = torch.zeros(2, 8, device="cuda"), torch.zeros(1, 2, device="cuda")
    for select in (2 ** 32 + 3, 2 ** 31, -2 ** 40):
        with pytest.raises(ValueError):
            kvb.beam_select(x, s, select)
    with pytest.raises(ValueError):  # 2^32 + 8 tokens are not 8
        kvb.beam_select(torch.zeros(1, 2 ** 32 + 8, dtype=torch.half, device="cuda"), s[:, :1], 3)


def test_status_words_of_other_types(kvb, cuda):
    import torch
    x, s = torch.zeros(2, 8, device="cuda"), torch.zeros(1, 2, device="cuda")
    for bad in (torch.zeros(4, dtype=torch.uint8, device="cuda")[1:], torch.zeros(0, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            kvb.beam_select(x, s, 3, status=bad)
        with pytest.raises(ValueError):
            kvb.qk_norm_rope(torch.zeros(1, 1, 16, device="cuda"), torch.zeros(1, 1, 16, device="cuda"),
                             torch.zeros(1, dtype=torch.int32, device="cuda"), kvb.rope_table(1, 16), status=bad)
