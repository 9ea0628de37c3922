"""The rotation with append, the shared-prefix attention, the beam selection and the reordering of states running
together in the paged engine (paged-kv-cache-manager_b200/model.py, fused_rope / shared_prefix / beam_search) on a small
random model, against the same model in 64 bits.

Tolerance of logits: a row's hidden state passes about 12 roundings to bf16 per layer (norm, projections, rotation,
probabilities, attention, two residual sums, the MLP's three), each off by up to 2^-8 of its value, 2^-9 / sqrt(3) * 2
= 2^-8 / sqrt(3) in the mean square, and independent.  4 layers: sqrt(48) * 2^-8 / sqrt(3) = 0.016 of the logits' root
mean square.  The largest of 1000 deviations is 3.3 times that, and so is the largest logit: 0.016 of the largest logit,
taken three times for growth through the layers' Jacobians: 0.05."""
import copy
import importlib

import numpy as np
import pytest

TOL = 0.05
VOCAB = 1000


def _model(device, dtype, norms=False):
    import torch
    from transformers import Qwen2Config, Qwen2ForCausalLM
    cfg = Qwen2Config(vocab_size=VOCAB, hidden_size=256, intermediate_size=704, num_hidden_layers=4,
                      num_attention_heads=8, num_key_value_heads=2, head_dim=64, max_position_embeddings=2048,
                      tie_word_embeddings=False)
    torch.manual_seed(0)
    model = Qwen2ForCausalLM(cfg).to(device=device, dtype=dtype).eval()
    truth = copy.deepcopy(model).double()
    if norms:  # the engine reads the attention modules' norms; the 64-bit copy has them behind its projections

        class Norm(torch.nn.Module):
            def __init__(self, weight):
                super().__init__()
                self.weight = torch.nn.Parameter(weight, requires_grad=False)
                self.variance_epsilon = 1e-5

        class Normed(torch.nn.Module):
            def __init__(self, proj, weight):
                super().__init__()
                self.proj, self.w = proj, weight.double()

            def forward(self, x):
                y = self.proj(x).unflatten(-1, (-1, self.w.numel()))
                return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5) * self.w).flatten(-2)

        for la, lb in zip(model.model.layers, truth.model.layers):
            for name in ("q", "k"):
                w = (0.5 + torch.rand(64, device=device)).to(dtype)
                setattr(la.self_attn, name + "_norm", Norm(w))
                setattr(lb.self_attn, name + "_proj", Normed(getattr(lb.self_attn, name + "_proj"), w))
    return model, truth


@pytest.fixture(scope="module")
def models(kvb, cuda):
    import torch
    return {n: _model("cuda", torch.bfloat16, n) for n in (False, True)}


def _engine():
    return importlib.import_module("paged-kv-cache-manager_b200.model").PagedEngine


def _rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).abs().max() / b.abs().max())


def _true(truth, tokens):
    import torch
    with torch.no_grad():
        return truth(torch.tensor([tokens], device="cuda")).logits[0, -1]


@pytest.fixture
def counted(kvb, monkeypatch):
    """How often the engine calls each operator."""
    calls = {}
    for name in ("rope_append", "append_scatter", "paged_attention", "shared_prefix_attention", "beam_select"):
        def call(*args, _fn=getattr(kvb, name), _name=name, **kw):
            calls[_name] = calls.get(_name, 0) + 1
            return _fn(*args, **kw)
        monkeypatch.setattr(kvb, name, call)
    return calls


@pytest.mark.gpu
@pytest.mark.parametrize("norms,shared,block", [(False, True, 16), (True, True, 16), (True, False, 16), (True, True, 8), (False, True, 5)])
def test_requests_that_share_blocks(models, counted, norms, shared, block):
    """Prefill, prefix sharing, a fork in a partial block and batched decode steps in an order in which those that share
    do not adjoin: every step's logits against the 64-bit model."""
    import torch
    model, truth = models[norms]
    r = np.random.default_rng(2)
    base = r.integers(0, VOCAB, 200).tolist()
    eng = _engine()(model, 200, block, fused_rope=True, shared_prefix=shared)
    seqs = {1: base[:97], 2: base[:80] + base[150:157], 3: base[100:101], 4: base[:80] + base[120:140], 5: base[100:137]}
    for i, parent in ((1, None), (2, 1), (3, None), (4, 1), (5, None)):
        lg = eng.prefill(i, seqs[i], parent, 80 if parent else 0)
        assert _rel(lg, _true(truth, seqs[i])) < TOL, i
    eng.fork(6, 1)
    seqs[6] = list(seqs[1])
    rids = [3, 2, 6, 5, 1, 4]
    for step in range(4):
        new = r.integers(0, VOCAB, len(rids)).tolist()
        lg = eng.decode_batch(rids, new)
        for i, t, row in zip(rids, new, lg):
            seqs[i].append(t)
            assert _rel(row, _true(truth, seqs[i])) < TOL, (step, i)
    seqs[2].append(7)
    assert _rel(eng.decode(2, 7), _true(truth, seqs[2])) < TOL
    assert int(eng.status.item()) == 0 and eng.kv.validate() == ""
    assert counted.get("shared_prefix_attention", 0) == (16 if shared else 0)  # 4 steps of 4 layers
    assert "append_scatter" not in counted and counted["rope_append"] == 4 * (5 + 4 + 1)


@pytest.mark.gpu
def test_only_sharing_and_the_order_of_requests(models, counted):
    """shared_prefix without fused_rope (a scatter appends), and the same bits whatever the order of the requests."""
    import torch
    model, truth = models[False]
    base = np.random.default_rng(3).integers(0, VOCAB, 100).tolist()
    got = []
    for order in ([1, 2, 3, 4], [4, 2, 1, 3]):
        eng = _engine()(model, 64, 16, shared_prefix=True)
        for i in (1, 2, 3, 4):
            eng.prefill(i, base[:50] if i < 4 else base[60:90], 1 if 1 < i < 4 else None, 48 if 1 < i < 4 else 0)
        lg = eng.decode_batch(order, [10 * i for i in order])
        got.append({i: row for i, row in zip(order, lg)})
    for i in (1, 2, 3, 4):
        assert torch.equal(got[0][i], got[1][i])
        assert _rel(got[0][i], _true(truth, (base[:50] if i < 4 else base[60:90]) + [10 * i])) < TOL
    assert counted["shared_prefix_attention"] == 8 and "rope_append" not in counted


@pytest.mark.gpu
@pytest.mark.parametrize("beams,eos,block,kw", [(4, None, 16, dict(fused_rope=True, shared_prefix=True)),
                                                (5, 17, 8, dict(fused_rope=True, shared_prefix=True)),
                                                (1, None, 16, dict(fused_rope=True, shared_prefix=True)),
                                                (3, 17, 16, {})])
def test_beam_search(models, counted, kvb, monkeypatch, beams, eos, block, kw):
    """Every step's logits belong to the beams that they are taken for (64-bit model over the beam's own tokens), the
    choices are those of a plain search in 64 bits over the same logits, and the pool is as before at the end."""
    import torch
    model, truth = models[False]
    prompt = np.random.default_rng(4).integers(0, VOCAB, 45).tolist()
    new = 7
    eng = _engine()(model, 64, block, **kw)
    if eos is not None:  # an end that is likely enough to be met: its row of the head follows the best tokens'
        monkeypatch.setattr(eng, "m", copy.deepcopy(model))
        with torch.no_grad():
            first = _true(truth, prompt).topk(2).indices
            eng.m.lm_head.weight[eos] = eng.m.lm_head.weight[first[1]]
        truth = copy.deepcopy(truth)
        truth.lm_head.weight.data[eos] = eng.m.lm_head.weight[eos].double()
    seen, chosen = [], []
    select = kvb.beam_select

    def keep(logits, scores, n, **k):
        out = select(logits, scores, n, **k)
        seen.append((logits.double().cpu(), scores.cpu()))
        chosen.append([t[0].tolist() for t in out])
        return out

    monkeypatch.setattr(kvb, "beam_select", keep)
    rids = list(range(20, 20 + beams))
    found = eng.beam_search(rids, prompt, new, eos)
    assert len(found) == beams and eng.kv.free_blocks() == 64 and eng.kv.validate() == "" and int(eng.status.item()) == 0
    # a plain search over the same logits
    running, done = [(0.0, [])], []
    for step, (lg, sc) in enumerate(seen):
        for row, (s, toks) in enumerate(running):
            assert _rel(lg[row].cuda(), _true(truth, prompt + toks)) < TOL, (step, row)
        assert sc.reshape(-1)[:len(running)].tolist() == [s for s, _ in running]
        lp = torch.log_softmax(lg, -1)[:len(running)] + torch.tensor([s for s, _ in running], dtype=torch.float64)[:, None]
        order = torch.sort(-lp.reshape(-1), stable=True).indices[: beams if eos is None else 2 * beams].tolist()
        value, parent, token = chosen[step]
        assert [(i // VOCAB, i % VOCAB) for i in order] == list(zip(parent, token))
        going = []
        for i, v in enumerate(value):  # the 32-bit sums that the search goes on with: within a rounding of the 64-bit ones
            want = float(lp[parent[i], token[i]])
            assert abs(v - want) <= 2.0 ** -24 * abs(want)
            if token[i] == eos and eos is not None:
                if i < beams:
                    done.append((v, running[parent[i]][1] + [eos]))
            elif len(going) < beams:
                going.append((v, running[parent[i]][1] + [token[i]]))
        running = going
        done = sorted(done, key=lambda e: -e[0])[:beams]
    if len(seen) == new:
        done += running
    else:
        assert len(done) == beams and running[0][0] <= done[-1][0]
    assert found == sorted(done, key=lambda e: -e[0])[:beams]
    assert eos is None or any(t[-1] == eos for _, t in found)
    if kw and beams > 1:
        assert counted["shared_prefix_attention"] == 4 * (len(seen) - 1)
    assert len(chosen) == 1 or beams == 1 or any(p != sorted(set(p)) for _, p, _ in chosen)  # beams did change places


@pytest.mark.gpu
def test_beam_search_without_room(models):
    model, _ = models[False]
    eng = _engine()(model, 4, 16, fused_rope=True, shared_prefix=True)
    assert eng.beam_search([1, 2], list(range(65)), 3) is None and eng.kv.free_blocks() == 4
    with pytest.raises(RuntimeError):  # the prompt fits, its beams' own blocks do not
        eng.beam_search([1, 2], list(range(63)), 5)
    assert eng.kv.free_blocks() == 4 and eng.kv.validate() == ""


def test_refusals(kvb):
    import torch
    model, _ = _model("cpu", torch.bfloat16)
    eng = _engine()(model, 8, 16, fused_rope=True)
    for rids, new, eos in (([], 1, None), (list(range(33)), 1, None), (list(range(17)), 1, 5), ([1, 1], 3, None), ([1], 0, None)):
        with pytest.raises(ValueError):
            eng.beam_search(rids, [1, 2, 3], new, eos)
    with pytest.raises(ValueError):
        eng.beam_search([1], [], 2)
    assert eng.kv.admit(4, 3)
    with pytest.raises(ValueError):
        eng.beam_search([3, 4], [1, 2, 3], 2)
    model.model.rotary_emb.rope_type = "dynamic"
    with pytest.raises(ValueError):
        _engine()(model, 8, 16, fused_rope=True)
    _engine()(model, 8, 16)


@pytest.mark.gpu
def test_a_long_context_among_those_that_share(models, counted):
    """One request whose own context would hold up the shared-prefix attention: the step runs as without the option, with the
    same bits; without that request it goes by groups."""
    import torch
    model, _ = models[False]
    r = np.random.default_rng(4)
    base = r.integers(0, VOCAB, 4000).tolist()
    logits = {}
    for shared in (False, True):
        eng = _engine()(model, 300, 16, shared_prefix=shared)
        assert eng.prefill(1, base[:70]) is not None and eng.prefill(2, base[:64] + base[100:110], 1, 64) is not None
        assert eng.prefill(3, base[:64] + base[200:], 1, 64) is not None
        counted.clear()
        logits[shared] = [eng.decode_batch([3, 2, 1], [5, 6, 7]), eng.decode_batch([2, 1], [8, 9])]
        assert counted.get("shared_prefix_attention", 0) == (4 if shared else 0) and int(eng.status.item()) == 0
    assert torch.equal(logits[True][0], logits[False][0]) and _rel(logits[True][1], logits[False][1]) < TOL
