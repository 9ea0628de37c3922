"""Cases for measuring the serving operators that surround the paged cache, and their plain forms.

Three operators, as one decode step of parallel sampling or beam search uses them one after the other:

  rope    the rows of one layer's fused QKV projection: RMS norms of each query and key head (where the model has
          them), position rotation from a cos/sin table, the queries written out, keys and values put into their
          slots of the paged cache
  prefix  decode attention of a batch in groups whose sequences share their leading cache blocks
  beam    the best continuations over beams and vocabulary from logits and running scores

With `own` false, `run` computes them from elementary torch operations; with `own` true it calls the library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def _kvb():
    import importlib
    return importlib.import_module("paged-kv-cache-manager_b200")


# ---------------------------------------------------------------------------------------------------- cases
def _rope(name, tokens, heads, kv_heads, dim, dtype, *, norm=False, cache=True, rot=None, interleaved=False, block=16,
          start=0, pad=0):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "norm": norm, "cache": cache, "rot": rot or dim, "interleaved": interleaved, "block": block, "start": start,
            "pad": pad}


def _prefix(name, groups, members, prefix, suffix, heads, kv_heads, dim, dtype, *, ragged=False, block=16):
    return {"name": name, "op": "prefix", "groups": groups, "members": members, "prefix": prefix, "suffix": suffix,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "ragged": ragged, "block": block}


def _beam(name, batch, beams, select, vocab, dtype, *, banned=0.0, first=False):
    return {"name": name, "op": "beam", "batch": batch, "beams": beams, "select": select, "vocab": vocab, "dtype": dtype,
            "banned": banned, "first": first}


def listed():
    return [
        # one request's next token at the Llama-3-8B head shape, far into its context
        _rope("rope_one_token", 1, 32, 8, 128, "bf16", start=8000),
        # a decode step of 256 requests, the last 19 rows of the captured batch being padding
        _rope("rope_decode_256", 256, 32, 8, 128, "bf16", start=4096, pad=19),
        # a prompt chunk at the Qwen2.5-0.5B head shape, fp16, of an odd length
        _rope("rope_prompt_2047", 2047, 14, 2, 64, "fp16", start=512),
        # a long prompt with normed query and key heads
        _rope("rope_norm_prompt_16384", 16384, 32, 8, 128, "bf16", norm=True),
        # the same pass without a cache behind it (what a step's fused append takes),
        # interleaved pairs over half of each head
        _rope("norm_rope_only_1111", 1111, 32, 4, 64, "bf16", norm=True, cache=False, rot=32, interleaved=True),
        # four beams of one request over its 2048-token prompt, a few tokens in
        _prefix("prefix_4_beams", 1, 4, 2048, 24, 32, 8, 128, "bf16"),
        # 16 conversations of different sizes, each over its own system prompt, TinyLlama's head shape
        _prefix("prefix_16_groups", 16, 17, 4000, 700, 32, 4, 64, "fp16", ragged=True),
        # parallel samples over the 2048-token shared prefix, 64 requests by 8 samples
        _prefix("prefix_512_samples", 1, 512, 2048, 100, 32, 8, 128, "bf16", ragged=True),
        # a whole batch asking about one long document
        _prefix("prefix_256_over_16384", 1, 256, 16384, 512, 32, 8, 128, "bf16", ragged=True),
        # the first step of one request's beam search: one live beam
        _beam("beam_first_step", 1, 4, 8, 32000, "bf16", first=True),
        # a batch of searches with a grammar's banned tokens, odd vocabulary
        _beam("beam_17x5_banned", 17, 5, 10, 50257, "fp16", banned=0.3),
        # a large batch of wide searches over a large vocabulary, fp32 logits
        _beam("beam_64x8", 64, 8, 16, 128000, "fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


SHAPES = [(8, 8, 64), (14, 2, 64), (32, 4, 64), (32, 8, 128)]


def draw(rng):
    op = rng.choice(["rope", "rope", "prefix", "prefix", "prefix", "beam", "beam"])
    heads, kv_heads, dim = rng.choice(SHAPES)
    dtype = rng.choice(["bf16", "fp16"])
    block = rng.choice([8, 16, 16, 16, 32, 5])
    if op == "rope":
        norm, cache = rng.random() < 0.5, rng.random() < 0.75
        c = _rope("", _log(rng, 1, 16000), heads, kv_heads, dim, dtype, norm=norm, cache=cache,
                  rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, block=block, start=_log(rng, 1, 30000))
    elif op == "prefix":
        groups = _log(rng, 1, 32)
        members = max(2, _log(rng, 2, 400) // groups)
        total = 256 * 16384  # rows times context of the largest listed case
        prefix = min(_log(rng, 64, 16000), total // (groups * members))
        suffix = min(_log(rng, 1, 1500), 100000 // (groups * members))
        c = _prefix("", groups, members, max(prefix, 64), max(suffix, 1), heads, kv_heads, dim, dtype,
                    ragged=rng.random() < 0.7, block=block)
    else:
        beams = rng.randint(1, 8)
        c = _beam("", _log(rng, 1, 60), beams, min(16, rng.randint(beams, 2 * beams)), _log(rng, 1000, 120000),
                  rng.choice(["bf16", "fp16", "fp32"]), banned=rng.choice([0.0, 0.0, 0.5]), first=rng.random() < 0.2)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(lo, hi, n, g):
    """n whole numbers of [lo, hi]."""
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV)


def _prepare_rope(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    n, nh, kvh, d, b = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["block"]
    qkv = torch.randn((n, (nh + 2 * kvh) * d), generator=g, device=DEV).to(dt)
    rot, far = c["rot"], c["start"] + n + 64
    freq = 1.0 / (500000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot))
    angle = torch.arange(far, dtype=torch.float64, device=DEV)[:, None] * freq
    s = {"op": "rope", "qkv": qkv, "table": torch.cat([angle.cos(), angle.sin()], 1).float().contiguous(), "heads": nh,
         "kv_heads": kvh, "dim": d, "rot": rot, "interleaved": c["interleaved"], "eps": 1e-6}
    if n >= 1000:  # a prompt: consecutive positions
        pos = c["start"] + torch.arange(n, device=DEV)
    else:  # a decode step: every token at its own request's length
        pos = _ints(c["start"] // 2, c["start"] + n, n, g)
    s["positions"] = pos.to(torch.int32)
    if c["norm"]:
        s["q_norm"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt)
        s["k_norm"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt)
    if c["cache"]:
        blocks = -(-2 * n // b) + 3
        s["k_cache"] = torch.randn((blocks, b, kvh, d), generator=g, device=DEV).to(dt)
        s["v_cache"] = torch.randn((blocks, b, kvh, d), generator=g, device=DEV).to(dt)
        if n >= 1000:  # whole blocks in a random order
            table = torch.randperm(blocks, generator=g, device=DEV)
            at = torch.arange(n, device=DEV)
            slots = table[at // b] * b + at % b
        else:
            slots = torch.randperm(blocks * b, generator=g, device=DEV)[:n]
        if c["pad"]:
            slots[n - c["pad"]:] = -1
        s["slots"] = slots.to(torch.int32)
    return s


def _prefix_lens(c, seed):
    """Members, prefix tokens of every group and suffix tokens of every sequence, on the host."""
    r = torch.Generator().manual_seed(seed)
    groups, b = c["groups"], c["block"]
    if c["ragged"]:
        members = torch.randint(max(1, c["members"] // 3), c["members"] + 1, (groups,), generator=r)
        members[0] = c["members"]
        prefix = torch.randint(max(1, c["prefix"] // 8), c["prefix"] + 1, (groups,), generator=r)
        prefix[0] = c["prefix"]
        suffix = torch.randint(1, c["suffix"] + 1, (int(members.sum()),), generator=r)
    else:
        members = torch.full((groups,), c["members"])
        prefix = torch.full((groups,), c["prefix"])
        suffix = torch.full((groups * c["members"],), c["suffix"])
    return members, prefix // b, suffix  # only whole blocks are shared


def _prepare_prefix(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    nh, kvh, d, b = c["heads"], c["kv_heads"], c["dim"], c["block"]
    # sizes are the case's own, the values the seed's
    members, pblocks, suffix = _prefix_lens(c, 1234)
    groups, ns = c["groups"], int(members.sum())
    group = torch.repeat_interleave(torch.arange(groups), members)
    sblocks = -(-suffix // b)
    pstart = torch.cumsum(pblocks, 0) - pblocks
    sstart = int(pblocks.sum()) + torch.cumsum(sblocks, 0) - sblocks
    blocks = int(pblocks.sum() + sblocks.sum()) + 5
    width = int((pblocks[group] + sblocks).max()) + 1
    col = torch.arange(width)[None]
    pb = pblocks[group][:, None]
    logical = torch.where(col < pb, pstart[group][:, None] + col, sstart[:, None] + col - pb)
    used = col < pb + sblocks[:, None]
    perm = torch.randperm(blocks, generator=g, device=DEV)
    tables = torch.where(used.to(DEV), perm[logical.clamp(0, blocks - 1).to(DEV)], 0)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(members, 0)])
    i32 = lambda t: t.to(device=DEV, dtype=torch.int32)  # noqa: E731
    return {"op": "prefix", "heads": nh, "kv_heads": kvh, "dim": d, "block": b,
            "q": torch.randn((ns, nh, d), generator=g, device=DEV).to(dt),
            "k_cache": torch.randn((blocks, b, kvh, d), generator=g, device=DEV).to(dt),
            "v_cache": torch.randn((blocks, b, kvh, d), generator=g, device=DEV).to(dt),
            "tables": i32(tables), "lens": i32(pblocks[group] * b + suffix), "prefix_blocks": i32(pblocks[group]),
            "starts": i32(starts), "most_members": int(members.max()), "most_prefix": int(pblocks.max()) * b,
            "most_suffix": int(suffix.max())}


def _prepare_beam(c, seed):
    g = _gen(seed)
    rows = c["batch"] * c["beams"]
    logits = torch.randn((rows, c["vocab"]), generator=g, device=DEV).mul_(2.5)
    if c["banned"]:
        logits.masked_fill_(torch.rand((rows, c["vocab"]), generator=g, device=DEV) < c["banned"], -math.inf)
    scores = -5.0 * torch.rand((c["batch"], c["beams"]), generator=g, device=DEV)
    if c["first"]:
        scores[:, 1:] = -math.inf
        scores[:, 0] = 0
    return {"op": "beam", "logits": logits.to(DTYPES[c["dtype"]]), "scores": scores, "select": c["select"]}


def prepare(case, seed):
    return {"rope": _prepare_rope, "prefix": _prepare_prefix, "beam": _prepare_beam}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------------- plain forms
def _split(s):
    nh, kvh, d = s["heads"], s["kv_heads"], s["dim"]
    n = s["qkv"].shape[0]
    q, k, v = s["qkv"].split([nh * d, kvh * d, kvh * d], 1)
    return q.view(n, nh, d), k.view(n, kvh, d), v.view(n, kvh, d)


def _rotate(x, s, norm):
    """RMS norm of each head, where there are weights, and the rotation, in 32 bits."""
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * norm.float()
    rot, half = s["rot"], s["rot"] // 2
    cs = s["table"][s["positions"].long()]
    cos, sin = cs[:, None, :half], cs[:, None, half:]
    if s["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope(s):
    q, k, v = _split(s)
    dt = q.dtype
    q_out, k_out = _rotate(q, s, s.get("q_norm")).to(dt), _rotate(k, s, s.get("k_norm")).to(dt)
    if "slots" not in s:
        return q_out, k_out
    kc, vc = (t.view(-1, s["kv_heads"], s["dim"]) for t in (s["k_cache"], s["v_cache"]))
    # a padded row has slot -1 and goes nowhere: it rewrites what the first row puts into its slot
    slots = s["slots"].long()
    real = (slots >= 0)[:, None, None]
    slots = torch.where(slots >= 0, slots, slots[0])
    kc[slots] = torch.where(real, k_out, k_out[:1])
    vc[slots] = torch.where(real, v, v[:1])
    return q_out, s["k_cache"], s["v_cache"]


def _plain_prefix(s):
    """Scores over the shared blocks once for a whole group, over each sequence's own blocks beside them, one
    softmax over both, in 32 bits."""
    ns, nh, d = s["q"].shape
    kvh, b = s["kv_heads"], s["block"]
    per, dev = nh // kvh, s["q"].device
    tables, lens, pb = s["tables"].long(), s["lens"].long(), s["prefix_blocks"].long()
    starts = s["starts"].long()
    groups, m, p, sfx = starts.numel() - 1, s["most_members"], s["most_prefix"], s["most_suffix"]
    kc, vc = s["k_cache"].view(-1, kvh, d), s["v_cache"].view(-1, kvh, d)
    q = s["q"].float().view(ns, kvh, per, d) / math.sqrt(d)
    # the groups' members, padded to the largest group, and every sequence's place among them
    member = (starts[:-1, None] + torch.arange(m, device=dev)).clamp(max=ns - 1)
    group = torch.searchsorted(starts, torch.arange(ns, device=dev), right=True) - 1
    place = torch.arange(ns, device=dev) - starts[group]
    # shared part: [groups, kvh, m * per, p]
    at = torch.arange(p, device=dev)
    first = starts[:-1]
    slot = tables[first][:, (at // b).clamp(max=tables.shape[1] - 1)] * b + at % b
    live = at < (pb[first] * b)[:, None]
    slot = torch.where(live, slot, 0)
    kp, vp = kc[slot].float().permute(0, 2, 1, 3), vc[slot].float().permute(0, 2, 1, 3)
    qg = q[member].permute(0, 2, 1, 3, 4).reshape(groups, kvh, m * per, d)
    shared = (qg @ kp.transpose(-1, -2)).masked_fill(~live[:, None, None], -math.inf)
    # own part: [ns, kvh, per, sfx]
    at = (pb * b)[:, None] + torch.arange(sfx, device=dev)
    mine = at < lens[:, None]
    slot = torch.where(mine, torch.gather(tables, 1, (at // b).clamp(max=tables.shape[1] - 1)) * b + at % b, 0)
    ks, vs = kc[slot].float().permute(0, 2, 1, 3), vc[slot].float().permute(0, 2, 1, 3)
    alone = (q @ ks.transpose(-1, -2)).masked_fill(~mine[:, None, None], -math.inf)
    # one softmax over both parts
    back = lambda t: t.view(groups, kvh, m, per, -1)[group, :, place]  # noqa: E731  [ns, kvh, per, .]
    top = alone.amax(-1, keepdim=True)
    if p:
        top = torch.maximum(top, back(shared.amax(-1, keepdim=True)))
    e = torch.exp(alone - top)
    out, total = e @ vs, e.sum(-1, keepdim=True)
    if p:
        gtop = torch.full((groups, kvh, m, per, 1), math.inf, device=dev)
        gtop[group, :, place] = top
        e = torch.exp(shared - gtop.view(groups, kvh, m * per, 1))
        out, total = out + back(e @ vp), total + back(e.sum(-1, keepdim=True))
    return (out / total).view(ns, nh, d).to(s["q"].dtype)


def _plain_beam(s):
    """In 64 bits, so that continuations of different beams are ordered by their values and not by a rounding; a
    stable sort gives ties to the lowest beam and token."""
    batch, beams = s["scores"].shape
    x = s["logits"].double().view(batch, beams, -1)
    top = x.amax(-1, keepdim=True)
    x = x - top
    value = s["scores"].double()[..., None] + (x - torch.exp(x).sum(-1, keepdim=True).log())
    value, at = torch.sort(value.flatten(1), dim=1, descending=True, stable=True)
    value, at = value[:, :s["select"]], at[:, :s["select"]]
    vocab = x.shape[-1]
    return value.float(), (at // vocab).to(torch.int32), (at % vocab).to(torch.int32)


# ---------------------------------------------------------------------------------------------------- the library's
def _own_rope(s):
    kvb = _kvb()
    q, k, v = _split(s)
    more = {"q_norm": s.get("q_norm"), "k_norm": s.get("k_norm"), "eps": s["eps"], "interleaved": s["interleaved"]}
    if "slots" not in s:
        return kvb.qk_norm_rope(q, k, s["positions"], s["table"], **more)
    q_out = kvb.rope_append(q, k, v, s["positions"], s["table"], s["k_cache"], s["v_cache"], s["slots"], **more)
    return q_out, s["k_cache"], s["v_cache"]


def _own_prefix(s):
    kvb = _kvb()
    if "workspace" not in s:  # a decode loop keeps it
        need = kvb.shared_prefix_workspace_bytes(s["q"], s["k_cache"], s["tables"], s["starts"], s["heads"], s["kv_heads"])
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device=s["q"].device)
    return kvb.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["prefix_blocks"],
                                       s["starts"], s["heads"], s["kv_heads"], workspace=s["workspace"])


def _own_beam(s):
    return _kvb().beam_select(s["logits"], s["scores"], s["select"])


def run(state):
    if own:
        return {"rope": _own_rope, "prefix": _own_prefix, "beam": _own_beam}[state["op"]](state)
    return {"rope": _plain_rope, "prefix": _plain_prefix, "beam": _plain_beam}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "rope":
        elem = 4 if c["dtype"] == "fp32" else 2
        cols = (c["heads"] + (2 if c["cache"] else 1) * c["kv_heads"]) * c["dim"]
        rows = min(c["tokens"], c["start"] + c["tokens"])
        return {"bytes": 2 * c["tokens"] * cols * elem + rows * c["rot"] * 4 + 8 * c["tokens"],
                "flops": c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"] * (3 + (4 if c["norm"] else 0))}
    if c["op"] == "prefix":
        members, pblocks, suffix = _prefix_lens(c, 1234)
        ns, b = int(members.sum()), c["block"]
        held = int(pblocks.sum()) * b + int(suffix.sum())
        read = int((members * pblocks).sum()) * b + int(suffix.sum())
        return {"bytes": held * c["kv_heads"] * c["dim"] * 4 + 2 * ns * c["heads"] * c["dim"] * 2,
                "flops": 4 * read * c["heads"] * c["dim"]}
    n = c["batch"] * c["beams"] * c["vocab"]
    return {"bytes": n * (4 if c["dtype"] == "fp32" else 2), "flops": 4 * n}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_rope(c, s):
    """The rotation as a product of complex numbers."""
    n, half = c["tokens"], c["rot"] // 2
    cs = s["table"].double()[s["positions"].long()]
    turn = torch.complex(cs[:, :half], cs[:, half:])[:, None]
    flat, at, got = s["qkv"].double(), 0, []
    for heads, norm in ((c["heads"], s.get("q_norm")), (c["kv_heads"], s.get("k_norm"))):
        x = flat[:, at:at + heads * c["dim"]].reshape(n, heads, c["dim"]).clone()
        at += heads * c["dim"]
        if norm is not None:
            x = norm.double() * x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + s["eps"]).sqrt()
        if c["interleaved"]:
            z = torch.complex(x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]) * turn
            x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., :half], x[..., half:c["rot"]]) * turn
            x[..., :half], x[..., half:c["rot"]] = z.real, z.imag
        got.append(x)
    if not c["cache"]:
        return tuple(got)
    pools = []
    for rows, pool in ((got[1], s["k_cache"]), (flat[:, at:].reshape(n, c["kv_heads"], c["dim"]), s["v_cache"])):
        pool = pool.double().reshape(-1, c["kv_heads"], c["dim"])
        real = s["slots"] >= 0
        pool[s["slots"][real].long()] = rows[real]
        pools.append(pool.view(s["k_cache"].shape))
    return got[0], pools[0], pools[1]


def _exact_prefix(c, s):
    """Sequence by sequence, each over its whole context."""
    nh, kvh, d, b = c["heads"], c["kv_heads"], c["dim"], c["block"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    kc, vc = s["k_cache"].view(-1, kvh, d), s["v_cache"].view(-1, kvh, d)
    lens = s["lens"].tolist()
    for i in range(len(lens)):
        at = torch.arange(lens[i], device=DEV)
        slot = s["tables"][i].long()[at // b] * b + at % b
        k, v = kc[slot].double(), vc[slot].double()
        q = s["q"][i].double().view(kvh, nh // kvh, d)
        w = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) * d ** -0.5, -1)
        out[i] = torch.einsum("hgt,thd->hgd", w, v).reshape(nh, d)
    return out


def _exact_beam(c, s):
    """The best one taken out again and again."""
    x = torch.log_softmax(s["logits"].double(), -1).view(c["batch"], -1)
    x = x + s["scores"].double().repeat_interleave(c["vocab"], 1)
    place, gone = torch.arange(x.shape[1], device=DEV), torch.zeros_like(x, dtype=torch.bool)
    best, at = [], []
    for _ in range(c["select"]):
        left = torch.where(gone, -math.inf, x)
        top = left.amax(1, keepdim=True)
        first = torch.where((left == top) & ~gone, place, x.shape[1]).amin(1, keepdim=True)
        gone.scatter_(1, first, True)
        best.append(top)
        at.append(first)
    best, at = torch.cat(best, 1), torch.cat(at, 1)
    return best, at // c["vocab"], at % c["vocab"]


def exact(case, seed):
    return {"rope": _exact_rope, "prefix": _exact_prefix, "beam": _exact_beam}[case["op"]](case, prepare(case, seed))
