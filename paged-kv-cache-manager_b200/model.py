"""A decoder-only HF model (Qwen2 / Llama architecture) running with its KV cache in paged blocks on the GPU.

The device form of the reference's Python harness (python/paged_model.py:14-158 of
prathameshpranjale/paged-kv-cache-manager), with the same request API -- prefill / fork / decode /
decode_batch / free -- and the same block bookkeeping (this library's KVManager).  What moves from torch to
this library's kernels:
  * writing each new token's K/V into its slot  -> kvp_append_scatter for prompts (paged_model.py:54-55), fused
                                                   into kvp_paged_attention for decode steps (paged_model.py:145-146)
  * the copy-on-write copy after a fork          -> kvp_cow_copy         (paged_model.py:92-95, 113-117)
  * attention over the context                   -> kvp_paged_attention  (paged_model.py:56-63, 147-151)
Prefill attention uses the same decode kernel: prompt position p is a one-query sequence of length p + 1
over the request's block table, which is exactly causal attention.  Norms, projections, rotary embedding and
the MLP stay the model's own torch modules.

Two options, off unless asked for (the roundings differ from those of the paths above):
  * fused_rope     the rotary embedding (with RMS norms of the query and key heads, where the attention modules have
                   q_norm / k_norm) and the append in one pass                          -> kvp_rope_append
  * shared_prefix  decode_batch reads blocks that several requests share once for all   -> kvp_prefix_attention
                   (steps in which a long context of a request's own would hold up the rest go as without it)
beam_search runs on either: one decode_batch per step over forked requests, the selection on the GPU
(kvp_beam_select), the states of the surviving beams taken over without moving bytes (kvp_mgr_reorder).
"""
from __future__ import annotations

import importlib
from typing import List, Optional, Sequence

import torch

_kvb = importlib.import_module(__package__) if __package__ else None


def _lib():
    global _kvb
    if _kvb is None:
        _kvb = importlib.import_module("paged-kv-cache-manager_b200")
    return _kvb


def _sharing_pays(prefix, starts, lens, block: int, kv_heads: int, head_dim: int, sms: int) -> bool:
    """Whether a step's attention is worth running by groups.  The shared-prefix attention cuts the own tokens of every
    request alike, into 1 to 8 parts of a (request, kv head), and takes about 0.08 us per token of the longest part; the
    decode attention deals all contexts out evenly, but reads what is shared once per request.  So a step goes by groups
    unless the longest part's time exceeds that of the bytes saved by more than 20 us.  Measured (32 / 8 heads of 128,
    us by groups / by whole contexts): 256 requests over 2048 tokens with 100 own ones 72 / 262, 16 over 16384 with 8192
    197 / 221; 255 over 16 with 100 and one with 30000 1227 / 96, 4 over 16384 with 8192 190 / 98, 128 over 256 with 100
    and one with 4000 121 / 49.  Near the border either is up to a fifth slower than the other."""
    n, parts = len(lens), 1
    while parts < 8 and n * kv_heads * parts < 16 * sms:
        parts *= 2
    longest = max(int(x) - int(p) * block for x, p in zip(lens, prefix))
    saved = sum((int(b) - int(a) - 1) * int(prefix[a]) * block for a, b in zip(starts[:-1], starts[1:]))
    return 0.08 * longest / parts <= 20 + saved * kv_heads * head_dim * 4 / 6.5e6


class PagedEngine:
    """Paged-KV inference for one model on one GPU.  K/V pools are [layers][num_blocks][B][kv_heads][head_dim]
    in the model's dtype (fp16 or bf16)."""

    def __init__(self, model, num_blocks: int, block_size: int, *, fused_rope: bool = False,
                 shared_prefix: bool = False):
        from transformers.models.llama.modeling_llama import apply_rotary_pos_emb  # same for Qwen2 and Llama

        kvb = _lib()
        self._rope = apply_rotary_pos_emb
        self.m = model.eval()
        c = model.config
        self.L = c.num_hidden_layers
        self.nh = c.num_attention_heads
        self.kvh = c.num_key_value_heads
        self.hd = getattr(c, "head_dim", None) or c.hidden_size // c.num_attention_heads
        self.B = block_size
        self.num_blocks = num_blocks
        self.dev = next(model.parameters()).device
        self.dtype = next(model.parameters()).dtype
        if self.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("the paged cache holds fp16 or bf16 K/V: load the model in one of them")
        self.kv = kvb.KVManager(num_blocks, block_size)
        self.K = torch.zeros(self.L, num_blocks, block_size, self.kvh, self.hd, dtype=self.dtype, device=self.dev)
        self.V = torch.zeros_like(self.K)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.dev)
        self.prefill_tokens_computed = 0
        self.cow_data_copies = 0
        self.fused_rope, self.shared_prefix = fused_rope, shared_prefix
        self._table = None
        if fused_rope:
            rot = model.model.rotary_emb
            kind = getattr(rot, "rope_type", "default")
            if "dynamic" in kind or kind == "longrope":  # frequencies that change with the length
                raise ValueError(f"fused_rope needs fixed rotary frequencies; this model's are {kind}")
            if self.hd % 16 or self.hd > 256 or rot.inv_freq.numel() % 8:
                raise ValueError("fused_rope needs head_dim and the rotated part of it to be multiples of 16, at most "
                                 "256")

    # ------------------------------------------------------------------ internals
    def _rope_table(self, positions: int) -> torch.Tensor:
        """The rotation table, of at least `positions` rows."""
        if self._table is None or self._table.shape[0] < positions:
            rot = self.m.model.rotary_emb
            rows = max(256, 1 << (positions - 1).bit_length())
            self._table = _lib().rope_table(rows, 2 * rot.inv_freq.numel(), inv_freq=rot.inv_freq.float(),
                                            scaling=float(getattr(rot, "attention_scaling", 1.0)), device=self.dev)
        return self._table

    def _slots(self, table: Sequence[int], positions: Sequence[int]) -> torch.Tensor:
        B = self.B
        return torch.tensor([table[p // B] * B + p % B for p in positions], dtype=torch.int32, device=self.dev)

    @torch.no_grad()
    def _layers(self, h, positions: Sequence[int], slots: Optional[torch.Tensor], tables: torch.Tensor,
                lens: torch.Tensor, groups=None):
        """Runs every layer for n query tokens (h: [1, n, H]); token i is at positions[i], writes its K/V to
        slots[i] and attends over its context: tables[i] / lens[i].  With slots None (a decode step: every
        token is the newest of its own request) the attention kernel writes the K/V itself (fused append);
        otherwise (several prompt positions of one request read each other's slots, or the rotation appends) they are
        written first.  groups: (prefix_blocks, group_starts) of requests that share blocks, or None."""
        kvb = _lib()
        mdl = self.m.model
        n = h.shape[1]
        at = torch.tensor(positions, device=self.dev)
        if self.fused_rope:
            at, table = at.int(), self._rope_table(max(positions) + 1)
        else:
            cos, sin = mdl.rotary_emb(h, at[None])
        for li, layer in enumerate(mdl.layers):
            a = layer.self_attn
            x = layer.input_layernorm(h)
            q = a.q_proj(x).view(1, n, self.nh, self.hd)
            k = a.k_proj(x).view(1, n, self.kvh, self.hd)
            v = a.v_proj(x).view(1, n, self.kvh, self.hd)
            kn = vn = None
            if self.fused_rope:
                qn, kw = getattr(a, "q_norm", None), getattr(a, "k_norm", None)
                q = kvb.rope_append(q[0], k[0], v[0], at, table, self.K[li], self.V[li], slots, status=self.status,
                                    q_norm=None if qn is None else qn.weight, k_norm=None if kw is None else kw.weight,
                                    eps=getattr(qn or kw, "variance_epsilon", 1e-6))
            else:
                q, k = self._rope(q.transpose(1, 2), k.transpose(1, 2), cos, sin)
                kn, vn = k[0].transpose(0, 1).contiguous(), v[0].contiguous()
                if slots is not None:
                    kvb.append_scatter(kn[None], vn[None], self.K[li:li + 1], self.V[li:li + 1], slots,
                                       status=self.status)
                    kn = vn = None
                q = q[0].transpose(0, 1).contiguous()
            if groups is not None:
                o = kvb.shared_prefix_attention(q, self.K[li], self.V[li], tables, lens, *groups, self.nh, self.kvh,
                                                out_dtype=self.dtype, status=self.status)
            else:
                o = kvb.paged_attention(q, self.K[li], self.V[li], tables, lens, self.nh,
                                        self.kvh, out_dtype=self.dtype, status=self.status, num_blocks=self.num_blocks,
                                        k_new=kn, v_new=vn)
            h = h + a.o_proj(o.reshape(1, n, self.nh * self.hd))
            h = h + layer.mlp(layer.post_attention_layernorm(h))
        return mdl.norm(h)

    def _table_rows(self, rows: List[List[int]]) -> torch.Tensor:
        return self._dense(rows).to(self.dev)

    @staticmethod
    def _dense(rows: List[List[int]]) -> torch.Tensor:
        mb = max(1, max(len(r) for r in rows))
        t = torch.zeros((len(rows), mb), dtype=torch.int32)
        for i, r in enumerate(rows):
            if r:
                t[i, : len(r)] = torch.tensor(r, dtype=torch.int32)
        return t

    @torch.no_grad()
    def _forward(self, rid: int, tokens: Sequence[int], start: int, fused: bool = False):
        """Tokens placed at positions start .. start+n-1 of request rid (the manager already holds them)."""
        n = len(tokens)
        total = start + n
        table = self.kv.block_table(rid)
        assert self.kv.num_tokens(rid) >= total
        positions = list(range(start, total))
        ctx = table[: (total + self.B - 1) // self.B]
        tables = self._table_rows([ctx] * n)
        lens = torch.tensor([p + 1 for p in positions], dtype=torch.int32, device=self.dev)
        h = self.m.model.embed_tokens(torch.tensor(tokens, device=self.dev))[None]
        slots = None if fused and not self.fused_rope else self._slots(table, positions)
        h = self._layers(h, positions, slots, tables, lens)
        return self.m.lm_head(h[:, -1])[0]

    def _cow(self, pairs):
        if len(pairs):
            _lib().cow_copy(self.K, self.V, torch.as_tensor(pairs, dtype=torch.int32).reshape(-1, 2).to(self.dev),
                            status=self.status)
            self.cow_data_copies += len(pairs)

    # ------------------------------------------------------------------ request lifecycle
    def prefill(self, rid: int, seq: Sequence[int], parent: Optional[int] = None, shared_tokens: int = 0):
        """Admit rid with context seq; returns the logits of the next token, or None if out of blocks.  Shared
        full prefix blocks of `parent` are reused, not recomputed."""
        if parent is None:
            ok = self.kv.admit(rid, len(seq))
            start = 0
        else:
            start = min(shared_tokens, self.kv.num_tokens(parent), len(seq)) // self.B * self.B
            ok = self.kv.admit_with_prefix(rid, parent, shared_tokens, len(seq))
        if not ok:
            return None
        self.prefill_tokens_computed += len(seq) - start
        return self._forward(rid, list(seq[start:]), start)

    def fork(self, rid: int, parent: int):
        self.kv.fork(rid, parent)

    def decode(self, rid: int, last_token: int):
        """Appends last_token; returns the next-token logits, or None if no block is available."""
        before = self.kv.num_tokens(rid)
        done, _, pairs = self.kv.append_batch([rid])
        if done != 1:
            return None
        self._cow(pairs)  # before the new token is written into the copied block
        return self._forward(rid, [last_token], before, fused=True)

    @torch.no_grad()
    def decode_batch(self, rids: Sequence[int], last_tokens: Sequence[int]):
        """One decode step for several requests in one batched forward: logits [len(rids)][vocab]."""
        kvb = _lib()
        before = [self.kv.num_tokens(r) for r in rids]
        done, slots, pairs = self.kv.append_batch(list(rids))
        if done != len(rids):
            raise RuntimeError("out of blocks in decode_batch")
        self._cow(pairs)
        rows = [self.kv.block_table(r)[: (p + self.B) // self.B] for r, p in zip(rids, before)]
        tables, lens = self._dense(rows), torch.tensor([p + 1 for p in before], dtype=torch.int32)
        order, groups = None, None
        if self.shared_prefix and len(rows) > 1:
            by_table = sorted(range(len(rows)), key=lambda i: rows[i])  # requests that share blocks side by side
            prefix, starts = kvb.shared_prefix_groups(tables[by_table], lens[by_table], self.B)
            if prefix.any() and _sharing_pays(prefix, starts, lens[by_table].tolist(), self.B, self.kvh, self.hd,
                                               torch.cuda.get_device_properties(self.dev).multi_processor_count):
                order, groups = by_table, (torch.from_numpy(prefix).to(self.dev), torch.from_numpy(starts).to(self.dev))
                tables, lens = tables[order], lens[order]
                before, slots = [before[i] for i in order], [slots[i] for i in order]
                last_tokens = [last_tokens[i] for i in order]
        if not (self.fused_rope or groups):
            slots = None  # fused append
        else:
            slots = torch.tensor([int(x) for x in slots], dtype=torch.int32, device=self.dev)
        h = self.m.model.embed_tokens(torch.tensor(list(last_tokens), device=self.dev))[None]
        h = self._layers(h, before, slots, tables.to(self.dev), lens.to(self.dev), groups)[0]
        if order is not None:
            back = torch.empty(len(order), dtype=torch.long)
            back[order] = torch.arange(len(order))
            h = h[back.to(self.dev)]
        return self.m.lm_head(h)

    @torch.no_grad()
    def beam_search(self, rids: Sequence[int], prompt: Sequence[int], new_tokens: int, eos: Optional[int] = None):
        """Beam search with len(rids) beams for the continuation of `prompt` with the largest sum of log-probabilities,
        of new_tokens tokens or up to and with `eos`.  Returns up to len(rids) pairs (sum, tokens), best first, or None
        if the prompt finds no room.  `rids`: ids for the beams, freed at the end.  Running out of blocks on the way
        raises RuntimeError, as in decode_batch."""
        kvb, beams = _lib(), len(rids)
        select = beams if eos is None else 2 * beams  # at most one continuation of each beam ends
        if not 1 <= select <= 32 or beams >= self.m.config.vocab_size or new_tokens < 1:
            raise ValueError("beam_search takes 1 to 32 beams (16 with eos), fewer than the vocabulary, and "
                             "new_tokens >= 1")
        if len(set(rids)) != beams or any(self.kv.contains(r) for r in rids):
            raise ValueError("rids must be distinct and not in use")
        if len(prompt) < 1:
            raise ValueError("beam_search needs a prompt")
        logits = self.prefill(rids[0], prompt)
        if logits is None:
            return None
        held, ended = [rids[0]], []
        try:
            for r in rids[1:]:
                self.fork(r, rids[0])
                held.append(r)
            logits = logits[None].expand(beams, -1).contiguous()
            scores = torch.full((1, beams), -float("inf"), device=self.dev)
            scores[0, 0] = 0.0  # the beams are still alike: one of them counts
            tokens = [[] for _ in rids]
            for step in range(new_tokens):
                picked = kvb.beam_select(logits, scores, select, status=self.status)
                value, parent, token = (t[0].tolist() for t in picked)
                going = []  # (score, parent, token)
                for i, pick in enumerate(zip(value, parent, token)):
                    if pick[2] == eos and eos is not None:
                        if i < beams and pick[0] > -float("inf"):
                            ended.append((pick[0], tokens[pick[1]] + [eos]))
                    elif len(going) < beams:
                        going.append(pick)
                ended = sorted(ended, key=lambda e: -e[0])[:beams]
                tokens = [tokens[p] + [t] for _, p, t in going]
                last = step + 1 == new_tokens
                # log-probabilities only lower a score: what runs cannot overtake
                if last or (len(ended) == beams and going[0][0] <= ended[-1][0]):
                    break
                self.kv.reorder(rids, [p for _, p, _ in going])
                logits = self.decode_batch(rids, [t for _, _, t in going])
                scores = torch.tensor([[v for v, _, _ in going]], dtype=torch.float32, device=self.dev)
            if last:
                ended += [(v, t) for (v, _, _), t in zip(going, tokens) if v > -float("inf")]
            return sorted(ended, key=lambda e: -e[0])[:beams]
        finally:
            for r in held:
                self.free(r)

    def free(self, rid: int):
        self.kv.free(rid)

    def kv_bytes_per_token(self) -> int:
        return 2 * self.L * self.kvh * self.hd * self.K.element_size()
