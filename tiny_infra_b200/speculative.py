"""Decoding several tokens a step: verify a tree of drafted tokens per sequence in one forward.

``TreeDecoder.step`` takes a tree per slot -- node 0 the sequence's last token, every other node a guess
for the token behind its parent, from whatever drafts the caller has -- runs the model over all nodes,
draws a token at each from the model's own distribution, and keeps the path that the draws confirm.  What
it emits is distributed as one token at a time drawn by ``sampler.sample`` with the slot's own parameters
would be (the batcher's rules for a whole batch's top-k and top-p, ``sampler.SamplingParams``, are not
applied); a step emits one token more than the guesses that held.

Per step: the host assigns blocks (``KVCacheManager.plan_tokens``, the reference's order),
``paging.reserve`` makes slots, positions and masks from the lengths on the device, the layers run with
``tree.attention``, ``sampler.sample`` draws at every node, ``tree.accept`` moves the kept nodes' K and V
behind the cached tokens and advances ``seq_len``.  Blocks behind what was kept stay assigned and serve
the next step.  A step copies its small inputs to the device and waits for its tokens at the end.
"""
from __future__ import annotations

import numpy as np
import torch

from . import paging, sampler, tree
from .qwen2 import PackedBatch, Qwen2ForCausalLM


class TreeDecoder:
    def __init__(self, model: Qwen2ForCausalLM, kv_cache) -> None:
        if kv_cache.kv_bits != 16:
            raise RuntimeError("drafted trees need the 16-bit KV pool")
        self.model, self.kv = model, kv_cache
        self.cos, self.sin = model.rope_tables(kv_cache.max_positions)
        # the host hands out the blocks; the device's calls find every entry assigned
        self.no_blocks = paging.free_list([], capacity=1, device=model.device)

    def _check(self, slots, trees) -> tuple[list[int], np.ndarray, np.ndarray]:
        """Node counts, packed tokens and parents of ``trees``."""
        if len(slots) != len(trees) or len(set(int(s) for s in slots)) != len(slots):
            raise ValueError("step needs one tree per slot, and distinct slots")
        if any(not 0 <= int(s) < self.kv.max_batch_size for s in slots):
            # (a negative one would count from the end on the host, and index the lengths on the device)
            raise ValueError(f"step needs slots from 0 to {self.kv.max_batch_size - 1}")
        counts, tokens, parents = [], [], []
        for toks, par in trees:
            n = len(toks)
            if n < 1 or len(par) != n or int(par[0]) >= 0:
                raise ValueError("a tree needs a token and a parent per node, and node 0 is its root")
            if any(not 0 <= int(p) < j for j, p in enumerate(par) if j > 0):
                raise ValueError("a node's parent is an earlier node")
            counts.append(n)
            tokens.extend(int(t) for t in toks)
            parents.extend(int(p) for p in par)
        return counts, np.asarray(tokens, np.int32), np.asarray(parents, np.int32)

    def batch(self, slots, counts, ids: torch.Tensor, parents: torch.Tensor) -> PackedBatch:
        """The packed batch of these trees (tokens and parents on the device), blocks assigned."""
        kv, dev = self.kv, self.model.device
        kv.plan_tokens(slots, counts)
        T, B = int(sum(counts)), len(slots)
        host = torch.tensor([list(map(int, slots)), counts], dtype=torch.int32)
        rows, n = host.to(dev)
        i32 = dict(dtype=torch.int32, device=dev)
        cu, positions = torch.empty(B + 1, **i32), torch.empty(T, **i32)
        mapping = torch.empty(T, dtype=torch.int64, device=dev)
        masks = torch.empty(T, -(-max(counts) // 32), **i32)
        paging.reserve(kv.block_tables, kv.seq_len, n, self.no_blocks, mapping, positions, cu,
                       block_size=kv.block_size, row_index=rows, parents=parents, masks=masks)
        start = kv.seq_len.index_select(0, rows)
        return PackedBatch(
            input_ids=ids, positions=positions, slot_mapping=mapping, seq_slots=rows, start_pos=start,
            cu_seqlens=cu, ctx_lens=start + n, tile_seq=None, tile_q0=None, num_tokens=T, num_seqs=B,
            decode=False, last_rows=None, tree_masks=masks)

    def step(self, slots, trees, *, temperatures=None, top_ks=None, top_ps=None, min_ps=None,
             uniforms=None) -> list[list[int]]:
        """New tokens of each slot, at least one.

        ``trees[i]``: (tokens, parents) of slot ``slots[i]``.  ``temperatures``, ``top_ks``, ``top_ps``,
        ``min_ps``: one value per slot (``sampler.sample``; default: greedy); ``uniforms``: one number
        per node, packed (needed once a temperature is above 0)."""
        if len(slots) == 0:
            return []
        counts, tokens, parents = self._check(slots, trees)
        T, B, dev = len(tokens), len(slots), self.model.device
        hot = temperatures is not None and any(float(t) > 0 for t in temperatures)
        if hot and (uniforms is None or len(uniforms) != T):
            raise ValueError("drawing needs a uniform number per node")
        for name, v in (("temperatures", temperatures), ("top_ks", top_ks), ("top_ps", top_ps),
                        ("min_ps", min_ps)):
            if v is not None and len(v) != B:
                raise ValueError(f"{name} needs one value per slot")
        ids, up = torch.from_numpy(np.stack([tokens, parents])).to(dev)
        pb = self.batch(slots, counts, ids, up)
        logits = self.model.forward_packed(pb, self.kv, self.cos, self.sin, rows="all")
        per = lambda v, d: torch.from_numpy(np.repeat(np.asarray(v, d), counts)).to(dev)     # noqa: E731
        t = per(temperatures if hot else np.zeros(B), np.float32)
        u = torch.from_numpy(np.asarray(uniforms, np.float32)).to(dev) if hot else torch.zeros_like(t)
        targets = sampler.sample(
            logits, t, u, top_ks=None if top_ks is None else per(top_ks, np.int32),
            top_ps=None if top_ps is None else per(top_ps, np.float32),
            min_ps=None if min_ps is None else per(min_ps, np.float32))
        deep = min(max(counts), 1024)
        num, path, new = (torch.empty(s, dtype=torch.int32, device=dev)
                          for s in ((B,), (B, deep), (B, deep)))
        tree.accept(self.kv.key_cache, self.kv.value_cache, ids, up, targets, pb.cu_seqlens,
                    pb.slot_mapping, num, path, new, seq_lens=self.kv.seq_len, row_index=pb.seq_slots)
        host = torch.cat([num.unsqueeze(1), new], 1).cpu().numpy()      # waits for the step
        self.kv.advance(slots, host[:, 0])
        return [[int(x) for x in row[1:1 + row[0]]] for row in host]
