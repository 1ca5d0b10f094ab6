"""Several sampled answers to one prompt, ranked by log probability.

The prompt is prefilled once; its cache pages are then shared by every answer
(``ops.fork_pages``), and each answer writes to pages of its own: ``ops.reserve_pages``
gives a row the page of its next token and replaces a shared, partly filled last page by
a private copy. Decode steps replay one CUDA graph (``DecodeGraph``) that also scores the
sampled tokens (``ops.token_logprobs``). At the end the answers that lost give their pages
back (``ops.free_pages``) and the kept ones' pages move to the front of the cache
(``ops.compact_pages``), where ``table`` / ``lens`` let a caller go on from them.

Everything between the prefill and the ranking stays on the device; with stop tokens the
host reads two numbers per step.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import ops
from ..models.mla_moe import DecodeGraph, ForwardBatch, KVCache, MLAMoEModel


@dataclass
class Answer:
    token_ids: list
    logprobs: list        # of each token, before temperature
    entropies: list
    top_logprobs: list    # per token [(id, log probability)], most probable first

    @property
    def mean_logprob(self) -> float:
        return sum(self.logprobs) / max(1, len(self.logprobs))


class ParallelAnswers:
    """Owns the pages of ``cache`` (nothing else may use it meanwhile). ``max_tokens_per_row``
    bounds prompt and answer together."""

    def __init__(self, model: MLAMoEModel, cache: KVCache, answers: int, max_tokens_per_row: int, top_logprobs: int = 0,
                 use_graph: bool = True):
        if not 1 <= answers <= ops.kernels().PAGES_MAX_ROWS or max_tokens_per_row < 1:
            raise ValueError("ParallelAnswers: 1 to 1,024 answers, and room for their tokens")
        if max_tokens_per_row > model.cos_sin.shape[0]:
            raise ValueError(f"ParallelAnswers: the model's positions end at {model.cos_sin.shape[0]}")
        if getattr(model, "ep", None) is not None:
            raise ValueError("ParallelAnswers: one rank only")
        most = min(ops.kernels().LOGPROBS_MAX_TOP, model.cfg.vocab_size)
        if not 0 <= top_logprobs <= most:
            raise ValueError(f"ParallelAnswers: 0 to {most} alternatives")
        self.model, self.cache, self.n = model, cache, answers
        self.cols = -(-max_tokens_per_row // cache.block_size)
        self.max_tokens = max_tokens_per_row
        i32 = dict(dtype=torch.int32, device=model.device)
        self.refs = torch.zeros(cache.num_blocks, **i32)
        self.table = torch.full((0, self.cols), -1, **i32)
        self.lens = torch.zeros(0, **i32)
        self.graph = DecodeGraph(model, cache, answers, self.cols, self.cols * cache.block_size, use_graph=use_graph,
                                 logprobs=top_logprobs)
        self._i32 = i32

    def _reserve(self, tokens):
        return ops.reserve_pages(self.table, self.lens, self.refs, self.cache.data, tokens,
                                 block_size=self.cache.block_size, cache_scales=self.cache.scales, strict=True)

    def _prefill(self, prompt) -> torch.Tensor:
        """Caches the prompt in row 0; returns the logits of its last token [1, V]."""
        P, c = len(prompt), self.cache
        self.refs.zero_()
        self.table = torch.full((1, self.cols), -1, **self._i32)
        self.lens = torch.zeros(1, **self._i32)
        if int(self._reserve(torch.tensor([P], **self._i32)).sum()):
            raise MemoryError("ParallelAnswers: the cache has too few pages for the prompt")
        self.lens.fill_(P)
        cu = torch.tensor([0, P], **self._i32)
        fb = ForwardBatch(mode="prefill", token_ids=torch.tensor([int(t) for t in prompt], **self._i32),
                          positions=torch.arange(P, **self._i32),
                          slot_mapping=ops.paged_slots(self.table, self.lens, P, block_size=c.block_size).view(-1),
                          cu_q=cu, cu_k=cu, max_q=P, logits_idx=cu[1:] - 1)
        return self.model.forward(fb, c)

    def generate(self, prompt, max_new_tokens: int, temperature: float = 1.0, seed: int = 0, keep: int = 1,
                 stop_token_ids: tuple = ()) -> list[Answer]:
        """The ``keep`` answers of the highest mean log probability, best first. Equal seeds
        give equal answers; answer i draws with noise key seed * answers + i. Too few pages for
        the answers are a MemoryError: before the first step, or with stop tokens, which may end
        answers sooner, within two steps of running out."""
        n, g, c = self.n, self.graph, self.cache
        if not 1 <= keep <= n:
            raise ValueError("ParallelAnswers: keep between 1 and the number of answers")
        if not prompt or max_new_tokens < 1 or len(prompt) + max_new_tokens > self.max_tokens:
            raise ValueError("ParallelAnswers: prompt and answer must fit max_tokens_per_row")
        if not all(0 <= int(t) < self.model.cfg.vocab_size for t in prompt):
            raise ValueError("ParallelAnswers: token ids outside the vocabulary")
        logits = self._prefill(prompt)
        P, bs = len(prompt), c.block_size
        # the prompt's whole pages once, the rest per answer; the last token is not cached
        pages = P // bs + n * (-(-(P + max_new_tokens - 1) // bs) - P // bs) if max_new_tokens > 1 else 0
        if pages > c.num_blocks and not stop_token_ids:
            raise MemoryError(f"ParallelAnswers: the cache ran out of pages: {pages} are needed, it has {c.num_blocks}")
        self.table, self.lens = ops.fork_pages(self.table, self.lens, torch.zeros(n, **self._i32), self.refs,
                                               block_size=c.block_size)
        temps = torch.full((n,), float(temperature), dtype=torch.float32, device=self.model.device)
        keys = torch.arange(n, dtype=torch.int64, device=self.model.device) + seed * n
        g.temps.copy_(temps)
        rows = logits.expand(n, logits.shape[1])
        # the noise of position t comes from key * (longest row) + t
        tokens = ops.sample_tokens(rows, row_temp=temps, row_key=keys * self.max_tokens)
        stops = torch.tensor(list(stop_token_ids), **self._i32) if stop_token_ids else None
        steps = [(tokens, ops.token_logprobs(rows, tokens, top_k=g.logprobs))]
        live = torch.ones(n, dtype=torch.bool, device=self.model.device)
        ended = [live]
        short = torch.zeros((), dtype=torch.int64, device=self.model.device)
        one = torch.ones(n, **self._i32)
        for t in range(1, max_new_tokens):
            if stops is not None:
                live = live & ~(tokens[:, None] == stops).any(1)
                any_live, lacking = torch.stack([live.sum(), short]).tolist()  # the step's one read
                if lacking:
                    raise MemoryError("ParallelAnswers: the cache ran out of pages")
                if not any_live:
                    break
            ended.append(live)
            short = short + self._reserve(live.int()).sum()
            slots = ops.paged_slots(self.table, one, 1, positions=self.lens[:, None].contiguous(),
                                    block_size=c.block_size).view(-1)
            g.ids.copy_(tokens)
            g.pos.copy_(self.lens)
            g.slots.copy_(torch.where(live, slots, -1))
            g.block_table.copy_(self.table.clamp(min=0))
            g.ctx.copy_(torch.where(live, self.lens + 1, 0))
            g.keys.copy_(keys * self.max_tokens + t)
            tokens = g.run().clone()
            steps.append((tokens, ops.TokenLogprobs(*(s.clone() for s in g.scores))))
            self.lens += live.int()
        if int(short):
            raise MemoryError("ParallelAnswers: the cache ran out of pages")
        ids = torch.stack([s[0] for s in steps]).tolist()
        lp, ent, top_lp, top_ids = (torch.stack([s[1][k] for s in steps]).tolist() for k in range(4))
        made = torch.stack(ended).sum(0).tolist()
        answers = [Answer([ids[t][i] for t in range(made[i])], [lp[t][i] for t in range(made[i])],
                          [ent[t][i] for t in range(made[i])],
                          [list(zip(top_ids[t][i], top_lp[t][i])) for t in range(made[i])]) for i in range(n)]
        order = sorted(range(n), key=lambda i: (-answers[i].mean_logprob, i))
        ops.free_pages(self.table, self.refs, torch.tensor(order[keep:], **self._i32))
        ops.compact_pages(self.table, self.refs, c.data, block_size=c.block_size, cache_scales=c.scales)
        best = torch.tensor(order[:keep], dtype=torch.int64, device=self.model.device)
        self.table, self.lens = self.table[best].contiguous(), self.lens[best].contiguous()
        return [answers[i] for i in order[:keep]]

    def release(self):
        self.graph.release()
