"""Generation and scoring of ragged batches: prompts of different lengths, packed
without padding, over a KV cache held in pages.

The reference pads every batch to one length and keeps one contiguous cache
(src/model/disaggregated.py:537-701); this is an addition for callers whose
requests differ in length. It runs both roles in one process (the workers of a
co-located ``DisaggregatedQwenModel``, or workers built on their own):

* ``PagedKVCache``   the page pool, and which sequence holds which pages
* ``RaggedGenerator.generate``   prompts -> tokens with their log-probabilities:
  packed prefill (whole prompts or chunks) and one-token steps over the pages
* ``RaggedGenerator.score``      log-probabilities of given token sequences,
  without a cache

A layer is ``sum_rmsnorm``, the qkv ``linear``, ``qk_norm_rope_paged``, the paged
attention, the o_proj ``linear`` and the FFN worker's block, on [tokens, hidden].
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import torch

from .. import ops
from ..config import ModelConfig
from ..ops.checks import AFDBoundsError
from ..utils.sampling import sample_next_token
from .attention import AttentionWorker
from .ffn import FFNWorker


class PagedKVCache:
    """K and V pages [layers, pages, n_kv, page_size, D] and their owners. A
    sequence's positions fill its pages in order; any free page will do."""

    def __init__(self, cfg: ModelConfig, num_pages: int, page_size: int, device,
                 dtype=torch.bfloat16):
        if num_pages < 1:
            raise ValueError(f"num_pages {num_pages} must be positive")
        if page_size < 16 or page_size % 16 or page_size > 4096:
            raise ValueError(f"page_size {page_size} must be a multiple of 16, at most 4096")
        self.page_size = page_size
        self.num_pages = num_pages
        shape = (cfg.num_hidden_layers, num_pages, cfg.num_key_value_heads, page_size,
                 cfg.head_dim)
        self.k = torch.empty(shape, device=device, dtype=dtype)
        self.v = torch.empty(shape, device=device, dtype=dtype)
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: Dict[int, List[int]] = {}
        self._next = 0

    def layer(self, l: int):
        return self.k[l], self.v[l]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def allocate(self, positions: int) -> int:
        """Pages for `positions` of a new sequence; returns its handle."""
        need = -(-positions // self.page_size)
        if need > len(self._free):
            raise ValueError(f"the page pool is full: {positions} positions need {need} pages, "
                             f"{len(self._free)} of {self.num_pages} are free")
        seq = self._next
        self._next += 1
        self._pages[seq] = [self._free.pop() for _ in range(need)]
        return seq

    def release(self, seq: int) -> None:
        self._free.extend(reversed(self._pages.pop(seq)))

    def table(self, seqs: Sequence[int]) -> torch.Tensor:
        """int32 [len(seqs), most pages of them]; unused entries are 0."""
        width = max([len(self._pages[s]) for s in seqs] + [1])
        t = torch.zeros(len(seqs), width, dtype=torch.int32)
        for i, s in enumerate(seqs):
            p = self._pages[s]
            t[i, : len(p)] = torch.tensor(p, dtype=torch.int32)
        return t.to(self.k.device)

    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()


@dataclass
class RaggedOutput:
    """One sequence of ``RaggedGenerator.generate``: the new tokens (int64 [n])
    and, per token, its log-probability and the entropy it was drawn from (fp32
    [n]) and the most likely tokens with theirs ([n, top_logprobs])."""
    tokens: torch.Tensor
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def slots_of(table: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor,
             page_size: int) -> torch.Tensor:
    """Page rows (page * page_size + row, int64) of `positions` of the table rows
    `rows`."""
    p = positions.long()
    return table[rows, p // page_size].long() * page_size + p % page_size


class RaggedGenerator:
    """Serves batches of prompts of different lengths on the workers of one
    process. `num_pages` * `page_size` positions are held at once. Every call reads
    once, at its end, what its kernels recorded: AFDBoundsError for an index out of
    range, RuntimeError for a wait inside a kernel that ran out."""

    def __init__(self, attention: AttentionWorker, ffn: FFNWorker, num_pages: int,
                 page_size: int = 64):
        self.aw = attention
        self.fw = ffn
        self.cfg = attention.cfg
        self.device = attention.device
        self.max_positions = attention.rope.shape[0]
        self.cache = PagedKVCache(attention.cfg, num_pages, page_size, attention.device,
                                  attention.dtype)
        cuda = attention.device.type == "cuda"
        self.status = torch.zeros(2, dtype=torch.int32, device=self.device) if cuda else None

    # ------------------------------------------------------------- helpers
    def _check_prompts(self, prompts: Sequence[Sequence[int]], new: int) -> List[torch.Tensor]:
        """The prompts as tensors; `new` positions follow each."""
        if len(prompts) == 0:
            raise ValueError("no prompts")
        got = []
        for i, p in enumerate(prompts):
            t = torch.as_tensor(p, dtype=torch.long).reshape(-1).cpu()
            if t.numel() == 0:
                raise ValueError(f"prompt {i} is empty")
            if t.numel() + new > self.max_positions:
                raise ValueError(f"prompt {i}: {t.numel()} tokens and {new} positions after them "
                                 f"exceed the {self.max_positions} positions of the workers")
            if int(t.min()) < 0 or int(t.max()) >= self.cfg.vocab_size:
                raise ValueError(f"prompt {i} has a token outside [0, {self.cfg.vocab_size})")
            got.append(t)
        return got

    def _check_status(self) -> None:
        """Raises what the kernels since the last check recorded (waits for them)."""
        if self.status is None:
            return
        code, site = self.status.tolist()
        if code != 0:
            self.status.zero_()
            error = AFDBoundsError if code == 3 else RuntimeError
            raise error(f"a kernel recorded a failure: code={code} site={site}")

    def _forward(self, ids: torch.Tensor, attend) -> torch.Tensor:
        """Every layer on the packed tokens `ids` [T]; attend(layer, qkv, lw) ->
        [T, nq * D]. Returns the hidden states [T, H]."""
        aw, fw = self.aw, self.fw
        x = aw.embed(ids)
        for l in range(self.cfg.num_hidden_layers):
            lw = aw.w.layers[l]
            xn = ops.rmsnorm(x, lw.in_norm, self.cfg.rms_norm_eps)
            o = attend(l, ops.linear(xn, lw.w_qkv), lw)
            x = fw.forward_ffn_layer(l, ops.linear(o, lw.w_o, residual=x))
        return x

    def _store(self, l, qkv, lw, positions, slots) -> torch.Tensor:
        cfg = self.cfg
        kp, vp = self.cache.layer(l)
        return ops.qk_norm_rope_paged(qkv, lw.q_norm, lw.k_norm, self.aw.rope, kp, vp, positions,
                                      slots, cfg.num_attention_heads, cfg.num_key_value_heads,
                                      cfg.rms_norm_eps, status=self.status)

    def _prefill(self, prompts: List[torch.Tensor], table: torch.Tensor,
                 chunk: Optional[int]) -> torch.Tensor:
        """Fills the pages; returns the hidden states of each prompt's last
        token. With `chunk`, at most that many tokens of each prompt at a time."""
        dev, page = self.device, self.cache.page_size
        lens = [p.numel() for p in prompts]
        last = [None] * len(prompts)
        start = 0
        while start < max(lens):
            live = [i for i, n in enumerate(lens) if n > start]
            ends = [min(lens[i], start + chunk) if chunk else lens[i] for i in live]
            news = [e - start for e in ends]
            ids = torch.cat([prompts[i][start:e] for i, e in zip(live, ends)]).to(dev)
            pos = torch.cat([torch.arange(start, e, dtype=torch.int32) for e in ends]).to(dev)
            row = torch.repeat_interleave(torch.tensor(live), torch.tensor(news)).to(dev)
            cu = torch.tensor([0] + news).cumsum(0).to(torch.int32).to(dev)
            total = torch.tensor(ends, dtype=torch.int32).to(dev)
            tab = table[torch.tensor(live, device=dev)]
            slots = slots_of(table, row, pos, page)

            def attend(l, qkv, lw):
                q = self._store(l, qkv, lw, pos, slots)
                kp, vp = self.cache.layer(l)
                return ops.paged_prefill_attention(q, kp, vp, tab, total, cu, status=self.status)

            x = self._forward(ids, attend)
            for j, i in enumerate(live):
                if ends[j] == lens[i]:
                    last[i] = x[sum(news[: j + 1]) - 1]
            start += chunk if chunk else max(lens)
        return torch.stack(last)

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return self.aw.lm_head_block([x], 1, last_only=False)

    # ------------------------------------------------------------ requests
    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int,
                 top_logprobs: int = 0, temperature: float = 1.0, top_k: int = 50,
                 top_p: float = 0.9, do_sample: bool = False,
                 prefill_chunk_size: Optional[int] = None, eos_token_id: Optional[int] = None,
                 generator: Optional[torch.Generator] = None) -> List[RaggedOutput]:
        """`max_new_tokens` tokens for each prompt (fewer where `eos_token_id` comes
        first), with the log-probabilities under the unmodified logits. The pages
        are released at the end, also after an error."""
        if max_new_tokens < 1:
            raise ValueError(f"max_new_tokens {max_new_tokens} must be positive")
        if prefill_chunk_size is not None and prefill_chunk_size < 1:
            raise ValueError(f"prefill_chunk_size {prefill_chunk_size} must be positive")
        ids = self._check_prompts(prompts, max_new_tokens - 1)  # the last has no position
        B, dev, page = len(ids), self.device, self.cache.page_size
        seqs: List[int] = []
        try:
            for p in ids:  # the last new token is never stored
                seqs.append(self.cache.allocate(p.numel() + max_new_tokens - 1))
            table = self.cache.table(seqs)
            logits = self._logits(self._prefill(ids, table, prefill_chunk_size))
            pos = torch.tensor([p.numel() for p in ids], dtype=torch.int32).to(dev)
            rows = torch.arange(B, device=dev)
            done = torch.zeros(B, dtype=torch.bool, device=dev)
            steps = []
            for step in range(max_new_tokens):
                tok = sample_next_token(logits, temperature, top_k, top_p, do_sample,
                                        generator).view(-1)
                steps.append((tok, ops.token_logprobs(logits, tok, top_logprobs)))
                if eos_token_id is not None:
                    done |= tok == eos_token_id
                    if bool(done.all()):
                        break
                if step == max_new_tokens - 1:
                    break
                slots, lens = slots_of(table, rows, pos, page), pos + 1

                def attend(l, qkv, lw):
                    q = self._store(l, qkv, lw, pos, slots)
                    kp, vp = self.cache.layer(l)
                    return ops.paged_decode_attention(q, kp, vp, table, lens, status=self.status)

                logits = self._logits(self._forward(tok, attend))
                pos = lens
            self._check_status()
        finally:
            for s in seqs:
                self.cache.release(s)
        cat = lambda f: torch.stack([f(t, r) for t, r in steps], 1)  # noqa: E731
        tok, lp = cat(lambda t, r: t), cat(lambda t, r: r.logprob)
        ent, ti = cat(lambda t, r: r.entropy), cat(lambda t, r: r.top_ids)
        tl = cat(lambda t, r: r.top_logprobs)
        out = []
        for b in range(B):
            n = tok.shape[1]
            if eos_token_id is not None:
                hit = (tok[b] == eos_token_id).nonzero()
                n = int(hit[0]) + 1 if len(hit) else n
            out.append(RaggedOutput(tok[b, :n], lp[b, :n], ent[b, :n], ti[b, :n], tl[b, :n]))
        return out

    @torch.no_grad()
    def score(self, sequences: Sequence[Sequence[int]], top_logprobs: int = 0,
              rows_at_once: int = 2048) -> List[ops.TokenLogprobs]:
        """Log-probability of each token of each sequence given the ones before it
        (from the second token on), the entropies, and the most likely tokens. The
        LM head runs on `rows_at_once` positions at a time."""
        if rows_at_once < 1:
            raise ValueError(f"rows_at_once {rows_at_once} must be positive")
        ids = self._check_prompts(sequences, 0)
        cfg, dev = self.cfg, self.device
        lens = [p.numel() for p in ids]
        cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
        pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(dev)
        flat = torch.cat(ids).to(dev)

        def attend(l, qkv, lw):
            q, k, v = ops.qk_norm_rope_packed(qkv, lw.q_norm, lw.k_norm, self.aw.rope, pos,
                                              cfg.num_attention_heads, cfg.num_key_value_heads,
                                              cfg.rms_norm_eps, status=self.status)
            return ops.packed_attention(q, k, v, cu, status=self.status)

        x = self._forward(flat, attend)
        after = torch.cat([torch.cat([p[1:], p[:1] * 0]) for p in ids]).to(dev)
        parts = [ops.token_logprobs(self._logits(x[a:a + rows_at_once]),
                                    after[a:a + rows_at_once], top_logprobs)
                 for a in range(0, x.shape[0], rows_at_once)]
        self._check_status()
        whole = [torch.cat([p[f] for p in parts]) for f in range(4)]
        out, a = [], 0
        for n in lens:  # a sequence's last row has no token after it
            out.append(ops.TokenLogprobs(*[w[a:a + n - 1] for w in whole]))
            a += n
        return out
