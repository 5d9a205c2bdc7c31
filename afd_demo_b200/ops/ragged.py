"""Operators of ragged batches: sequences of different lengths, packed one after
another without padding, over a KV cache held in pages, and the
log-probabilities of what was sampled or given.

Page pool: ``k_pages``, ``v_pages`` [pages, n_kv, page_size, D]; position p of
sequence b lies in page ``page_table[b, p // page_size]`` at row
``p % page_size``. Any page order; ``page_size`` a multiple of 16. A pool may be
a slice of a larger buffer as long as each page is contiguous.

On CUDA tensors these run the sm_100a kernels (bf16 or fp16, D 64 or 128) on the
current stream, without a host synchronisation, so they can be captured in CUDA
graphs; the lengths, tables and offsets are read on the device at each replay.
On CPU tensors they run the PyTorch statements of ``torch_ref``. Wrong types,
shapes or devices raise ValueError. Index data is checked on the device: an
entry out of range is never dereferenced and is recorded in the optional
``status`` word pair (int32 [2], code 3), as the other kernels do. Offsets of rows
are clamped to the rows there are; query offsets that decrease give zeros throughout.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import torch_ref


_mod = None


def _ext():
    """The extension, looked up once: these calls are short enough to notice."""
    global _mod
    if _mod is None:
        from . import ext
        _mod = ext()
    return _mod


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns, per row of logits."""
    logprob: torch.Tensor        # fp32 [R]: of the given token
    entropy: torch.Tensor        # fp32 [R], in nats
    top_ids: torch.Tensor        # int64 [R, top_k]: larger logits first, equal ones by index
    top_logprobs: torch.Tensor   # fp32 [R, top_k]


def qk_norm_rope_paged(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
                       rope: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                       positions: torch.Tensor, slots: torch.Tensor, nq: int, nkv: int,
                       eps: float, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-head RMSNorm of q and k and RoPE at ``positions`` (int32 [T]) for the
    packed projections ``qkv`` [T, (nq + 2 nkv) D]; k and v are stored at the
    page rows ``slots`` (int64 [T], page * page_size + row; a negative slot
    stores nothing). Slots are distinct. Returns q [T, nq, D]. All in fp32 with
    one rounding, where ``qk_norm_rope_cache`` rounds at each step as HF does."""
    if not qkv.is_cuda:
        return torch_ref.qk_norm_rope_paged(qkv, q_norm, k_norm, rope, k_pages, v_pages,
                                            positions, slots, nq, nkv, eps)
    return _ext().norm_rope(qkv, q_norm, k_norm, rope, positions, nq, nkv, eps, k_pages, v_pages,
                            slots, status)[0]


def qk_norm_rope_packed(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
                        rope: torch.Tensor, positions: torch.Tensor, nq: int, nkv: int,
                        eps: float, status: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """As ``qk_norm_rope_paged`` without a cache: (q [T, nq, D], k [T, nkv, D],
    v), v being the view of ``qkv``."""
    T, D = qkv.shape[0], q_norm.shape[0]
    if not qkv.is_cuda:
        q, k = torch_ref.qk_norm_rope(qkv, q_norm, k_norm, rope, positions, nq, nkv, eps)
    else:
        q, k = _ext().norm_rope(qkv, q_norm, k_norm, rope, positions, nq, nkv, eps, None, None,
                                None, status)
    return q, k, qkv[:, (nq + nkv) * D:].view(T, nkv, D)


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           page_table: torch.Tensor, seq_lens: torch.Tensor,
                           scale: Optional[float] = None,
                           status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GQA attention of one new token per sequence: q [B, nq, D] over positions
    0 .. seq_lens[b] - 1 of the paged cache (page_table int32 [B, max_pages],
    seq_lens int32 [B], the new token included). Returns [B, nq * D]; a sequence
    of length 0 gives zeros. `scale` defaults to 1 / sqrt(D)."""
    if not q.is_cuda:
        return torch_ref.paged_decode_attention(q, k_pages, v_pages, page_table, seq_lens, scale)
    return _ext().paged_decode_attention(q, k_pages, v_pages, page_table, seq_lens, scale, status)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal GQA attention of packed sequences: q [T, nq, D], k and v
    [Tk, n_kv, D] (any row stride, e.g. views of one projection), sequence i in
    rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1 (int32 [n + 1], rising). With
    `cu_seqlens_k` the keys have rows of their own and the queries are the last
    positions of their sequence; a query before the first key gives zeros, and so
    do rows before cu_seqlens[0] and past cu_seqlens[n]. Returns [T, nq * D].

    The softmax weights are rounded to q's type for their product with v. A NaN or an
    infinity in v reaches, besides the queries that see it, earlier ones that share a
    tile with it, up to 63 + 256 nkv / nq positions before it (on CPU any of its
    sequence): it meets their weights of zero. One in k does not."""
    if not q.is_cuda:
        return torch_ref.packed_attention(q, k, v, cu_seqlens, cu_seqlens_k, scale)
    return _ext().packed_attention(q, k, v, cu_seqlens, cu_seqlens_k, scale, status)


def paged_prefill_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                            page_table: torch.Tensor, seq_lens: torch.Tensor,
                            cu_seqlens: torch.Tensor, scale: Optional[float] = None,
                            status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``packed_attention`` over the paged cache: sequence i has seq_lens[i]
    positions in its pages and its queries (rows cu_seqlens[i] ..
    cu_seqlens[i + 1] - 1 of q) are the last of them: a whole prompt, or a chunk
    that continues one. Returns [T, nq * D]."""
    if not q.is_cuda:
        return torch_ref.paged_prefill_attention(q, k_pages, v_pages, page_table, seq_lens,
                                                 cu_seqlens, scale)
    return _ext().paged_prefill_attention(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens,
                                          scale, status)


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Log-probabilities of the tokens `ids` (int64 [R]) under softmax(logits)
    (bf16, fp16 or fp32 [R, V], V at most 2^21), the entropy of each row, and its `top_k` (at
    most 32) most likely tokens. Masked logits may be -inf. An id outside
    [0, V) gives NaN; a row without a finite maximum has no distribution and
    gives NaN throughout (its top_ids still follow the order of the logits, a
    NaN first)."""
    if not logits.is_cuda:
        return TokenLogprobs(*torch_ref.token_logprobs(logits, ids, top_k))
    return TokenLogprobs(*_ext().token_logprobs(logits, ids, top_k))
