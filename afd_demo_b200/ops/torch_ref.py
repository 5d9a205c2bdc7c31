"""Pure-PyTorch statements of every op the framework runs.

These are (1) the CPU execution path (the reference's ``--backend cpu`` /
gloo mode, src/utils/device.py:55-63) and (2) the oracle the CUDA kernels are
tested against. Numerics follow HF Qwen3-MoE (transformers 5.x,
``modeling_qwen3_moe``): RMSNorm in fp32 then cast, weight multiply in the
activation dtype; router softmax in fp32 over the projected logits, top-k,
renormalise; experts ``down(silu(gate(x)) * up(x)) * w``.

The kernels accumulate in fp32 and round once where HF rounds several times,
so GPU-vs-oracle comparisons are tolerance based.
"""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    dt = x.dtype
    xf = x.float()
    var = xf.pow(2).mean(-1, keepdim=True)
    return w * (xf * torch.rsqrt(var + eps)).to(dt)


def sum_rmsnorm(parts: Sequence[torch.Tensor], w: torch.Tensor, eps: float
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """x = sum(parts) (fp32 sum, one rounding); returns (x, rmsnorm(x))."""
    if len(parts) == 1:
        x = parts[0]
    else:
        acc = parts[0].float()
        for p in parts[1:]:
            acc = acc + p.float()
        x = acc.to(parts[0].dtype)
    return x, rmsnorm(x, w, eps)


def linear(x: torch.Tensor, w: torch.Tensor, residual: Optional[torch.Tensor] = None
           ) -> torch.Tensor:
    y = F.linear(x, w)
    if residual is not None:
        y = y + residual
    return y


def rope_table(max_pos: int, head_dim: int, theta: float, device, dtype=torch.float32
               ) -> torch.Tensor:
    """[max_pos, head_dim] table: cos in the first half, sin in the second,
    for the half-dim frequencies (HF default RoPE). Values are rounded to the
    activation dtype as HF does (``cos.to(x.dtype)``) but stored as fp32."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.int64, device=device)
                                .float() / head_dim))
    pos = torch.arange(max_pos, device=device, dtype=torch.float32)
    freqs = pos[:, None] * inv_freq[None, :]
    cos = freqs.cos().to(dtype).float()
    sin = freqs.sin().to(dtype).float()
    return torch.cat([cos, sin], dim=-1).contiguous()


def _rotate_half(x):
    h = x.shape[-1] // 2
    return torch.cat((-x[..., h:], x[..., :h]), dim=-1)


def apply_rope(x: torch.Tensor, cos_sin: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """x [T, nh, D]; pos [T] int; table from rope_table."""
    D = x.shape[-1]
    cs = cos_sin[pos.long()]  # [T, D]
    cos = torch.cat([cs[:, : D // 2], cs[:, : D // 2]], -1).to(x.dtype)[:, None, :]
    sin = torch.cat([cs[:, D // 2:], cs[:, D // 2:]], -1).to(x.dtype)[:, None, :]
    return (x * cos) + (_rotate_half(x) * sin)


def qk_norm_rope_cache(qkv: torch.Tensor, q_norm_w: torch.Tensor, k_norm_w: torch.Tensor,
                       cos_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       batch_offset: int, q_len: int, start_pos: int, n_q: int, n_kv: int,
                       eps: float) -> torch.Tensor:
    """Split qkv [T, (nq+2nkv)*D]; per-head RMSNorm of q and k; RoPE; write k,v
    into the cache at rows batch_offset + t // q_len, positions
    start_pos + t % q_len. Returns q [T, nq, D]."""
    T = qkv.shape[0]
    D = q_norm_w.shape[0]
    q = qkv[:, : n_q * D].view(T, n_q, D)
    k = qkv[:, n_q * D: (n_q + n_kv) * D].view(T, n_kv, D)
    v = qkv[:, (n_q + n_kv) * D:].view(T, n_kv, D)
    q = rmsnorm(q, q_norm_w, eps)
    k = rmsnorm(k, k_norm_w, eps)
    t = torch.arange(T, device=qkv.device)
    pos = start_pos + t % q_len
    b = batch_offset + t // q_len
    q = apply_rope(q, cos_sin, pos)
    k = apply_rope(k, cos_sin, pos)
    k_cache[b, :, pos] = k.to(k_cache.dtype)
    v_cache[b, :, pos] = v.to(v_cache.dtype)
    return q.contiguous()


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              batch_offset: int, q_len: int, start_pos: int,
              key_range: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """Causal GQA attention of q [B*q_len, nq, D] against cache rows
    [batch_offset, batch_offset+B) and positions [0, start_pos+q_len).
    Query i of a sequence sits at position start_pos+i and sees keys <= it.
    `key_range` = (lo, hi), int tensors indexed by cache row: only keys in
    [lo, hi) are visible (padding); a query that sees no key outputs zeros.
    Returns [B*q_len, nq*D]."""
    T, nq, D = q.shape
    B = T // q_len
    kv_len = start_pos + q_len
    k = k_cache[batch_offset:batch_offset + B, :, :kv_len].float()
    v = v_cache[batch_offset:batch_offset + B, :, :kv_len].float()
    nkv = k.shape[1]
    g = nq // nkv
    k = k.repeat_interleave(g, dim=1)
    v = v.repeat_interleave(g, dim=1)
    qf = q.view(B, q_len, nq, D).transpose(1, 2).float()  # [B, nq, q_len, D]
    s = torch.matmul(qf, k.transpose(-1, -2)) / math.sqrt(D)
    qpos = start_pos + torch.arange(q_len, device=q.device)
    kpos = torch.arange(kv_len, device=q.device)
    mask = (kpos[None, :] > qpos[:, None])[None, None]  # [1, 1, q_len, kv_len]
    if key_range is not None:
        lo = key_range[0][batch_offset:batch_offset + B].to(q.device).long()
        hi = key_range[1][batch_offset:batch_offset + B].to(q.device).long()
        out_of_range = (kpos[None, :] < lo[:, None]) | (kpos[None, :] >= hi[:, None])
        mask = mask | out_of_range[:, None, None, :]
    s = s.masked_fill(mask, float("-inf"))
    p = torch.softmax(s, dim=-1).nan_to_num(0.0)  # rows with no visible key -> 0
    o = torch.matmul(p, v)  # [B, nq, q_len, D]
    return o.transpose(1, 2).reshape(T, nq * D).to(q.dtype)


def router_topk(h: torch.Tensor, post_norm_w: torch.Tensor, w_router: torch.Tensor,
                top_k: int, eps: float, norm_topk_prob: bool = True
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """post-attention RMSNorm + router: returns (normed x, ids int32 [T,k],
    weights fp32 [T,k])."""
    xn = rmsnorm(h, post_norm_w, eps)
    logits = F.linear(xn, w_router)
    probs = torch.softmax(logits, dim=-1, dtype=torch.float32)
    w, ids = torch.topk(probs, top_k, dim=-1)
    if norm_topk_prob:
        w = w / w.sum(-1, keepdim=True)
    return xn, ids.to(torch.int32), w.float()


def moe_experts(xn: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                w_gate_up: torch.Tensor, w_down: torch.Tensor, expert_start: int = 0
                ) -> torch.Tensor:
    """Sum over the token's top-k experts that live in [expert_start,
    expert_start + E_local) of w * down(silu(gate x) * up x). fp32 accumulate."""
    T, H = xn.shape
    E_loc = w_gate_up.shape[0]
    I = w_gate_up.shape[1] // 2
    out = torch.zeros(T, H, dtype=torch.float32, device=xn.device)
    local = ids.long() - expert_start
    for e in range(E_loc):
        tok, slot = torch.where(local == e)
        if tok.numel() == 0:
            continue
        x = xn[tok]
        gu = F.linear(x, w_gate_up[e])
        a = F.silu(gu[:, :I]) * gu[:, I:]
        y = F.linear(a, w_down[e]).float() * weights[tok, slot, None]
        out.index_add_(0, tok, y)
    return out


def dense_mlp(xn: torch.Tensor, w_gate_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    I = w_gate_up.shape[0] // 2
    gu = F.linear(xn, w_gate_up)
    return F.linear(F.silu(gu[:, :I]) * gu[:, I:], w_down)


def ffn_layer(h: torch.Tensor, post_norm_w, w_router, w_gate_up, w_down, top_k: int,
              eps: float, expert_start: int = 0, add_residual: bool = True,
              norm_topk_prob: bool = True, dense: Optional[Tuple] = None) -> torch.Tensor:
    """Full FFN block on the pre-combined input h = attn_out + residual:
    returns h + moe(norm(h)) (or only the local-expert partial sum when
    add_residual is False)."""
    if dense is not None:
        xn = rmsnorm(h, post_norm_w, eps)
        y = dense_mlp(xn, *dense).float()
    else:
        xn, ids, w = router_topk(h, post_norm_w, w_router, top_k, eps, norm_topk_prob)
        y = moe_experts(xn, ids, w, w_gate_up, w_down, expert_start)
    if add_residual:
        y = y + h.float()
    return y.to(h.dtype)


def argmax(logits: torch.Tensor) -> torch.Tensor:
    return logits.argmax(dim=-1)


def stack_parts(parts: List[torch.Tensor]) -> torch.Tensor:
    return torch.stack(parts, 0)


# ---------------------------------------------- ragged batches, paged cache --
def _check(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _check_heads(nq: int, nkv: int) -> None:
    _check(nkv >= 1 and nq >= 1 and nq % nkv == 0,
           f"query heads ({nq}) must be a multiple of the kv heads ({nkv})")


def _check_pool(k_pages: torch.Tensor, v_pages: torch.Tensor, D: int) -> None:
    _check(k_pages.dim() == 4 and k_pages.shape == v_pages.shape,
           "k_pages and v_pages must be [pages, kv heads, page_size, head_dim], laid out alike")
    _check(k_pages.shape[3] == D, "q and the pages differ in head_dim")
    _check(k_pages.shape[0] >= 1, "the pool has no page")
    _check(16 <= k_pages.shape[2] <= 4096 and k_pages.shape[2] % 16 == 0,
           "page_size must be a multiple of 16, at most 4096")


def _check_scale(scale: Optional[float]) -> None:
    s = 1.0 if scale is None else float(torch.tensor(scale, dtype=torch.float32))
    _check(s > 0 and math.isfinite(s), "scale must be positive, in 32 bits")


def qk_norm_rope(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
                 rope: torch.Tensor, positions: torch.Tensor, nq: int, nkv: int, eps: float
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-head RMSNorm and RoPE in fp32 with one rounding: (q, k)."""
    D = q_norm.shape[0]
    T = qkv.shape[0]
    _check_heads(nq, nkv)
    _check(qkv.dim() == 2 and qkv.shape[1] == (nq + 2 * nkv) * D,
           f"qkv must be [tokens, {(nq + 2 * nkv) * D}]")
    _check(positions.dtype == torch.int32 and positions.numel() == T,
           f"positions must be a contiguous int32 tensor of {T} on the same device")
    x = qkv[:, : (nq + nkv) * D].reshape(T, nq + nkv, D).float()
    w = torch.cat([q_norm.expand(nq, D), k_norm.expand(nkv, D)]).float()
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    cs = rope[positions.long()][:, None]
    cos, sin = cs[..., : D // 2], cs[..., D // 2:]
    lo, hi = x[..., : D // 2], x[..., D // 2:]
    x = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(qkv.dtype)
    return x[:, :nq].contiguous(), x[:, nq:].contiguous()


def qk_norm_rope_paged(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
                       rope: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                       positions: torch.Tensor, slots: torch.Tensor, nq: int, nkv: int,
                       eps: float) -> torch.Tensor:
    """``qk_norm_rope`` with k and v stored at the page rows `slots` (negative:
    not stored). Returns q."""
    D, T = q_norm.shape[0], qkv.shape[0]
    _check_pool(k_pages, v_pages, D)
    _check(k_pages.shape[1] == nkv, "the pages' heads differ from qkv's")
    _check(slots.dtype == torch.int64 and slots.numel() == T,
           "slots must be a contiguous int64 tensor, one per token")
    q, k = qk_norm_rope(qkv, q_norm, k_norm, rope, positions, nq, nkv, eps)
    at = slots >= 0
    page, row = slots[at] // k_pages.shape[2], slots[at] % k_pages.shape[2]
    k_pages[page, :, row] = k[at]
    v_pages[page, :, row] = qkv[:, (nq + nkv) * D:].reshape(T, nkv, D)[at]
    return q


def _causal_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float]
                 ) -> torch.Tensor:
    """q [n, nq, D] as the last n of the m positions of k, v [m, nkv, D]; a
    query before the first key gives zeros. [n, nq * D]."""
    n, nq, D = q.shape
    m, nkv, _ = k.shape
    kf = k.float().repeat_interleave(nq // nkv, 1)
    vf = v.float().repeat_interleave(nq // nkv, 1)
    s = torch.einsum("nhd,mhd->hnm", q.float(), kf) * (D ** -0.5 if scale is None else scale)
    pos = m - n + torch.arange(n, device=q.device)
    s = s.masked_fill(torch.arange(m, device=q.device)[None] > pos[:, None], float("-inf"))
    p = torch.softmax(s, -1).masked_fill((pos < 0)[None, :, None], 0.0)
    return torch.einsum("hnm,mhd->nhd", p, vf).reshape(n, nq * D).to(q.dtype)


def _paged_rows(pages: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    """The first n positions of a sequence's pages, [n, nkv, D]."""
    ps = pages.shape[2]
    x = pages[table[: (n + ps - 1) // ps].long()]
    return x.transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[3])[:n]


def _offsets(cu: torch.Tensor, rows: int) -> List[int]:
    return [min(max(c, 0), rows) for c in cu.tolist()]


def _decrease(offsets: List[int]) -> bool:
    return any(b < a for a, b in zip(offsets, offsets[1:]))


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None
                     ) -> torch.Tensor:
    _check(q.dim() == 3 and k.dim() == 3 and k.shape == v.shape and k.shape[2] == q.shape[2],
           "k and v must be [rows, kv heads, head_dim] with the queries' head_dim")
    _check_heads(q.shape[1], k.shape[1])
    _check(q.shape[1] // k.shape[1] <= 128, "at most 128 query heads per kv head")
    _check_scale(scale)
    _check(cu_seqlens_k is not None or k.shape[0] == q.shape[0],
           "k has other rows than q: give cu_seqlens_k")
    cu_k = cu_seqlens if cu_seqlens_k is None else cu_seqlens_k
    for c in (cu_seqlens, cu_k):
        _check(c.dtype == torch.int32 and c.numel() == cu_seqlens.numel() >= 1,
               "cu_seqlens must hold n + 1 int32 offsets")
    out = torch.zeros(q.shape[0], q.shape[1] * q.shape[2], dtype=q.dtype, device=q.device)
    cq, ck = _offsets(cu_seqlens, q.shape[0]), _offsets(cu_k, k.shape[0])
    if _decrease(cq):
        return out
    for i in range(len(cq) - 1):
        if cq[i + 1] > cq[i] and ck[i + 1] > ck[i]:
            out[cq[i]:cq[i + 1]] = _causal_rows(q[cq[i]:cq[i + 1]], k[ck[i]:ck[i + 1]],
                                                v[ck[i]:ck[i + 1]], scale)
    return out


def paged_prefill_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                            page_table: torch.Tensor, seq_lens: torch.Tensor,
                            cu_seqlens: torch.Tensor, scale: Optional[float] = None
                            ) -> torch.Tensor:
    _check(q.dim() != 3 or k_pages.dim() != 4 or q.shape[1] <= 128 * k_pages.shape[1],
           "at most 128 query heads per kv head")
    return _paged_attention(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale)


def _paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     page_table: torch.Tensor, seq_lens: torch.Tensor, cu_seqlens: torch.Tensor,
                     scale: Optional[float]) -> torch.Tensor:
    _check(q.dim() == 3, "q must be [rows, heads, head_dim]")
    _check_pool(k_pages, v_pages, q.shape[2])
    _check_heads(q.shape[1], k_pages.shape[1])
    _check_scale(scale)
    n = cu_seqlens.numel() - 1
    for t in (page_table, seq_lens, cu_seqlens):
        _check(t.dtype == torch.int32, "page_table, seq_lens and cu_seqlens must be int32")
    _check(page_table.dim() == 2 and page_table.shape[0] == n and seq_lens.numel() == n,
           f"page_table and seq_lens must have a row for each of the {n} sequences")
    out = torch.zeros(q.shape[0], q.shape[1] * q.shape[2], dtype=q.dtype, device=q.device)
    cq = _offsets(cu_seqlens, q.shape[0])
    if _decrease(cq):
        return out
    for i in range(n):
        m = int(seq_lens[i])
        if cq[i + 1] > cq[i] and m > 0:
            out[cq[i]:cq[i + 1]] = _causal_rows(q[cq[i]:cq[i + 1]],
                                                _paged_rows(k_pages, page_table[i], m),
                                                _paged_rows(v_pages, page_table[i], m), scale)
    return out


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           page_table: torch.Tensor, seq_lens: torch.Tensor,
                           scale: Optional[float] = None) -> torch.Tensor:
    cu = torch.arange(q.shape[0] + 1, dtype=torch.int32)
    return _paged_attention(q, k_pages, v_pages, page_table, seq_lens, cu, scale)


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    _check(logits.dim() == 2 and 1 <= logits.shape[1] <= 1 << 21,
           "logits must be [rows, vocab] of 1 to 2097152 values a row")
    _check(logits.dtype in (torch.bfloat16, torch.float16, torch.float32),
           "logits must be bf16, fp16 or fp32")
    R, V = logits.shape
    _check(ids.dtype == torch.int64 and ids.numel() == R,
           "ids must be a contiguous int64 tensor, one per row")
    _check(0 <= top_k <= min(32, V), "top_k must be at most 32 and the vocabulary")
    ls = torch.log_softmax(logits.float(), -1)
    p = ls.exp()
    entropy = -(torch.where(p == 0, torch.zeros_like(p), p * ls)).sum(-1)
    ok = (ids >= 0) & (ids < V)
    lp = ls.gather(1, ids.clamp(0, V - 1)[:, None])[:, 0].masked_fill(~ok, float("nan"))
    # stable: equal logits in index order; a NaN sorts first
    top = torch.sort(logits.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top_k]
    return lp, entropy, top, ls.gather(1, top)
