"""CPU statements of the ragged-batch operators: against the padded path's ops on
the same data, and their refusals."""

import math

import pytest
import torch

from afd_demo_b200 import ops
from afd_demo_b200.ops import torch_ref


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _pool(lens, nkv, D, page, g):
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=g).tolist()
    kp = torch.full((sum(need) + 2, nkv, page, D), float("nan"))
    vp = kp.clone()
    table = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32)
    dense, at = [], 0
    for i, n in enumerate(lens):
        k, v = torch.randn(n, nkv, D, generator=g), torch.randn(n, nkv, D, generator=g)
        for p in range(n):
            if p % page == 0:
                table[i, p // page] = order[at]
                at += 1
            kp[table[i, p // page], :, p % page] = k[p]
            vp[table[i, p // page], :, p % page] = v[p]
        dense.append((k, v))
    return kp, vp, table, dense


def test_paged_decode_is_padded_decode():
    """Each sequence as the padded op computes it at its own length."""
    g = torch.Generator().manual_seed(0)
    lens = [0, 1, 17, 40]
    kp, vp, table, dense = _pool(lens, 2, 32, 16, g)
    q = torch.randn(4, 6, 32, generator=g)
    out = ops.paged_decode_attention(q, kp, vp, table, _i32(lens))
    assert not out[0].any()
    for b in range(1, 4):
        k, v = (x.transpose(0, 1)[None] for x in dense[b])
        want = torch_ref.attention(q[b:b + 1], k, v, 0, 1, lens[b] - 1)
        assert torch.allclose(out[b:b + 1], want, atol=1e-5)


def test_packed_is_padded_prefill():
    g = torch.Generator().manual_seed(1)
    lens = [3, 0, 21, 1]
    T = sum(lens)
    q, k, v = (torch.randn(T, h, 32, generator=g) for h in (6, 2, 2))
    cu = _i32([0, 3, 3, 24, 25])
    out = ops.packed_attention(q, k, v, cu)
    a = 0
    for n in lens:
        if n:
            kk, vv = (x[a:a + n].transpose(0, 1)[None] for x in (k, v))
            want = torch_ref.attention(q[a:a + n], kk, vv, 0, n, 0)
            assert torch.allclose(out[a:a + n], want, atol=1e-5)
        a += n


def test_packed_own_keys_and_paged_agree():
    """Chunks that continue a cache: packed keys and pages give the same; a query
    before the first key gives zeros."""
    g = torch.Generator().manual_seed(2)
    total, news = [20, 5, 33], [4, 7, 33]
    kp, vp, table, dense = _pool(total, 1, 16, 16, g)
    q = torch.randn(sum(news) + 2, 3, 16, generator=g)
    cu = _i32([0, 4, 11, 44])
    k, v = (torch.cat([d[i] for d in dense]) for i in (0, 1))
    a = ops.packed_attention(q, k, v, cu, _i32([0, 20, 25, 58]))
    b = ops.paged_prefill_attention(q, kp, vp, table, _i32(total), cu)
    assert torch.allclose(a, b, atol=1e-6)
    assert not a[4:6].any() and a[6:11].any() and not a[44:].any()


def test_norm_rope_stores_pages():
    g = torch.Generator().manual_seed(3)
    T, nq, nkv, D = 5, 4, 2, 16
    qkv = torch.randn(T, (nq + 2 * nkv) * D, generator=g)
    qn, kn = torch.rand(D, generator=g) + 0.5, torch.rand(D, generator=g) + 0.5
    rope = torch_ref.rope_table(64, D, 1e4, "cpu")
    kp, vp = torch.zeros(3, nkv, 16, D), torch.zeros(3, nkv, 16, D)
    pos, slots = _i32([7, 8, 0, 63, 1]), torch.tensor([33, 0, -1, 47, 16])
    q = ops.qk_norm_rope_paged(qkv, qn, kn, rope, kp, vp, pos, slots, nq, nkv, 1e-6)
    q2, k, v = ops.qk_norm_rope_packed(qkv, qn, kn, rope, pos, nq, nkv, 1e-6)
    assert torch.equal(q, q2) and q.shape == (T, nq, D)
    # one token through the padded op (same values in fp32 up to the last bits)
    kc, vc = torch.zeros(1, nkv, 64, D), torch.zeros(1, nkv, 64, D)
    for t in range(T):
        w = torch_ref.qk_norm_rope_cache(qkv[t:t + 1], qn, kn, rope, kc, vc, 0, 1, int(pos[t]),
                                         nq, nkv, 1e-6)
        assert torch.allclose(q[t], w[0], atol=1e-5)
        assert torch.allclose(k[t], kc[0, :, int(pos[t])], atol=1e-5)
        if slots[t] >= 0:
            p, r = divmod(int(slots[t]), 16)
            assert torch.equal(kp[p, :, r], k[t]) and torch.equal(vp[p, :, r], v[t])
    assert int((kp != 0).any(-1).any(1).sum()) == 4  # the token with a negative slot is not stored


def test_token_logprobs_definition():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(4, 50, generator=g) * 3
    x[1, 10:] = -math.inf
    x[2] = 1.0
    x[3] = -math.inf
    ids = torch.tensor([3, 9, 49, 0])
    r = ops.token_logprobs(x, ids, top_k=12)
    p = torch.softmax(x.double(), -1)
    assert torch.allclose(r.logprob[:3].double(), p[range(3), ids[:3]].log(), atol=1e-6)
    assert torch.allclose(r.entropy[:3].double(), torch.special.entr(p[:3]).sum(-1), atol=1e-5)
    assert r.top_ids[2].tolist() == list(range(12))
    assert r.top_ids[1, 10:].tolist() == [10, 11] and r.top_logprobs[1, 10] == -math.inf
    assert r.logprob[3].isnan() and r.entropy[3].isnan()
    assert ops.token_logprobs(x[:1], torch.tensor([50])).logprob.isnan().all()
    assert ops.token_logprobs(x, ids).top_ids.shape == (4, 0)


def test_refusals():
    q, kp = torch.randn(2, 4, 16), torch.randn(3, 2, 16, 16)
    t, n = _i32([[0], [1]]), _i32([1, 2])
    ops.paged_decode_attention(q, kp, kp, t, n)
    for bad in ((q[:, :3], kp, kp, t, n), (q, kp, kp[:2], t, n), (q, kp, kp, t.long(), n),
                (q, kp, kp, t[:1], n), (q, kp[..., :8], kp[..., :8], t, n),
                (q, kp[:, :, :8], kp[:, :, :8], t, n)):
        with pytest.raises(ValueError):
            ops.paged_decode_attention(*bad)
    with pytest.raises(ValueError):
        ops.packed_attention(q, q[:1], q[:1], _i32([0, 2]))
    with pytest.raises(ValueError):
        ops.packed_attention(q, q, q, torch.tensor([0, 2]))
    x = torch.randn(2, 9)
    for bad in ((x, torch.zeros(2, dtype=torch.int32), 1), (x, torch.zeros(1).long(), 1),
                (x, torch.zeros(2).long(), 10), (x.double(), torch.zeros(2).long(), 1)):
        with pytest.raises(ValueError):
            ops.token_logprobs(*bad)


@pytest.mark.parametrize("cu,same", [([0, 10, 5, 12], None), ([9, 0], None),
                                     ([0, 8, 70], [0, 8, 12]), ([-3, 5, 12], [0, 5, 12]),
                                     ([4, 6, 9], [4, 6, 9])])
def test_query_offsets_are_clamped_and_decreasing_ones_give_zeros(cu, same):
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(12, h, 32, generator=g) for h in (4, 2, 2))
    n = len(cu) - 1
    kp, vp, table, _ = _pool([20] * n, 2, 32, 16, g)
    for call in (lambda c: ops.packed_attention(q, k, v, _i32(c)),
                 lambda c: ops.paged_prefill_attention(q, kp, vp, table, _i32([20] * n), _i32(c))):
        out = call(cu)
        if same is None:
            assert not out.any()
        else:
            assert torch.equal(out, call(same))
            assert not out[: same[0]].any() and not out[same[-1]:].any()
            assert out[same[0]: same[-1]].any(-1).all()


def test_refusals_are_the_kernels():
    """What the bindings refuse by value, the CPU statements refuse too."""
    q, kv = torch.randn(4, 2, 32), torch.randn(4, 1, 32)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            ops.packed_attention(q, kv, kv, _i32([0, 4]), scale=scale)
    with pytest.raises(ValueError):
        ops.packed_attention(torch.randn(4, 129, 32), kv, kv, _i32([0, 4]))
    table, lens = _i32([[0]] * 4), _i32([1] * 4)
    for pages, kw in ((torch.randn(2, 1, 16, 32), dict(scale=-1.0)), (torch.randn(1, 1, 4112, 32), {}),
                      (torch.randn(0, 1, 16, 32), {})):
        with pytest.raises(ValueError):
            ops.paged_decode_attention(q, pages, pages, table, lens, **kw)
    wide, pages = torch.randn(4, 129, 32), torch.randn(2, 1, 16, 32)
    assert ops.paged_decode_attention(wide, pages, pages, table, lens).isfinite().all()
    with pytest.raises(ValueError):
        ops.paged_prefill_attention(wide, pages, pages, table, lens, _i32([0, 1, 2, 3, 4]))
    pages, w = torch.zeros(2, 4, 16, 32), torch.ones(32)
    with pytest.raises(ValueError):  # one kv head into pages of four
        ops.qk_norm_rope_paged(torch.randn(4, 4 * 32), w, w, torch.ones(8, 32), pages, pages.clone(),
                               _i32([0] * 4), torch.arange(4), 2, 1, 1e-6)


@pytest.mark.parametrize("scale", [1e-50, 1e39])
def test_scales_that_are_no_float_are_refused(scale):
    q = torch.randn(4, 2, 32)
    with pytest.raises(ValueError):
        ops.packed_attention(q, q, q, _i32([0, 4]), scale=scale)
