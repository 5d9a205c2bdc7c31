"""Ragged-batch kernels against plain statements in 64 bits.

Tolerances, per element, from the arithmetic, with u the largest relative error
of one rounding (2^-8 for bf16's 8 significant bits, 2^-11 for fp16's 11): an
attention output is rounded once (u |o|), its weights are rounded to the type
for the second product (u sum p |v|, and 2^-25 per key for fp16's subnormal
weights), and scores, exponentials and sums are fp32 (at most 2^-13 sum p |v| at
these sizes). Log-probabilities and entropies are fp32 sums of fp32 terms.
"""

import math

import pytest
import torch

from afd_demo_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAN = float("nan")


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    ops.ext()  # must load: no silent fallback


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cu(lens):
    return _i32([0] + torch.tensor(lens).cumsum(0).tolist()) if lens else _i32([0])


def _exact_rows(q, k, v, scale=None):
    """(out, sum p |v|, sum |v|) in 64 bits of q [n, nq, D] at the last n
    positions of k, v [m, nkv, D]."""
    n, nq, D = q.shape
    m, nkv, _ = k.shape
    z = torch.zeros(n, nq, D, dtype=torch.float64, device=DEV)
    if m == 0:
        return z, z.clone(), z.clone()
    G = nq // nkv
    q, k, v = q.double(), k.double(), v.double()
    s = torch.einsum("nkgd,mkd->kgnm", q.view(n, nkv, G, D), k) * (scale or D ** -0.5)
    pos = m - n + torch.arange(n, device=DEV)
    seen = torch.arange(m, device=DEV)[None] <= pos[:, None]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1))
    mix = lambda w, x: torch.einsum("kgnm,mkd->nkgd", w, x).reshape(n, nq, D)  # noqa: E731
    return mix(p, v), mix(p, v.abs()), mix(seen.double().expand_as(p), v.abs())


def _close(out, exact, dtype):
    o, a, t = (x.reshape(out.shape) for x in exact)
    u = U[dtype]
    tol = u * (1 + u) * o.abs() + (u + 2.0 ** -13) * a + 2.0 ** -25 * t + 2.0 ** -25
    bad = ~((out.double() - o).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((out.double() - o).abs().max()))


def _pool(g, lens, nkv, D, page, dtype, poison=True, extra=2):
    """Pages of the sequences in a scattered order (with NaN in every row that
    holds no position), the table (with ids past the pool where no page is
    needed) and the dense k, v."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=g, device=DEV).tolist()
    kp = torch.full((total, nkv, page, D), NAN if poison else 0.0, device=DEV, dtype=dtype)
    vp = kp.clone()
    table = torch.full((len(lens), max(need + [1]) + 1), 1 << 30, dtype=torch.int32)
    dense, at = [], 0
    for i, n in enumerate(lens):
        k, v = _randn(g, n, nkv, D, dtype=dtype), _randn(g, n, nkv, D, dtype=dtype)
        for j in range(need[i]):
            p, rows = order[at], min(page, n - j * page)
            table[i, j] = p
            kp[p, :, :rows] = k[j * page:j * page + rows].transpose(0, 1)
            vp[p, :, :rows] = v[j * page:j * page + rows].transpose(0, 1)
            at += 1
        dense.append((k, v))
    return kp, vp, table.to(DEV), dense


HEADS = [(8, 8, 128), (32, 4, 128), (16, 2, 64), (4, 2, 64), (3, 1, 128), (10, 2, 64),
         (14, 2, 128), (16, 1, 128), (24, 1, 64), (40, 1, 128)]
DTYPES = [torch.bfloat16, torch.float16]


# --------------------------------------------------------------------- decode --
@pytest.mark.parametrize("nq,nkv,D", HEADS)
@pytest.mark.parametrize("page", [16, 48, 64])
def test_paged_decode_lengths(nq, nkv, D, page):
    lens = [0, 1, 2, 15, 16, 17, 31, 47, 48, 49, 63, 64, 65, 127, 128, 129, 300, 1025]
    for dtype in DTYPES:
        g = _gen(nq + page)
        kp, vp, table, dense = _pool(g, lens, nkv, D, page, dtype)
        q = _randn(g, len(lens), nq, D, dtype=dtype, scale=2.0)
        out = ops.paged_decode_attention(q, kp, vp, table, _i32(lens))
        for b, (k, v) in enumerate(dense):
            _close(out[b:b + 1], _exact_rows(q[b:b + 1], k, v), dtype)
        assert not out[0].any()  # no key: zeros


@pytest.mark.parametrize("B,length", [(1, 1), (1, 40000), (2, 9000), (3, 513), (150, 40),
                                      (300, 129), (1100, 5)])
def test_paged_decode_batches(B, length):
    g = _gen(B)
    lens = [max(0, length - 7 * (i % 5)) for i in range(B)]
    kp, vp, table, dense = _pool(g, lens, 2, 128, 64, torch.bfloat16)
    q = _randn(g, B, 8, 128, scale=1.5)
    seq = _i32(lens)
    out = ops.paged_decode_attention(q, kp, vp, table, seq)
    for b in range(0, B, max(1, B // 17)):
        _close(out[b:b + 1], _exact_rows(q[b:b + 1], *dense[b]), torch.bfloat16)
    assert torch.equal(out, ops.paged_decode_attention(q, kp, vp, table, seq))  # same bits


def test_paged_decode_large_scores_and_scale():
    """Scores far apart (one key takes all) and a scale of the caller's."""
    g = _gen(5)
    lens = [200, 4097]
    kp, vp, table, dense = _pool(g, lens, 1, 128, 32, torch.bfloat16)
    q = _randn(g, 2, 4, 128, scale=30.0)
    out = ops.paged_decode_attention(q, kp, vp, table, _i32(lens))
    for b in range(2):
        _close(out[b:b + 1], _exact_rows(q[b:b + 1], *dense[b]), torch.bfloat16)
    out = ops.paged_decode_attention(q, kp, vp, table, _i32(lens), scale=0.003)
    for b in range(2):
        _close(out[b:b + 1], _exact_rows(q[b:b + 1], *dense[b], scale=0.003), torch.bfloat16)


@pytest.mark.parametrize("nq,nkv,D", [(8, 2, 128), (32, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens", [[1, 40, 300, 16], [9000], [20, 30000, 1]])
def test_paged_decode_nan_is_kept(nq, nkv, D, lens):
    """NaN in a query, in one key, in a block of keys and in every key reach the
    heads that see them and no others: items of one CTA and items cut over several."""
    g = _gen(13)
    G, page = nq // nkv, 32
    kp, vp, table, dense = _pool(g, lens, nkv, D, page, torch.bfloat16)
    q = _randn(g, len(lens), nq, D)
    seq = _i32(lens)
    want = ops.paged_decode_attention(q, kp, vp, table, seq).view(len(lens), nq, D)
    assert want.isfinite().all()

    def check(got, b, heads):
        got = got.view(len(lens), nq, D)
        hit = torch.zeros(len(lens), nq, dtype=torch.bool, device=DEV)
        hit[b, heads] = True
        assert got[hit].isnan().all() and torch.equal(got[~hit], want[~hit])

    b = lens.index(max(lens))
    q2 = q.clone()
    q2[b, nq - 2, 5] = NAN
    check(ops.paged_decode_attention(q2, kp, vp, table, seq), b, [nq - 2])
    for b, n in enumerate(lens):
        for first, count in ((0, 1), (n - 1, 1), (n // 2 // 16 * 16, 16), (0, n)):
            k2 = kp.clone()
            at = torch.arange(first, min(n, first + count), device=DEV)
            k2[table[b].long()[at // page], 1, at % page, 3] = NAN
            check(ops.paged_decode_attention(q, k2, vp, table, seq), b, list(range(G, 2 * G)))


@pytest.mark.parametrize("dtype,power", [(t, p) for t in DTYPES for p in (0, 8, 16, 24)] +
                         [(torch.bfloat16, p) for p in (32, 48, 90)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("n,total", [(40, 700), (8, 5000)])
def test_attention_of_huge_scores(dtype, power, sign, n, total):
    """Finite scores of any size, exact in fp32: 2^power times a whole number of 13 at
    most (13 scale log2(e) is no float). From 2^8 on the keys with the largest share the
    weight and the others have none (2^-30 of it at most)."""
    g = _gen(20)
    nq, nkv, D, pages, a = 4, 2, 64, -(-total // 64), power // 2
    q = torch.zeros(n, nq, D, device=DEV, dtype=dtype)
    q[..., 3] = 2.0 ** a
    k, v = torch.zeros(total, nkv, D, device=DEV, dtype=dtype), _randn(g, total, nkv, D, dtype=dtype)
    k[..., 3] = (sign * torch.randint(0, 14, (total, nkv), generator=g, device=DEV)
                 * 2.0 ** (power - a)).to(dtype)
    kp, vp = (torch.cat([x, x[:64 * pages - total]]).view(pages, 64, nkv, D).transpose(1, 2)
              .contiguous() for x in (k, v))
    table = torch.arange(pages, device=DEV, dtype=torch.int32)[None]
    exact = _exact_rows(q, k, v)
    for out in (ops.packed_attention(q, k, v, _cu([n]), _cu([total])),
                ops.paged_prefill_attention(q, kp, vp, table, _i32([total]), _cu([n]))):
        _close(out, exact, dtype)
    _close(ops.paged_decode_attention(q[-1:], kp, vp, table, _i32([total])),
           tuple(x[-1:] for x in exact), dtype)


def test_paged_decode_strides():
    """q as a view of a projection; the pool as a layer of a larger buffer, with
    k and v interleaved page by page; a table wider than its view."""
    g = _gen(6)
    lens = [70, 1, 33]
    kp, vp, table, dense = _pool(g, lens, 2, 64, 16, torch.bfloat16)
    both = torch.stack([kp, vp], 1)  # [pages, 2, nkv, page, D]
    qkv = _randn(g, 3, 12 * 64)
    q = qkv[:, : 8 * 64].view(3, 8, 64)
    want = ops.paged_decode_attention(q.contiguous(), kp, vp, table, _i32(lens))
    wide = torch.cat([table, table], 1)[:, : table.shape[1]]
    assert torch.equal(ops.paged_decode_attention(q, both[:, 0], both[:, 1], wide, _i32(lens)),
                       want)
    # rows off a 16-byte boundary are copied
    odd = torch.empty(3 * 8 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(3, 8, 64)
    odd.copy_(q)
    assert torch.equal(ops.paged_decode_attention(odd, kp, vp, table, _i32(lens)), want)


def test_paged_decode_bad_indices_are_recorded():
    g = _gen(7)
    lens = [40, 40, 40]
    kp, vp, table, dense = _pool(g, lens, 2, 128, 16, torch.bfloat16)
    q = _randn(g, 3, 8, 128)
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    ok = ops.paged_decode_attention(q, kp, vp, table, _i32(lens), status=status)
    assert status.tolist()[0] == 0
    # a length beyond the table, and a negative one: no key
    out = ops.paged_decode_attention(q, kp, vp, table, _i32([40, 16 * table.shape[1] + 1, -1]),
                                     status=status)
    assert status.tolist()[0] == 3
    assert torch.equal(out[0], ok[0]) and not out[1:].any()
    # a page id outside the pool: its keys and values read as zeros
    status.zero_()
    for bad in (-1, kp.shape[0], 1 << 30):
        t = table.clone()
        t[1, 1] = bad
        out = ops.paged_decode_attention(q, kp, vp, t, _i32(lens), status=status)
        assert status.tolist()[0] == 3
        status.zero_()
        k, v = (x.clone() for x in dense[1])
        k[16:32] = 0
        v[16:32] = 0
        _close(out[1:2], _exact_rows(q[1:2], k, v), torch.bfloat16)
        assert torch.equal(out[0], ok[0]) and torch.equal(out[2], ok[2])


def test_paged_decode_graph_replay_and_streams():
    """A captured call follows lengths and tables as they change; calls on two
    streams do not disturb each other."""
    g = _gen(8)
    lens = [100, 700, 1, 64]
    kp, vp, table, dense = _pool(g, lens, 4, 128, 64, torch.bfloat16)
    q = _randn(g, 4, 32, 128)
    seq = _i32([1, 1, 1, 1])
    call = lambda: ops.paged_decode_attention(q, kp, vp, table, seq)  # noqa: E731
    call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        graph.capture_begin()
        out = call()
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
    for now in ([1, 5, 1, 64], lens, [0, 699, 1, 3]):
        seq.copy_(_i32(now))
        graph.replay()
        for b, n in enumerate(now):
            k, v = dense[b]
            _close(out[b:b + 1], _exact_rows(q[b:b + 1], k[:n], v[:n]), torch.bfloat16)
    seq.copy_(_i32(lens))
    want = call()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


# --------------------------------------------------------------------- prompts --
PACKS = [[1], [2, 1, 3], [15, 16, 17, 0, 31, 32, 33], [127, 128, 129, 1], [0, 0, 5, 0],
         [300, 64, 511, 1, 70]]


@pytest.mark.parametrize("nq,nkv,D", HEADS)
@pytest.mark.parametrize("lens", PACKS)
def test_packed_attention(nq, nkv, D, lens):
    for dtype in DTYPES:
        g = _gen(sum(lens) + nq)
        T = sum(lens)
        q = _randn(g, T, nq, D, dtype=dtype, scale=2.0)
        k, v = _randn(g, T, nkv, D, dtype=dtype), _randn(g, T, nkv, D, dtype=dtype)
        out = ops.packed_attention(q, k, v, _cu(lens))
        a = 0
        for n in lens:
            _close(out[a:a + n], _exact_rows(q[a:a + n], k[a:a + n], v[a:a + n]), dtype)
            a += n


@pytest.mark.parametrize("nq,nkv,D", [(32, 4, 128), (16, 2, 64), (7, 1, 128), (2, 2, 128)])
def test_packed_attention_long(nq, nkv, D):
    lens = [2111, 7, 1500]
    g = _gen(D)
    T = sum(lens)
    qkv = _randn(g, T, (nq + 2 * nkv) * D, scale=1.5)  # strided views of one projection
    q = qkv[:, : nq * D].view(T, nq, D)
    k = qkv[:, nq * D: (nq + nkv) * D].view(T, nkv, D)
    v = qkv[:, (nq + nkv) * D:].view(T, nkv, D)
    out = ops.packed_attention(q, k, v, _cu(lens))
    a = 0
    for n in lens:
        _close(out[a:a + n], _exact_rows(q[a:a + n], k[a:a + n], v[a:a + n]), torch.bfloat16)
        a += n
    assert torch.equal(out, ops.packed_attention(q, k, v, _cu(lens)))


@pytest.mark.parametrize("nq,nkv,D", [(8, 1, 128), (3, 1, 64), (2, 2, 128)])
def test_packed_attention_own_keys(nq, nkv, D):
    """Keys with offsets of their own: more keys than queries, as many, fewer
    (queries before the first key get zeros) and none; rows past the last offset
    get zeros."""
    q_lens, k_lens = [5, 40, 130, 3, 20, 1], [300, 40, 17, 0, 129, 1000]
    g = _gen(3)
    q = _randn(g, sum(q_lens) + 37, nq, D)
    k, v = (_randn(g, sum(k_lens), nkv, D) for _ in range(2))
    out = ops.packed_attention(q, k, v, _cu(q_lens), _cu(k_lens))
    a = b = 0
    for n, m in zip(q_lens, k_lens):
        _close(out[a:a + n], _exact_rows(q[a:a + n], k[b:b + m], v[b:b + m]), torch.bfloat16)
        if n > m:
            assert not out[a:a + n - m].any()
        a, b = a + n, b + m
    assert not out[a:].any()


def test_packed_attention_neighbours_do_not_mix():
    """NaN and infinities in one sequence leave the others as they are."""
    g = _gen(4)
    lens = [100, 60, 200]
    q, k, v = (_randn(g, 360, 4, 128) for _ in range(3))
    want = ops.packed_attention(q, k, v, _cu(lens))
    for bad in (NAN, math.inf, -math.inf):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for x in (q2, k2, v2):
            x[100:160] = bad
        out = ops.packed_attention(q2, k2, v2, _cu(lens))
        assert torch.equal(out[:100], want[:100]) and torch.equal(out[160:], want[160:])


@pytest.mark.parametrize("nq,nkv,D", [(32, 4, 128), (8, 2, 64), (2, 2, 128)])
def test_packed_attention_what_nan_reaches(nq, nkv, D):
    """In k: the queries that see it. In v: those, and at most 63 + 256 nkv / nq
    positions before them, in its dim alone. Whole keys and split ones."""
    g = _gen(17)
    G = nq // nkv
    for news, total in ((1000, 1000), (16, 5000)):
        q = _randn(g, news, nq, D)
        k, v = _randn(g, total, nkv, D), _randn(g, total, nkv, D)
        cu, cu_k = _cu([news]), _cu([total])
        want = ops.packed_attention(q, k, v, cu, cu_k).view(news, nkv, G, D)
        for back in (1, news // 2 + 3, news):
            at = total - back  # a position that the last `back` queries see
            first = news - back
            for bad in (NAN, math.inf):
                k2, v2 = k.clone(), v.clone()
                k2[at, 1] = bad
                v2[at, 1, 7] = bad
                got = ops.packed_attention(q, k2, v, cu, cu_k).view(news, nkv, G, D)
                assert torch.equal(got[:, 0], want[:, 0])
                assert torch.equal(got[:first], want[:first])
                if bad != bad:
                    assert got[first:, 1].isnan().all()
                got = ops.packed_attention(q, k, v2, cu, cu_k).view(news, nkv, G, D)
                near = max(0, first - 63 - 256 // G)
                assert torch.equal(got[:near], want[:near])
                assert not got[first:, 1, :, 7].isfinite().any()
                got[:, 1, :, 7] = want[:, 1, :, 7]
                assert torch.equal(got, want)


def _leave_nan(rows, width):
    """NaN where the next output of this size will lie."""
    torch.full((rows, width), NAN, device=DEV, dtype=torch.bfloat16)


@pytest.mark.parametrize("first", [1, 31, 32, 37, 300])
@pytest.mark.parametrize("nq,nkv,D", [(32, 4, 128), (4, 2, 64)])
def test_packed_attention_rows_before_the_first_offset(first, nq, nkv, D):
    """They get zeros, as the rows past the last offset do, and the sequences what
    they get without them; also where the keys are split."""
    g = _gen(14)
    lens, after = [60, 0, 200, 3], 41
    T = first + sum(lens) + after
    q = _randn(g, T, nq, D, scale=2.0)
    k, v = _randn(g, T, nkv, D), _randn(g, T, nkv, D)
    cu = _cu(lens) + first
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    _leave_nan(T, nq * D)
    out = ops.packed_attention(q, k, v, cu, status=status)
    a = first
    for n in lens:
        _close(out[a:a + n], _exact_rows(q[a:a + n], k[a:a + n], v[a:a + n]), torch.bfloat16)
        a += n
    assert not out[:first].any() and not out[a:].any()
    totals = [5000, 40]
    kp, vp, table, dense = _pool(g, totals, nkv, D, 64, torch.bfloat16)
    T = first + 8 + 5
    _leave_nan(T, nq * D)
    out = ops.paged_prefill_attention(q[:T], kp, vp, table, _i32(totals),
                                      _i32([first, first + 8, T]), status=status)
    _close(out[first:first + 8], _exact_rows(q[first:first + 8], *dense[0]), torch.bfloat16)
    _close(out[first + 8:], _exact_rows(q[first + 8:T], *dense[1]), torch.bfloat16)
    assert not out[:first].any() and status.tolist()[0] == 0


@pytest.mark.parametrize("T", [1, 200])
def test_attention_of_rows_that_share_memory(T):
    """One row expanded to many, rows that overlap, and single rows of any stride."""
    g = _gen(16)
    flat = _randn(g, T * 8 + 4 * 64)

    def forms(h):
        yield _randn(g, 1, h, 64).expand(T, h, 64)
        yield flat.as_strided((T, h, 64), (8, 64, 1))
        if T == 1:
            yield flat.as_strided((1, h, 64), (3, 64, 1))

    cu, dec = _cu([T]), torch.zeros(T, 1, dtype=torch.int32, device=DEV)
    kp, vp = _randn(g, 1, 2, 64, 64), _randn(g, 1, 2, 64, 64)
    for q in forms(4):
        for k in forms(2):
            v = next(forms(2))
            out = ops.packed_attention(q, k, v, cu)
            assert torch.equal(out, ops.packed_attention(*(x.contiguous() for x in (q, k, v)), cu))
            _close(out, _exact_rows(q, k, v), torch.bfloat16)
        args = (kp, vp, dec, torch.full((T,), 40, dtype=torch.int32, device=DEV))
        assert torch.equal(ops.paged_decode_attention(q, *args),
                           ops.paged_decode_attention(q.contiguous(), *args))


def test_packed_attention_bad_offsets_are_recorded():
    g = _gen(9)
    q, k, v = (_randn(g, 64, 2, 64) for _ in range(3))
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.packed_attention(q, k, v, _i32([0, 30, 64]), status=status)
    assert status.tolist()[0] == 0
    ops.packed_attention(q, k, v, _i32([0, 64]), _i32([0, 65]), status=status)
    assert status.tolist()[0] == 3


@pytest.mark.parametrize("cu,T", [([0, 10, 5, 12], 12), ([0, 200, 40, 300], 300), ([9, 0], 40),
                                  ([0, 64, 70], 64), ([-3, 20, 64], 64), ([0, 1 << 30, 64], 64),
                                  (list(range(700)) + [698, 700], 700)])
def test_packed_attention_bad_query_offsets(cu, T):
    """Recorded, and a defined output: what the clamped offsets give, or zeros where
    they decrease; whole keys and split ones; the next call is not disturbed."""
    g = _gen(15)
    q, k, v = _randn(g, T, 8, 128), _randn(g, T, 2, 128), _randn(g, T, 2, 128)
    n = len(cu) - 1
    kp, vp, table, _ = _pool(g, [3000 if n < 10 else 20] * n, 2, 128, 64, torch.bfloat16)
    lens = _i32([3000 if n < 10 else 20] * n)
    clamped = [min(max(c, 0), T) for c in cu]
    for call in (lambda c, s=None: ops.packed_attention(q, k, v, _i32(c), status=s),
                 lambda c, s=None: ops.paged_prefill_attention(q, kp, vp, table, lens, _i32(c),
                                                               status=s)):
        good = [0] * n + [T]
        before = call(good)
        want = call(clamped) if clamped == sorted(clamped) else torch.zeros_like(before)
        for _ in range(2):
            status = torch.zeros(2, dtype=torch.int32, device=DEV)
            _leave_nan(T, 8 * 128)
            out = call(cu, status)
            assert status.tolist()[0] == 3 and torch.equal(out, want)
        assert torch.equal(call(good), before)


@pytest.mark.parametrize("nq,nkv,D", [(32, 4, 128), (16, 2, 64), (6, 2, 128)])
@pytest.mark.parametrize("page", [16, 48, 64, 128, 256])
def test_paged_prefill(nq, nkv, D, page):
    """Whole prompts, chunks that continue the cache, single tokens and an empty
    sequence, with NaN in every page row that holds no position."""
    news, total = [40, 1, 200, 0, 17, 128], [40, 513, 777, 33, 17, 1000]
    for dtype in DTYPES:
        g = _gen(page)
        kp, vp, table, dense = _pool(g, total, nkv, D, page, dtype)
        q = _randn(g, sum(news), nq, D, dtype=dtype, scale=2.0)
        status = torch.zeros(2, dtype=torch.int32, device=DEV)
        out = ops.paged_prefill_attention(q, kp, vp, table, _i32(total), _cu(news), status=status)
        a = 0
        for n, (k, v) in zip(news, dense):
            _close(out[a:a + n], _exact_rows(q[a:a + n], k, v), dtype)
            a += n
        assert status.tolist()[0] == 0


def test_paged_prefill_bad_indices_are_recorded():
    g = _gen(10)
    kp, vp, table, dense = _pool(g, [100, 100], 1, 128, 16, torch.bfloat16)
    q = _randn(g, 20, 8, 128)
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    cu = _i32([0, 10, 20])
    ok = ops.paged_prefill_attention(q, kp, vp, table, _i32([100, 100]), cu, status=status)
    assert status.tolist()[0] == 0
    out = ops.paged_prefill_attention(q, kp, vp, table, _i32([100, 10000]), cu, status=status)
    assert status.tolist()[0] == 3 and torch.equal(out[:10], ok[:10]) and not out[10:].any()
    status.zero_()
    t = table.clone()
    t[1, 2] = kp.shape[0]
    out = ops.paged_prefill_attention(q, kp, vp, t, _i32([100, 100]), cu, status=status)
    assert status.tolist()[0] == 3 and torch.equal(out[:10], ok[:10])
    k, v = (x.clone() for x in dense[1])
    k[32:48] = 0
    v[32:48] = 0
    _close(out[10:], _exact_rows(q[10:], k, v), torch.bfloat16)


@pytest.mark.parametrize("nq,nkv,D", [(32, 4, 128), (16, 2, 64), (3, 1, 128), (40, 1, 128), (8, 8, 64)])
@pytest.mark.parametrize("news,total", [
    ([16], [20011]), ([1], [1024]), ([1], [1023]), ([1, 16, 5, 0], [20000, 4097, 1087, 700]),
    ([40, 3], [8200, 0]), ([130], [5000]), ([9, 0, 1, 1], [512, 0, 1, 64])])
def test_paged_prefill_few_tokens_over_long_caches(nq, nkv, D, news, total):
    """The keys are split over CTAs and the parts joined."""
    for dtype in DTYPES:
        g = _gen(sum(total))
        kp, vp, table, dense = _pool(g, total, nkv, D, 64, dtype)
        q = _randn(g, sum(news), nq, D, dtype=dtype, scale=2.0)
        status = torch.zeros(2, dtype=torch.int32, device=DEV)
        args = (q, kp, vp, table, _i32(total), _cu(news))
        out = ops.paged_prefill_attention(*args, status=status)
        a = 0
        for n, (k, v) in zip(news, dense):
            if k.shape[0] == 0:
                assert not out[a:a + n].any()
            else:
                _close(out[a:a + n], _exact_rows(q[a:a + n], k, v), dtype)
            a += n
        assert status.tolist()[0] == 0
        assert torch.equal(out, ops.paged_prefill_attention(*args))  # same bits


@pytest.mark.parametrize("D", [64, 128])
def test_packed_attention_split_keys_rows_without_any(D):
    """Queries before the first key, and rows past the last offset, in a call
    whose keys are split; a part's keys may all lie after a row's position."""
    g = _gen(D)
    q_lens, k_lens = [70, 30], [2100, 20]
    q = _randn(g, 110, 4, D, scale=2.0)
    k, v = _randn(g, 2120, 2, D), _randn(g, 2120, 2, D)
    out = ops.packed_attention(q, k, v, _cu(q_lens), _cu(k_lens))
    _close(out[:70], _exact_rows(q[:70], k[:2100], v[:2100]), torch.bfloat16)
    assert not out[70:80].any() and not out[100:].any()
    _close(out[80:100], _exact_rows(q[80:100], k[2100:], v[2100:]), torch.bfloat16)


def test_paged_prefill_split_replays_with_other_lengths():
    """One captured call, replayed as the cache grows from no split to many parts."""
    g = _gen(21)
    kp, vp, table, dense = _pool(g, [9000], 4, 128, 64, torch.bfloat16)
    q, cu, seq = _randn(g, 8, 32, 128), _i32([0, 8]), _i32([9000])
    ops.paged_prefill_attention(q, kp, vp, table, seq, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefill_attention(q, kp, vp, table, seq, cu)
    for n in (9000, 8, 600, 1100, 64, 8999):
        seq.fill_(n)
        graph.replay()
        _close(out, _exact_rows(q, *(x[:n] for x in dense[0])), torch.bfloat16)


# ----------------------------------------------------------------- norm + RoPE --
def _exact_norm_rope(x, w, cs, eps):
    D = x.shape[-1]
    x = x.double()
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    c, s = cs.double()[:, None, : D // 2], cs.double()[:, None, D // 2:]
    lo, hi = x[..., : D // 2], x[..., D // 2:]
    return (torch.cat([lo * c - hi * s, hi * c + lo * s], -1),
            torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1))


@pytest.mark.parametrize("T", [0, 1, 3, 33, 500])
@pytest.mark.parametrize("nq,nkv,D", [(32, 4, 128), (16, 2, 64), (3, 3, 128), (5, 1, 64)])
def test_qk_norm_rope_paged(T, nq, nkv, D):
    """u |y| for the one rounding and 2^-20 of the two products for the fp32
    arithmetic before it."""
    eps = 1e-6
    for dtype in DTYPES:
        g = _gen(T + D)
        wide = _randn(g, T, (nq + 2 * nkv) * D + 64, dtype=dtype, scale=3.0)
        qkv = wide[:, 64:]
        qn, kn = (1 + 0.3 * torch.randn(2, D, generator=g, device=DEV)).to(dtype)
        rope = ops.rope_table(777, D, 1e6, DEV)
        pos = torch.randint(0, 777, (T,), generator=g, device=DEV).to(torch.int32)
        page, n = 16, T // 16 + 3
        kp, vp = _randn(g, n, nkv, page, D, dtype=dtype), _randn(g, n, nkv, page, D, dtype=dtype)
        k0, v0 = kp.clone(), vp.clone()
        slots = torch.randperm(n * page, generator=g, device=DEV)[:T]
        slots[::7] = -1
        q = ops.qk_norm_rope_paged(qkv, qn, kn, rope, kp, vp, pos, slots, nq, nkv, eps)
        x = qkv.reshape(T, nq + 2 * nkv, D)
        cs = rope[pos.long()]
        eq, aq = _exact_norm_rope(x[:, :nq], qn, cs, eps)
        ek, ak = _exact_norm_rope(x[:, nq:nq + nkv], kn, cs, eps)
        u = U[dtype]

        def near(got, want, mag):
            tol = u * (1 + u) * want.abs() + 2.0 ** -20 * mag + 2.0 ** -25
            return bool(((got.double() - want).abs() <= tol).all())

        assert q.shape == (T, nq, D) and near(q, eq, aq)
        st = slots >= 0
        p, r = slots[st] // page, slots[st] % page
        assert near(kp[p, :, r], ek[st], ak[st]) and torch.equal(vp[p, :, r], x[st, nq + nkv:])
        # nothing else was touched
        kp[p, :, r], vp[p, :, r] = k0[p, :, r], v0[p, :, r]
        assert torch.equal(kp, k0) and torch.equal(vp, v0)
        q2, k2, v2 = ops.qk_norm_rope_packed(qkv, qn, kn, rope, pos, nq, nkv, eps)
        assert torch.equal(q2, q) and near(k2, ek, ak) and torch.equal(v2, x[:, nq + nkv:])


def test_qk_norm_rope_bad_indices_are_recorded():
    g = _gen(2)
    qkv = _randn(g, 4, 6 * 64)
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    rope = ops.rope_table(32, 64, 1e4, DEV)
    kp, vp = (torch.zeros(2, 1, 16, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    call = lambda pos, slots: ops.qk_norm_rope_paged(  # noqa: E731
        qkv, w, w, rope, kp, vp, _i32(pos), torch.tensor(slots, device=DEV), 4, 1, 1e-6,
        status=status)
    call([0, 1, 2, 31], [0, 1, -1, 31])
    assert status.tolist()[0] == 0
    kp.zero_(), vp.zero_()
    call([0, 1, 2, 3], [32, 1 << 40, -1, -5])
    assert status.tolist()[0] == 3 and not kp.any() and not vp.any()
    status.zero_()
    call([0, 1, 2, 32], [0, 1, 2, 3])
    assert status.tolist()[0] == 3


# ----------------------------------------------------------------- log-probs --
def _check_logprobs(x, ids, k):
    """fp32 terms: each within 2^-20 of max(1, its magnitude); the order of the
    top tokens exactly."""
    r = ops.token_logprobs(x, ids, top_k=k)
    xd = x.double()
    ls = xd - xd.amax(-1, keepdim=True)  # the lowest finite values cancel here first
    ls = ls - ls.exp().sum(-1, keepdim=True).log()
    p = ls.exp()
    ent = -torch.where(p == 0, torch.zeros_like(p), p * ls).sum(-1)
    top = torch.sort(xd + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]

    def near(a, b):
        same = (a == b) | (a.isnan() & b.isnan())
        return bool((same | ((a - b).abs() <= 2.0 ** -20 * b.abs().clamp_min(1.0))).all())

    assert near(r.logprob.double(), ls.gather(1, ids[:, None])[:, 0])
    assert near(r.entropy.double(), ent)
    assert torch.equal(r.top_ids, top)
    assert near(r.top_logprobs.double(), ls.gather(1, top))
    assert r.top_ids.shape == r.top_logprobs.shape == (x.shape[0], k)


def _near_logprobs(r, x, ids, k):
    """``_check_logprobs`` of a result that is there."""
    xd = x.double()
    ls = xd - xd.amax(-1, keepdim=True)
    ls = ls - ls.exp().sum(-1, keepdim=True).log()
    p = ls.exp()
    ent = -torch.where(p == 0, torch.zeros_like(p), p * ls).sum(-1)
    top = torch.sort(xd + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]
    for got, want in ((r.logprob, ls.gather(1, ids[:, None])[:, 0]), (r.entropy, ent),
                      (r.top_logprobs, ls.gather(1, top))):
        off = (got.double() - want).abs()
        off = torch.where(got.double() == want, torch.zeros_like(off), off)
        worst = (off / want.abs().clamp_min(1.0)).nan_to_num(math.inf, math.inf)
        assert bool((worst <= 2.0 ** -20).all()), float(worst.max())
    assert torch.equal(r.top_ids, top)


@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 2), (2, 31, 5), (5, 255, 32), (4, 256, 0),
                                   (7, 257, 20), (1, 50257, 20), (33, 4096, 8), (2, 151936, 32),
                                   (300, 1000, 3), (1, 300000, 20), (0, 100, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_token_logprobs(R, V, k, dtype):
    g = _gen(V)
    x = _randn(g, R, V, dtype=dtype, scale=4.0)
    _check_logprobs(x, torch.randint(V, (R,), generator=g, device=DEV), k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_token_logprobs_hard_rows(dtype):
    """Equal logits, sorted ones both ways, masks of -inf and of the type's
    lowest value, one token left, signed zeros, large magnitudes."""
    V, k = 5001, 20
    g = _gen(1)
    base = _randn(g, V, dtype=dtype, scale=3.0)
    low = torch.finfo(dtype).min
    one = torch.full((V,), -math.inf, device=DEV, dtype=dtype)
    one[4321] = 2.0
    few = torch.full((V,), -math.inf, device=DEV, dtype=dtype)
    few[[7, 700, 4999]] = torch.tensor([1.0, 5.0, 1.0], device=DEV, dtype=dtype)
    lowest = base.clone()
    lowest[torch.rand(V, generator=g, device=DEV) < 0.99] = low
    zeros = torch.zeros(V, device=DEV, dtype=dtype)
    zeros[::3] = -0.0
    x = torch.stack([torch.zeros_like(base), base.sort().values,
                     base.sort(descending=True).values, one, few, lowest,
                     torch.full_like(base, low), zeros, base * 2000, base - 30000,
                     torch.full_like(base, 7.0)])
    _check_logprobs(x, torch.full((x.shape[0],), 4321, device=DEV), k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("repeat", [1, 25])
def test_token_logprobs_finite_fills(dtype, repeat):
    """Rows, and blocks of rows, filled with a finite value of large magnitude, as
    masks do; few rows (split over CTAs) and many (a CTA each)."""
    V, k = 5001, 20
    g = _gen(11)
    base = _randn(g, V, dtype=dtype, scale=3.0)
    rows = []
    for c in (-1e9, -1e10, -1e12, -1e20, -1e29, 1e9, 1e10, 1e20, 1e29):
        first, last, one = base.clone(), base.clone(), base.clone()
        first[:1024] = c
        last[:4608] = c
        one[2048:2560] = c
        steps = torch.full_like(base, c) * (1 + torch.randint(3, (V,), generator=g, device=DEV)
                                            * 2.0 ** (-7 if dtype == torch.bfloat16 else -23))
        rows += [torch.full_like(base, c), first, last, one, steps.to(dtype)]
    x = torch.stack(rows).repeat(repeat, 1)
    _check_logprobs(x, torch.randint(V, (x.shape[0],), generator=g, device=DEV), k)


def _many_blocks(g, R, V, dtype):
    """Rows of V logits that rise, fall, are shifted and have their first blocks
    masked, in turn."""
    x = _randn(g, R, V, dtype=dtype, scale=3.0)
    x[0::6] = x[0::6].sort(dim=-1).values
    x[1::6] = x[1::6].sort(dim=-1, descending=True).values
    x[2::6, : V - 100] = -math.inf
    x[3::6, : V // 2] = -1e4
    x[4::6] = (x[4::6].float() - 30000.0).to(dtype)
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,V,k,offset", [(600, 50257, 20, 7), (1200, 50264, 3, 0),
                                          (700, 20000, 32, 0), (600, 262656, 5, 0)])
def test_token_logprobs_many_blocks_a_warp(R, V, k, offset, dtype):
    """One CTA a row, several blocks a warp: rows on the 16-byte grid and off it."""
    g = _gen(R)
    x = torch.zeros(R, V + offset, dtype=dtype, device=DEV)[:, offset:]
    x.copy_(_many_blocks(g, R, V, dtype))
    ids = torch.randint(V, (R,), generator=g, device=DEV)
    for a in range(0, R, 200):  # the 64-bit form in pieces, the operator on all rows
        r = ops.token_logprobs(x, ids, k)
        _near_logprobs(ops.TokenLogprobs(*(t[a:a + 200] for t in r)), x[a:a + 200],
                       ids[a:a + 200], k)


@pytest.mark.parametrize("shift", [0.0, 1e3, 1e4, 3e4, 1e6, -1e6, 3e7])
def test_token_logprobs_shifted_rows_that_rise(shift):
    """A maximum that moves from block to block of a warp, far from zero: the sums
    so far keep their weight."""
    g = _gen(12)
    x = (torch.randn(600, 20000, generator=g, device=DEV) * 3.0).sort(dim=-1).values
    x[300:] = x[300:, torch.randperm(20000, generator=g, device=DEV)]
    x += shift
    _check_logprobs(x, torch.randint(20000, (600,), generator=g, device=DEV), 5)


def test_token_logprobs_no_distribution():
    V = 3000
    x = torch.randn(5, V, device=DEV)
    x[0] = -math.inf
    x[1, 77] = math.inf
    x[2, 5] = NAN
    x[3, 2999] = -NAN
    r = ops.token_logprobs(x, torch.full((5,), 9, device=DEV), top_k=4)
    for t in (r.logprob, r.entropy, r.top_logprobs):
        assert t[:4].isnan().all() and not t[4].isnan().any()
    assert r.top_ids[0].tolist() == [0, 1, 2, 3]
    assert r.top_ids[1, 0] == 77 and r.top_ids[2, 0] == 5 and r.top_ids[3, 0] == 2999
    # ids that name no token
    r = ops.token_logprobs(x[4:].repeat(3, 1), torch.tensor([-1, V, 1 << 40], device=DEV))
    assert r.logprob.isnan().all() and not r.entropy.isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs_strides(dtype):
    """Rows at any offset of a wider buffer, and columns of a transposed one."""
    g = _gen(3)
    for width, a, V in [(1001, 0, 1001), (1003, 1, 1000), (4099, 3, 4096), (2048, 8, 777)]:
        x = _randn(g, 6, width, dtype=dtype, scale=3.0)[:, a:a + V]
        _check_logprobs(x, torch.randint(V, (6,), generator=g, device=DEV), 7)
    x = _randn(g, 900, 5, dtype=dtype, scale=3.0).t()
    _check_logprobs(x, torch.randint(900, (5,), generator=g, device=DEV), 7)


def test_token_logprobs_streams():
    g = _gen(4)
    x = _randn(g, 2, 151936, scale=3.0)
    ids = torch.randint(151936, (2,), generator=g, device=DEV)
    want = ops.token_logprobs(x, ids, 20)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(ops.token_logprobs(x, ids, 20))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))


# ------------------------------------------------------------------ refusals --
def test_refusals():
    g = _gen(0)
    q, k, v = (_randn(g, 8, 4, 128) for _ in range(3))
    pages = _randn(g, 4, 4, 16, 128)
    table, lens, cu = _i32([[0]] * 8), _i32([1] * 8), _i32([0, 8])
    dec = lambda q=q, kp=pages, vp=pages, t=table, n=lens: (  # noqa: E731
        ops.paged_decode_attention(q, kp, vp, t, n))
    dec()
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :96]), dict(q=q[0]),
                dict(kp=pages.half()), dict(vp=pages[:2]), dict(kp=pages[..., :64]),
                dict(kp=pages[:, :, :8], vp=pages[:, :, :8]), dict(t=table.long()),
                dict(t=table[:3]), dict(n=lens[:3]), dict(n=lens.long()), dict(n=lens.cpu()),
                dict(kp=pages.transpose(1, 2), vp=pages.transpose(1, 2))):
        with pytest.raises(ValueError):
            dec(**bad)
    packed = lambda q=q, k=k, v=v, c=cu, ck=None: ops.packed_attention(q, k, v, c, ck)  # noqa: E731
    packed()
    for bad in (dict(k=k.half()), dict(k=k[:7]), dict(c=cu.long()), dict(ck=_i32([0, 4, 8])),
                dict(q=q.double()), dict(k=k[:7], v=v[:7]), dict(c=_i32([[0, 8]])),
                dict(k=k[:, :3], v=v[:, :3])):
        with pytest.raises(ValueError):
            packed(**bad)
    with pytest.raises(ValueError):
        ops.paged_prefill_attention(q, pages, pages, table, lens, cu)  # one sequence, 8 tables
    x, ids = _randn(g, 3, 100), torch.zeros(3, dtype=torch.int64, device=DEV)
    for a in ((x.double(), ids, 1), (x, ids.int(), 1), (x, ids[:2], 1), (x, ids, 33),
              (x, ids, 101), (x, ids, -1), (x[0], ids, 1)):
        with pytest.raises(ValueError):
            ops.token_logprobs(*a)
    qkv, w = _randn(g, 8, 12 * 128), torch.ones(128, device=DEV, dtype=torch.bfloat16)
    rope, pos = ops.rope_table(16, 128, 1e4, DEV), _i32([0] * 8)
    slots = torch.arange(8, device=DEV)
    args = [qkv, w, w, rope, pages, pages.clone(), pos, slots, 4, 4, 1e-6]
    ops.qk_norm_rope_paged(*args)
    for i, bad in ((0, qkv[:, :-128]), (1, w[:96]), (2, w.float()), (3, rope.half()),
                   (6, pos.long()), (7, slots.int()), (8, 5)):
        with pytest.raises(ValueError):
            ops.qk_norm_rope_paged(*[bad if j == i else a for j, a in enumerate(args)])


def test_page_tables_past_the_positions_of_an_int_are_refused():
    q = torch.zeros(1, 1, 64, device=DEV, dtype=torch.half)
    pages = torch.zeros(1, 1, 4096, 64, device=DEV, dtype=torch.half)
    for columns, fits in ((2 ** 18 - 1, True), (2 ** 18, False)):
        table = torch.zeros(1, columns, dtype=torch.int32, device=DEV)
        for call in (lambda t: ops.paged_decode_attention(q, pages, pages, t, _i32([5000])),
                     lambda t: ops.paged_prefill_attention(q, pages, pages, t, _i32([5000]),
                                                           _i32([0, 1]))):
            if fits:
                assert not call(table).any()
            else:
                with pytest.raises(ValueError):
                    call(table)


def test_status_of_other_layouts_is_refused():
    """The kernels write two neighbouring words."""
    g = _gen(18)
    q, pages = _randn(g, 2, 4, 64), _randn(g, 2, 4, 16, 64)
    one, three = _i32([0]), _i32([0, 0, 0])
    for bad in (one, one.expand(2), three[::2], three.long(), three.cpu()):
        for call in (lambda s: ops.paged_decode_attention(q, pages, pages, _i32([[0], [1]]),
                                                          _i32([3, 99]), status=s),
                     lambda s: ops.packed_attention(q, q, q, _i32([0, 2]), status=s)):
            with pytest.raises(ValueError):
                call(bad)
    ops.paged_decode_attention(q, pages, pages, _i32([[0], [1]]), _i32([3, 99]), status=three)
    assert three.tolist()[0] == 3 and three.tolist()[2] == 0


@pytest.mark.parametrize("scale", [0.0, -1.0, NAN, math.inf, 1e-50, 1e39])
def test_scales_that_are_no_positive_float_are_refused(scale):
    g = _gen(19)
    q, pages, table, lens = _randn(g, 2, 4, 64), _randn(g, 2, 4, 16, 64), _i32([[0]] * 2), _i32([3, 4])
    for call in (lambda: ops.paged_decode_attention(q, pages, pages, table, lens, scale=scale),
                 lambda: ops.packed_attention(q, q, q, _i32([0, 2]), scale=scale),
                 lambda: ops.paged_prefill_attention(q, pages, pages, table, lens, _i32([0, 1, 2]),
                                                     scale=scale)):
        with pytest.raises(ValueError):
            call()
