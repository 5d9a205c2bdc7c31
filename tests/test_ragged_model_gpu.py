"""Ragged generation and scoring of the GPU test models: the paged steps against one
packed pass over the same tokens, page sizes, chunked prefill, reuse of pages.

Tolerance: both passes round their logits to bf16; below 16 in magnitude (checked)
that is 2^-5 a logit, of the token's and of the log-sum each, in either pass, and
the activations' own roundings in two layers may do as much again: 2^-2 in all.
"""

import pytest
import torch

from afd_demo_b200 import ops
from afd_demo_b200.models import DisaggregatedQwenModel
from afd_demo_b200.utils import device as devmod

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -2


@pytest.fixture(scope="module", params=["small", "mini"])
def model(request):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    ops.ext()
    devmod.init_backend("cuda")
    return DisaggregatedQwenModel.from_pretrained(request.param, device="cuda:0",
                                                  dtype=torch.bfloat16, max_seq_len=512,
                                                  max_batch_size=2)


def _prompts(model, lens):
    g = torch.Generator().manual_seed(0)
    return [torch.randint(model.config.vocab_size, (n,), generator=g) for n in lens]


@pytest.mark.parametrize("page,chunk", [(64, None), (16, 50)])
def test_paged_steps_score_as_one_packed_pass(model, page, chunk):
    prompts = _prompts(model, [1, 130, 17, 300, 64])
    need = sum(-(-(p.numel() + 7) // page) for p in prompts)
    gen = model.ragged(num_pages=need, page_size=page)
    before = ops.LAUNCHES.count
    for _ in range(2):  # the second time on pages that were used before
        outs = gen.generate(prompts, 8, top_logprobs=4, prefill_chunk_size=chunk)
        assert gen.cache.free_pages == need
    assert ops.LAUNCHES.count > before
    full = [torch.cat([p, o.tokens.cpu()]) for p, o in zip(prompts, outs)]
    for p, o, s in zip(prompts, outs, gen.score(full, top_logprobs=4)):
        n = p.numel() - 1
        assert float(s.entropy.max()) < 16 and o.logprobs.isfinite().all()
        assert (s.logprob[n:] - o.logprobs).abs().max() < TOL
        assert (s.entropy[n:] - o.entropy).abs().max() < TOL
        assert torch.equal(o.top_ids[:, 0], o.tokens)
        assert (o.top_logprobs[:, :-1] >= o.top_logprobs[:, 1:]).all()


def test_ragged_agrees_with_the_padded_model(model):
    """The same prompts through the padded forward, one at a time (its norm and RoPE
    round at every step)."""
    prompts = _prompts(model, [40, 128])
    gen = model.ragged(num_pages=1)
    for p, s in zip(prompts, gen.score(prompts)):
        logits = model.forward_prefill(p[None].cuda())[0, :-1].float()
        assert float(logits.abs().max()) < 16
        want = torch.log_softmax(logits, -1).gather(1, p[1:, None].cuda())[:, 0]
        assert (s.logprob - want).abs().max() < TOL


def test_bad_indices_raise_and_leave_the_generator_usable(model):
    """What the kernels record is read: pages outside the pool, positions past the
    RoPE table."""
    from afd_demo_b200.ops.checks import AFDBoundsError

    prompts = _prompts(model, [20, 70])
    gen = model.ragged(num_pages=8, page_size=32)
    want = gen.generate(prompts, 4)
    table = gen.cache.table
    gen.cache.table = lambda seqs: table(seqs) + 8
    with pytest.raises(AFDBoundsError):
        gen.generate(prompts, 4)
    gen.cache.table = table
    assert gen.cache.free_pages == 8
    most, gen.max_positions = gen.max_positions, 1 << 20
    with pytest.raises(AFDBoundsError):
        gen.score(_prompts(model, [most + 1]))
    gen.max_positions = most
    for a, b in zip(gen.generate(prompts, 4), want):
        assert torch.equal(a.tokens, b.tokens)
    gen.score(prompts)
