"""Ragged generation and scoring on CPU in fp32, against the padded path run on each
prompt alone."""

import pytest
import torch

from afd_demo_b200.models import DisaggregatedQwenModel, PagedKVCache
from afd_demo_b200.utils import device as devmod


@pytest.fixture(scope="module")
def model():
    devmod.init_backend("cpu")
    return DisaggregatedQwenModel.from_pretrained("tiny", device="cpu", dtype=torch.float32,
                                                  max_seq_len=96, max_batch_size=1)


def _prompts(model, lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(model.config.vocab_size, (n,), generator=g) for n in lens]


def _alone(model, prompt, new):
    out = model.generate(prompt[None], max_new_tokens=new, do_sample=False, use_decode_dbo=False)
    return out[0, prompt.numel():]


@pytest.mark.parametrize("chunk", [None, 1, 7, 64])
def test_generate_matches_each_prompt_alone(model, chunk):
    prompts = _prompts(model, [1, 33, 16, 5])
    gen = model.ragged(num_pages=12, page_size=16)
    outs = gen.generate(prompts, 6, top_logprobs=3, prefill_chunk_size=chunk)
    assert gen.cache.free_pages == 12
    for p, o in zip(prompts, outs):
        assert torch.equal(o.tokens, _alone(model, p, 6))
        # greedy: the token is the most likely one, and its log-probability is the top's
        assert torch.equal(o.top_ids[:, 0], o.tokens)
        assert torch.allclose(o.top_logprobs[:, 0], o.logprobs)
        assert o.logprobs.shape == o.entropy.shape == (6,) and o.top_ids.shape == (6, 3)


def test_score_matches_the_padded_forward(model):
    seqs = _prompts(model, [9, 2, 40], seed=1)
    gen = model.ragged(num_pages=1, page_size=16)
    for rows in (2048, 7):
        for p, r in zip(seqs, gen.score(seqs, top_logprobs=2, rows_at_once=rows)):
            ls = torch.log_softmax(model.forward_prefill(p[None])[0, :-1].float(), -1)
            assert torch.allclose(r.logprob, ls.gather(1, p[1:, None])[:, 0], atol=1e-4)
            assert torch.allclose(r.entropy, -(ls.exp() * ls).sum(-1), atol=1e-4)
            assert r.top_ids.shape == (p.numel() - 1, 2)


def test_generated_tokens_score_as_they_were_drawn(model):
    prompts = _prompts(model, [12, 3], seed=2)
    gen = model.ragged(num_pages=8, page_size=16)
    outs = gen.generate(prompts, 5, do_sample=True, generator=torch.Generator().manual_seed(3))
    scored = gen.score([torch.cat([p, o.tokens]) for p, o in zip(prompts, outs)])
    for p, o, s in zip(prompts, outs, scored):
        assert torch.allclose(s.logprob[p.numel() - 1:], o.logprobs, atol=1e-4)


def test_eos_ends_a_sequence(model):
    prompts = _prompts(model, [8, 20], seed=4)
    gen = model.ragged(num_pages=8, page_size=16)
    free = gen.generate(prompts, 6)
    eos = int(free[0].tokens[2])
    outs = gen.generate(prompts, 6, eos_token_id=eos)
    for f, o in zip(free, outs):
        hit = (f.tokens == eos).nonzero()
        n = int(hit[0]) + 1 if len(hit) else 6
        assert torch.equal(o.tokens, f.tokens[:n])


def test_refusals_leave_the_pool_whole(model):
    gen = model.ragged(num_pages=3, page_size=16)
    p = _prompts(model, [20, 20])
    for bad in (dict(prompts=[], max_new_tokens=1), dict(prompts=[[]], max_new_tokens=1),
                dict(prompts=[[-1]], max_new_tokens=1),
                dict(prompts=[[model.config.vocab_size]], max_new_tokens=1),
                dict(prompts=p, max_new_tokens=0), dict(prompts=p, max_new_tokens=80),
                dict(prompts=p, max_new_tokens=2, prefill_chunk_size=0),
                dict(prompts=p, max_new_tokens=2)):  # four pages needed, three there
        with pytest.raises(ValueError):
            gen.generate(**bad)
        assert gen.cache.free_pages == 3
    for bad in (dict(num_pages=0), dict(num_pages=1, page_size=8), dict(num_pages=1, page_size=20)):
        with pytest.raises(ValueError):
            model.ragged(**bad)


def test_paged_cache_reuses_pages():
    from afd_demo_b200.config import PRESETS
    c = PagedKVCache(PRESETS["tiny"](), 6, 16, "cpu", torch.float32)
    a, b = c.allocate(33), c.allocate(1)
    assert c.free_pages == 2 and c.table([a, b]).shape == (2, 3)
    with pytest.raises(ValueError):
        c.allocate(33)
    held = set(c.table([a])[0].tolist())
    c.release(a)
    d = c.allocate(80)
    assert c.free_pages == 0 and held <= set(c.table([d])[0].tolist())
    assert not set(c.table([b])[0, :1].tolist()) & set(c.table([d])[0].tolist())


@pytest.mark.parametrize("code", [1, 3])
def test_what_a_kernel_recorded_is_raised_once(model, code):
    from afd_demo_b200.ops.checks import AFDBoundsError

    gen = model.ragged(num_pages=2, page_size=16)
    p = _prompts(model, [5])
    for call in (lambda: gen.generate(p, 2), lambda: gen.score(p)):
        gen.status = torch.tensor([code, 223], dtype=torch.int32)
        with pytest.raises(AFDBoundsError if code == 3 else RuntimeError, match="site=223"):
            call()
        assert gen.cache.free_pages == 2
        call()


def test_generate_up_to_the_last_position(model):
    """As the padded path does: the last new token needs no position."""
    p = _prompts(model, [90])
    gen = model.ragged(num_pages=6, page_size=16)
    out = gen.generate(p, 7)
    assert torch.equal(out[0].tokens, _alone(model, p[0], 7))
    with pytest.raises(ValueError):
        gen.generate(p, 8)
    assert gen.cache.free_pages == 6


def test_more_refusals(model):
    with pytest.raises(ValueError):
        model.ragged(num_pages=1, page_size=4112)
    for rows in (0, -1):
        with pytest.raises(ValueError):
            model.ragged(num_pages=1, page_size=16).score([[1, 2]], rows_at_once=rows)
