"""Example: a batch of prompts of different lengths over the paged cache, with the
log-probabilities of what was generated.

    python -m afd_demo_b200.scripts.ragged_generate --model-name small --prompts 8 \
        --max-prompt 300 --new-tokens 16 --top-logprobs 3

Prompts are random token ids (no tokenizer is needed). Prints one line per
sequence and the time per generated token.
"""

from __future__ import annotations

import argparse
import random
import time

import torch


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model-name", default="small", help="preset or checkpoint directory")
    ap.add_argument("--prompts", type=int, default=8)
    ap.add_argument("--min-prompt", type=int, default=1)
    ap.add_argument("--max-prompt", type=int, default=300)
    ap.add_argument("--new-tokens", type=int, default=16)
    ap.add_argument("--prefill-chunk-size", type=int, default=None)
    ap.add_argument("--page-size", type=int, default=64)
    ap.add_argument("--top-logprobs", type=int, default=3)
    ap.add_argument("--sample", action="store_true", help="sample instead of greedy decoding")
    ap.add_argument("--backend", choices=("cuda", "cpu"),
                    default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)

    from ..models import DisaggregatedQwenModel
    from ..utils import device as devmod

    devmod.init_backend(a.backend)
    cuda = a.backend == "cuda"
    positions = a.max_prompt + a.new_tokens
    model = DisaggregatedQwenModel.from_pretrained(
        a.model_name, device="cuda:0" if cuda else "cpu",
        dtype=torch.bfloat16 if cuda else torch.float32, max_seq_len=positions, max_batch_size=1)
    rng = random.Random(a.seed)
    lens = [rng.randint(a.min_prompt, a.max_prompt) for _ in range(a.prompts)]
    prompts = [[rng.randrange(model.config.vocab_size) for _ in range(n)] for n in lens]
    pages = sum(-(-(n + a.new_tokens) // a.page_size) for n in lens)
    gen = model.ragged(pages, a.page_size)

    def run():
        return gen.generate(prompts, a.new_tokens, top_logprobs=a.top_logprobs,
                            do_sample=a.sample, prefill_chunk_size=a.prefill_chunk_size)

    run()  # warm-up
    if cuda:
        torch.cuda.synchronize()
    t = time.perf_counter()
    outs = run()
    if cuda:
        torch.cuda.synchronize()
    t = time.perf_counter() - t
    for n, o in zip(lens, outs):
        print(f"prompt {n:5d} tokens -> {o.tokens.tolist()}  mean logprob "
              f"{float(o.logprobs.mean()):.3f}  mean entropy {float(o.entropy.mean()):.3f}")
    full = [p + o.tokens.tolist() for p, o in zip(prompts, outs)]
    scored = gen.score(full)
    worst = max(float((s.logprob[n - 1:] - o.logprobs).abs().max())
                for n, s, o in zip(lens, scored, outs))
    print(f"{t * 1e3 / a.new_tokens:.2f} ms per step of {a.prompts} sequences (prefill included); "
          f"scored again without a cache: log-probabilities differ by at most {worst:.2g}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
