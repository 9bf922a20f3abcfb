"""Requests that share a model and a grammar, each with its own adapter, decoded
several tokens to a step.

    python -m examples.speculative_step [--batch 64] [--drafts 4] [--temperature 0.8]
        [--grammar email]

The model is a table of hidden rows, one for each token, and a projection to
the vocabulary with random weights. What the projection gives without the
adapters drafts a few tokens for each request, the likeliest that the grammar
allows; one projection with them scores all drafts; one ``verify_drafts`` keeps
the ones that the model and the grammar agree to, adds a token, and commits. A
request ends with its end-of-sequence token and then takes no part. Prints one
line of JSON.
"""

from __future__ import annotations

import argparse
import json

import torch

from bpdecode_b200 import tables
from bpdecode_b200.adapters import AdapterBank, check_device, project
from bpdecode_b200.batch import ConstraintBatch
from bpdecode_b200.ops import FsaTensors, advance_state, apply_mask_
from bpdecode_b200.workloads import vocab_config1


def run(batch: int = 64, drafts: int = 4, temperature: float = 0.8, grammar: str = "email",
        max_tokens: int = 24, hidden: int = 512, vocab_size: int = 4096, adapters: int = 8,
        rank: int = 16, seed: int = 0) -> dict:
    """Decode ``batch`` requests; returns their tokens and the steps it took."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device=dev)

    vocab = vocab_config1(seed, vocab_size)
    fsa = FsaTensors.from_arrays(tables.load_dfa(grammar), vocab).to(dev)
    requests = ConstraintBatch(fsa, capacity=batch)
    ids = tuple(range(batch))
    requests.add_many(ids)
    states = torch.full((batch,), fsa.start, dtype=torch.int32, device=dev)

    rows = randn(vocab_size, hidden).bfloat16()
    weight = (randn(vocab_size, hidden) * (4 / hidden**0.5)).bfloat16()
    bank = AdapterBank(hidden, vocab_size, adapters, rank, device=dev)
    for i in range(adapters):
        bank.load(i, randn(rank, hidden) / hidden**0.5, randn(vocab_size, rank), scaling=0.2)
    of_request = torch.arange(batch, device=dev) % (adapters + 1) - 1  # some have none

    last = torch.randint(0, vocab_size, (batch,), generator=g, device=dev)
    live = torch.ones(batch, dtype=torch.bool, device=dev)
    texts: list[list[int]] = [[] for _ in ids]
    steps = 0
    while steps < max_tokens and bool(live.any()):
        line, ahead = [last], states.clone()
        for _ in range(drafts):
            guess = apply_mask_(project(rows[line[-1]], weight), fsa, ahead).argmax(-1)
            line.append(guess)
            ahead = advance_state(fsa, ahead, guess)
        chain = torch.stack(line, 1)  # [batch, drafts + 1]: what each position continues
        logits = project(rows[chain.reshape(-1)], weight, bank,
                         of_request.repeat_interleave(drafts + 1), out_dtype=torch.float32)
        got = requests.verify_drafts(
            ids, logits, chain[:, 1:], torch.rand(batch, drafts, generator=g, device=dev),
            torch.empty(batch, vocab_size, device=dev).exponential_(generator=g),
            draft_lens=torch.where(live, drafts, -1).to(torch.int32), temperature=temperature,
            src_rows=torch.arange(batch, device=dev) * (drafts + 1))
        states = got.states
        steps += 1
        counts = got.counts.tolist()
        for b, (n, tokens) in enumerate(zip(counts, got.tokens.tolist())):
            for t in tokens[:n]:
                if len(texts[b]) < max_tokens and (not texts[b] or texts[b][-1] != vocab.eos_id):
                    texts[b].append(t)
        done = torch.tensor([n == 0 or len(t) >= max_tokens or t[-1] == vocab.eos_id
                             for n, t in zip(counts, texts)], device=dev)
        live &= ~done
        at = (got.counts - 1).clamp(min=0).long()[:, None]
        last = torch.where(live, got.tokens.gather(1, at)[:, 0], last)
    check_device()
    return {"vocab": vocab, "texts": texts, "steps": steps}


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--batch", type=int, default=64)
    p.add_argument("--drafts", type=int, default=4)
    p.add_argument("--temperature", type=float, default=0.8)
    p.add_argument("--grammar", default="email", choices=tables.names("dfa"))
    a = p.parse_args()
    out = run(a.batch, a.drafts, a.temperature, a.grammar)
    vocab = out["vocab"]
    first = b"".join(vocab.token_bytes[t] for t in out["texts"][0] if t != vocab.eos_id)
    print(json.dumps({"requests": a.batch, "steps": out["steps"],
                      "tokens": sum(map(len, out["texts"])),
                      "first": first.decode(errors="replace")}))


if __name__ == "__main__":
    main()
