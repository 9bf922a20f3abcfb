"""The example of a whole step runs, and its texts are in the grammar."""

from __future__ import annotations

import os
import re
import runpy

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafts", [0, 3])
@pytest.mark.parametrize("grammar", ["ipv4", "email", "float"])
def test_texts_are_in_the_grammar(grammar: str, drafts: int) -> None:
    from bpdecode_b200.workloads import DENSE_PATTERNS

    run = runpy.run_path(os.path.join(ROOT, "examples", "speculative_step.py"))["run"]
    out = run(batch=20, drafts=drafts, temperature=0.7, grammar=grammar)
    vocab = out["vocab"]
    ended = 0
    for tokens in out["texts"]:
        text = b"".join(vocab.token_bytes[t] for t in tokens if t != vocab.eos_id).decode()
        if tokens and tokens[-1] == vocab.eos_id:
            ended += 1
            assert re.fullmatch(dict(DENSE_PATTERNS)[grammar], text), text
    assert grammar != "ipv4" or ended >= 3  # the only one that has an end


def test_greedy_text_does_not_depend_on_the_drafts() -> None:
    """A draft is kept where it is the token that would have come anyway."""
    run = runpy.run_path(os.path.join(ROOT, "examples", "speculative_step.py"))["run"]
    alone, drafted = (run(batch=12, drafts=k, temperature=0.0) for k in (0, 2))
    assert alone["texts"] == drafted["texts"]
    assert drafted["steps"] < alone["steps"]
