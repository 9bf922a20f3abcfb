"""verify_drafts where many tokens are equally likely, or nearly: the noise alone
decides, at any temperature and any size of the logits."""

from __future__ import annotations

import math

import pytest
import torch

from test_speculative_gpu import BF16, F16, F32, check, make, plain, run

pytestmark = pytest.mark.gpu

# where the tied tokens stand: in a vector of one thread, in vectors of one thread, in a
# warp, and in several
PLACES = {"a vector": [0, 1, 2, 3], "a thread": [0, 256, 512, 768], "a warp": [0, 8, 40, 88],
          "warps": [0, 1024, 3072, 5120]}


def _ties(B, V, dtype, place, near, seed, top=20.0, low=-30.0):
    """Rows of four tokens at `top` and the rest far below; their noise is drawn, or
    (near) 0.3 and steps of 2^-15 of it."""
    c = make(B, 0, V, dtype, seed=seed, heats="one")
    g = torch.Generator().manual_seed(seed + 1)
    c["src"][:] = low
    at = torch.tensor(PLACES[place])[None, :] + torch.randint(0, V - 5200, (B, 1), generator=g)
    c["src"].scatter_(1, at, top)
    if near:
        order = torch.rand(B, 4, generator=g).argsort(1)
        c["noise"].scatter_(1, at, 0.3 * (1.0 + order.float() * 2.0**-15))
    return c


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("heat", [1.0, 0.05, 0.01, 1e-3, 1e-4, 1e-5, 1e-6])
def test_ties_at_low_temperatures(heat: float, place: str, near: bool) -> None:
    for dtype, V in ((BF16, 8192), (F32, 8195)):
        c = _ties(150, V, dtype, place, near, seed=int(-math.log10(heat)) + 3)
        c["heats"] = torch.full((150,), heat)
        run(c)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("offset", [3e3, 1e6, -1e6, 1e9])
def test_ties_of_large_logits(offset: float, place: str) -> None:
    c = _ties(150, 8192, F32, place, True, seed=7, top=offset, low=offset - abs(offset) / 64)
    run(c)


def test_tokens_nearly_as_likely_at_low_temperatures() -> None:
    """Logits that differ, by less than the temperature."""
    for heat in (0.05, 1e-3, 1e-5):
        c = make(200, 0, 9001, F32, seed=17, heats="one")
        c["src"] = 20.0 + c["src"].clamp(-8, 8) * (heat / 2)
        c["heats"] = torch.full((200,), heat)
        got = run_tokens(c)
        # fp32 arithmetic has p to 2^-20 or so here (an argument of up to 8 rounded three
        # times, 2^-21, and the exponential): the token is the best up to that
        z = (c["src"].double() - c["src"].double().max(1, keepdim=True).values)
        score = torch.exp(z / c["heats"].double()[:, None]) / c["noise"].double()
        mine = score.gather(1, got.tokens[:, :1].cpu())[:, 0]
        assert bool((mine >= score.max(1).values * (1 - 2.0**-18)).all())


def run_tokens(c, **more):
    from bpdecode_b200.speculative import verify_drafts

    return verify_drafts(
        c["src"].cuda(), c["drafts"].cuda() if c["drafts"].shape[1] else None,
        c["uniforms"].cuda() if c["drafts"].shape[1] else None, c["noise"].cuda(),
        draft_probs=None if c["probs"] is None else c["probs"].cuda(),
        temperature=c["heats"].cuda(), **more)


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("heat", [1e-8, 1e-9, 1e-20, 1e-36])
def test_ties_at_the_lowest_temperatures(heat: float, place: str) -> None:
    """The logits over the temperature have no room for their differences, or none at all."""
    for dtype, V in ((BF16, 8192), (F32, 8195)):
        c = _ties(150, V, dtype, place, True, seed=int(-math.log10(heat)) + 3)
        c["heats"] = torch.full((150,), heat)
        run(c)


@pytest.mark.parametrize("heat", [1.0, 0.1, 1e-3])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("V", [1024, 1003])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_of_one_value(dtype, V: int, given: bool, heat: float) -> None:
    """The lowest value of a type stands for what is masked in many programs; where
    a row has nothing else all of its tokens are equally likely, and so at the
    highest. Behind the last draft, and in place of a refused one."""
    info = torch.finfo(dtype)
    for value in (info.min, info.max, 0.0, -5.0):
        c = make(6, 1, V, dtype, seed=V, ragged=False, heats="one", probs=F32 if given else None)
        c["src"][:] = value
        c["heats"] = torch.full((6,), heat)
        c["uniforms"] = torch.tensor([0.0, 0.0, 0.0, 1.0, 1.0, 1.0])[:, None] * (1 - 2.0**-24)
        got, _ = run(c)
        assert bool((got.counts >= 1).all())


def test_rows_of_the_lowest_value_under_a_grammar() -> None:
    from test_speculative_gpu import tables

    V = 2000
    fsa, tn = tables(6, V, seed=3)
    states = torch.arange(12, dtype=torch.int32) % 6
    for dtype in (F32, BF16):
        c = make(12, 2, V, dtype, seed=5, heats="one")
        c["src"][:] = torch.finfo(dtype).min
        got, _ = run(c, fsa, tn, states)
        assert bool((got.counts >= 1).all())


def test_temperatures_that_take_the_logits_out_of_range() -> None:
    for heat in (1e-37, 1e-38, 2.0**-140):
        c = make(8, 1, 1024, F32, seed=1, ragged=False, heats="one")
        c["src"][:] = torch.where(c["src"] > 4.0, 50.0, c["src"])
        c["heats"] = torch.full((8,), heat)
        got, _ = run(c)
        assert bool((got.counts >= 1).all())


def test_ties_are_decided_alike_each_time() -> None:
    case = _ties(150, 8192, BF16, "warps", True, seed=4)
    case["heats"] = torch.full((150,), 0.01)
    first = run_tokens(case)
    for _ in range(40):
        again = run_tokens(case)
        assert torch.equal(first.tokens, again.tokens)
        assert torch.equal(first.logprobs, again.logprobs)


def test_token_does_not_depend_on_its_place_in_the_batch() -> None:
    """Rows with ties alone and beside others, which splits them otherwise."""
    c = _ties(300, 30000, BF16, "warps", True, seed=6)
    c["heats"] = torch.full((300,), 1e-4)
    whole = run_tokens(c)
    check(whole, plain(c["src"], c["drafts"], c["uniforms"], c["noise"], c["lens"], None,
                       c["heats"], None, None, c["first"], c["pfirst"]))
    for b in (0, 17, 299):
        one = {**c, "src": c["src"][b:b + 1], "noise": c["noise"][b:b + 1],
               "drafts": c["drafts"][b:b + 1], "heats": c["heats"][b:b + 1]}
        assert torch.equal(run_tokens(one).tokens[0], whole.tokens[b])


def _close(B: int, V: int, seed: int):
    """Refused drafts whose probabilities are those of the target but for a thousandth,
    and noise that makes what is left of all tokens nearly equal in the race."""
    c = make(B, 1, V, F32, seed=seed, ragged=False, heats="one", probs=F32, scale=1.0)
    g = torch.Generator().manual_seed(seed)
    p = torch.softmax(c["src"][0::2].double(), -1)
    gap = torch.rand(B, V, generator=g, dtype=torch.float64) * 2e-3 - 1e-3
    c["probs"] = (p * (1 + gap)).float()
    c["drafts"] = gap.argmax(1, keepdim=True)
    c["uniforms"][:] = 1.0 - 2.0**-24
    left = (p - c["probs"].double()).clamp(min=0)
    jitter = 1 + 1e-4 * torch.rand(B, V, generator=g, dtype=torch.float64)
    c["noise"] = torch.where(left > 0, left / left.max() * jitter, 1.0).float().clamp(min=1e-12)
    return c, p, left


def test_refused_drafts_of_nearly_the_targets_probability() -> None:
    c, p, left = _close(40, 20000, seed=2)
    got = run_tokens(c)
    assert bool((got.counts == 1).all())
    # p in fp32: an argument of up to 10 rounded once, an exponential, the sum and a quotient,
    # 2^-20 of it together at most; the token is the best up to what that does to p - q
    slop = p * 2.0**-20
    noise = c["noise"].double()
    sure = ((left - slop) / noise).max(1).values
    mine = ((left + slop) / noise).gather(1, got.tokens[:, :1].cpu())[:, 0]
    assert bool((mine >= sure).all())


def test_refused_drafts_are_replaced_alike_each_time() -> None:
    c, _, _ = _close(64, 32000, seed=9)
    first = run_tokens(c)
    for _ in range(40):
        again = run_tokens(c)
        assert torch.equal(first.tokens, again.tokens)
        assert torch.equal(first.logprobs, again.logprobs)
