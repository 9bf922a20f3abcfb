"""verify_drafts and step_sample of the two batches against their parts: the
function on the same states, and masks and commits one token at a time."""

from __future__ import annotations

import pytest
import torch

from conftest import golden_npz, small_dfa, vocab_of
from test_pda_gpu import _dev

pytestmark = pytest.mark.gpu

NEG = float("-inf")
SMALL = golden_npz("small.npz")


def _rows(B, K, V, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    src = (torch.randn(B * (K + 1), V, generator=g) * 3).to(dtype)
    drafts = torch.randint(0, V, (B, K), generator=g)
    uniforms = torch.rand(B, K, generator=g)
    noise = torch.empty(B, V).exponential_(generator=g)
    return [t.cuda() for t in (src, drafts, uniforms, noise)]


def _dense(n: int):
    """A batch of two regular grammars and sequences spread over its slots."""
    from bpdecode_b200.batch import ConstraintBatch
    from bpdecode_b200.ops import FsaTensors

    patterns = list(SMALL["meta/patterns"])
    grammars = [FsaTensors.from_arrays(small_dfa(SMALL, "batch", patterns.index(p)),
                                       vocab_of("batch")).to("cuda")
                for p in ("[01]+", "-?[0-9]+(\\.[0-9]+)?")]
    batch = ConstraintBatch(grammars, capacity=n + 3)
    ids = [f"s{i}" for i in range(n)]
    batch.add_many(["gone"] + ids, [0] + [i % 2 for i in range(n)])
    batch.evict("gone")
    return batch, ids[::-1]


@pytest.mark.parametrize("K", [0, 1, 4])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_dense_batch_commits_what_was_accepted(K: int, temperature: float) -> None:
    from bpdecode_b200.ops import FsaTensors
    from bpdecode_b200.speculative import verify_drafts

    B = 33
    batch, ids = _dense(B)
    V = batch._t.vocab_size
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    S = batch._t.num_states
    both = FsaTensors(trans=zero.repeat(S), accept=zero.repeat(S).to(torch.uint8),
                      live=zero.repeat(S).to(torch.uint8), num_symbols=1, dead=-1,
                      offsets=zero.repeat(V + 1), symbols=zero, eos_id=-1,
                      tok_next=batch._t.tok_next)
    lens = torch.randint(0, K + 1, (B,), generator=torch.Generator().manual_seed(5))
    lens[3] = -1  # takes no part
    lens = lens.to(torch.int32).cuda()
    for step in range(4):
        src, drafts, uniforms, noise = _rows(B, K, V, 10 * step + K)
        first = torch.arange(B, device="cuda") * (K + 1)
        before = batch._state[batch._slots(ids)]
        want = verify_drafts(src, drafts, uniforms, noise, draft_lens=lens, fsa=both,
                             states=before.clone(), temperature=temperature, src_rows=first)
        others = batch._state.clone()
        got = batch.verify_drafts(ids, src, drafts, uniforms, noise, draft_lens=lens,
                                  temperature=temperature, src_rows=first)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(batch._state[batch._slots(ids)], got.states)
        assert int(got.states[3]) == int(before[3]) and int(got.counts[3]) == 0
        others[batch._slots(ids)] = got.states
        assert torch.equal(batch._state, others)  # nobody else moved


def test_dense_batch_samples_a_token_that_commit_takes() -> None:
    batch, ids = _dense(12)
    twin, _ = _dense(12)
    V = batch._t.vocab_size
    for step in range(5):
        src, _, _, noise = _rows(12, 0, V, 70 + step)
        keep = src.clone()
        tokens = batch.step_sample(ids, src, noise, temperature=1.3)
        assert torch.equal(src, keep)
        masked = src.clone()
        twin.apply_mask(ids, masked)
        p = torch.softmax(masked.double() / 1.3, -1)
        assert torch.equal(tokens, (p / noise.double()).argmax(-1))
        assert torch.equal(twin.commit(ids, tokens), batch._state[batch._slots(ids)])


def test_dense_batch_breaks_where_nothing_is_allowed() -> None:
    from bpdecode_b200.batch import BROKEN

    batch, ids = _dense(4)
    src, drafts, uniforms, noise = _rows(4, 2, batch._t.vocab_size, 3)
    src[3:6] = NEG  # the second sequence's rows
    got = batch.verify_drafts(ids, src, drafts, uniforms, noise)
    assert got.tokens[1].tolist() == [-1, -1, -1] and int(got.counts[1]) == 0
    assert int(batch._state[batch._slots(ids)][1]) == BROKEN == int(got.states[1])
    again = batch.verify_drafts(ids, src.nan_to_num(neginf=0.0), drafts, uniforms, noise)
    assert int(again.counts[1]) == 0 and int(again.states[1]) == BROKEN


def _pda_twins(name: str, n: int):
    from bpdecode_b200.grammar.device import CFGConstraintBatch

    g = _dev(name)
    out = []
    for _ in range(2):
        batch = CFGConstraintBatch(g, capacity=n + 2)
        batch.add_many(["gone", *range(n)])
        batch.evict("gone")
        out.append(batch)
    return g, *out, list(range(n))[::-1]


@pytest.mark.parametrize("name", ["paren", "pairs", "xy", "jsonvalue_v4096", "schema_v4096"])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("K", [0, 1, 3])
def test_pda_batch_equals_masks_and_commits(name: str, temperature: float, K: int) -> None:
    from bpdecode_b200.speculative import verify_drafts

    B = 9
    g, batch, twin, ids = _pda_twins(name, B)
    V = g.vocab_size
    slots = batch._slots(ids)
    for step in range(4):
        src, drafts, uniforms, noise = _rows(B, K, V, 100 * step + K)
        lens = torch.full((B,), K, dtype=torch.int32)
        if step:
            lens[0], lens[1] = -1, 0
        # drafts that the grammar allows on every second sequence, and the masked rows on the way
        masked = src.view(B, K + 1, V).clone()
        configs, broken = twin._configs.clone(), twin._broken.clone()
        trail = []
        for i in range(K + 1):
            row = masked[:, i].contiguous()
            twin.apply_mask(ids, row)
            masked[:, i] = row
            trail.append(twin._configs.clone())
            if i < K:
                drafts[::2, i] = row[::2].argmax(-1)
                twin.commit(ids, drafts[:, i].contiguous())
                # off the grammar: a rejected draft, behind which nothing is looked at
        trail = torch.stack(trail)
        twin._configs.copy_(configs)
        twin._broken.copy_(broken)
        want = verify_drafts(masked.view(-1, V), drafts, uniforms, noise, draft_lens=lens.cuda(),
                             temperature=temperature)
        got = batch.verify_drafts(ids, src, drafts, uniforms, noise, draft_lens=lens.cuda(),
                                  temperature=temperature)
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.counts, want.counts)
        # sums of the same terms in another order: V 2^-24 of them at most, far from reached
        assert torch.allclose(got.logprobs, want.logprobs, rtol=0, atol=V * 2.0**-24 + 1e-5)
        # the twin takes the tokens one by one
        for b, sid in enumerate(ids):
            n = int(got.counts[b])
            for t in got.tokens[b, :n].tolist():
                status = twin.commit([sid], torch.tensor([t], device="cuda"))
                assert status.item() == 1
            if lens[b] >= 0 and (n == 0 or int(got.tokens[b, n - 1]) < 0):
                twin._broken[slots[b]] = True
        status = torch.where(twin._broken[slots], -1, 1).to(torch.int32)
        assert torch.equal(got.states, status)
        assert torch.equal(batch._broken, twin._broken)
        assert torch.equal(batch._configs, twin._configs)


def test_pda_batch_samples() -> None:
    g, batch, twin, ids = _pda_twins("jsonvalue_v4096", 6)
    for step in range(4):
        src, _, _, noise = _rows(6, 0, g.vocab_size, 40 + step, torch.bfloat16)
        tokens = batch.step_sample(ids, src, noise)
        masked = src.clone()
        twin.apply_mask(ids, masked)
        p = torch.softmax(masked.double(), -1)
        assert torch.equal(tokens, (p / noise.double()).argmax(-1))
        twin.commit(ids, tokens)
        assert torch.equal(batch._configs, twin._configs)


def test_refusals() -> None:
    batch, ids = _dense(4)
    _, pda, _, pids = _pda_twins("xy", 4)
    for b, i, V in ((batch, ids, batch._t.vocab_size), (pda, pids, pda.g.vocab_size)):
        src, drafts, uniforms, noise = _rows(4, 2, V, 1)
        with pytest.raises(RuntimeError, match="one row of drafts"):
            b.verify_drafts(i, src, drafts[:3], uniforms, noise)
        with pytest.raises(RuntimeError, match="fewer rows"):
            b.verify_drafts(i, src[:-1], drafts, uniforms, noise)
        with pytest.raises(RuntimeError, match="must be on"):
            b.verify_drafts(i, src.cpu(), drafts, uniforms, noise)
        with pytest.raises(RuntimeError, match="noise"):
            b.step_sample(i, src, noise.double())
        with pytest.raises(KeyError):
            b.verify_drafts(["nobody"], src, drafts, uniforms, noise)


def test_dense_step_captured_in_a_graph() -> None:
    batch, ids = _dense(20)
    twin, _ = _dense(20)
    ids = tuple(ids)
    src, drafts, uniforms, noise = _rows(20, 3, batch._t.vocab_size, 11)
    twin.verify_drafts(ids, src, drafts, uniforms, noise)  # loads the kernels
    batch._slots(ids)  # the slots are on the device
    twin.reset_many(ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = batch.verify_drafts(ids, src, drafts, uniforms, noise)
    for step in range(4):
        for t, new in zip((src, drafts, uniforms, noise),
                          _rows(20, 3, batch._t.vocab_size, 20 + step)):
            t.copy_(new)
        graph.replay()
        want = twin.verify_drafts(ids, src, drafts, uniforms, noise)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(batch._state, twin._state)
