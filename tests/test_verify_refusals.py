"""What the projection and the draft verification refuse before anything runs:
C entries called with pointers that are never followed, and the Python checks
that come before them. No kernel is launched."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from bpdecode_b200 import _capi

OK, INVALID, CAPACITY = 0, 1, 3
HERE = 4096  # an aligned address that is never followed


def _verify(**fields) -> tuple[int, str]:
    L = _capi.lib()
    a = _capi.VerifyArgs()
    given = dict(src=HERE, src_stride=100, src_total=20, batch=4, vocab_size=100, noise=HERE,
                 noise_stride=100, tokens_out=HERE, counts_out=HERE, logprobs_out=HERE,
                 workspace=HERE, temperature_all=1.0)
    given.update(fields)
    for k, v in given.items():
        setattr(a, k, v)
    return L.bpd_verify_drafts(C.byref(a), None), L.bpd_last_error().decode()


_DRAFTS = dict(max_drafts=2, drafts=HERE, draft_stride=2, uniforms=HERE, uniform_stride=2)
_BITS = dict(allow_bits=HERE, words_stride=4, num_states=3)


@pytest.mark.parametrize("fields, code, words", [
    (dict(src_dtype=9), INVALID, ""),
    (dict(max_drafts=32), CAPACITY, ""),
    (dict(max_drafts=-1), INVALID, "bad sizes"),
    (dict(vocab_size=0), INVALID, "bad sizes"),
    (dict(batch=-1), INVALID, "bad sizes"),
    (dict(src_total=-1), INVALID, "bad sizes"),
    (dict(src=None), INVALID, "null pointer"),
    (dict(tokens_out=None), INVALID, "null pointer"),
    (dict(counts_out=None), INVALID, "null pointer"),
    (dict(logprobs_out=None), INVALID, "null pointer"),
    (dict(workspace=None), INVALID, "null pointer"),
    (dict(workspace=HERE + 8), INVALID, "16-byte"),
    (dict(src_stride=99), INVALID, "row stride"),
    (dict(noise=None), INVALID, "noise"),
    (dict(noise_stride=99), INVALID, "noise"),
    (dict(noise=None, temperature_all=0.0, temperature=HERE), INVALID, "noise"),
    (dict(_DRAFTS, drafts=None), INVALID, "drafts"),
    (dict(_DRAFTS, draft_stride=1), INVALID, "drafts"),
    (dict(_DRAFTS, uniforms=None), INVALID, "uniform"),
    (dict(_DRAFTS, uniform_stride=1), INVALID, "uniform"),
    (dict(_DRAFTS, probs=HERE, probs_stride=99, probs_total=8), INVALID, "draft prob"),
    (dict(_DRAFTS, probs=HERE, probs_stride=100, probs_total=8, probs_dtype=7), INVALID,
     "draft prob"),
    (dict(_BITS, words_stride=3, path=HERE), INVALID, "words_stride"),
    (dict(_BITS, num_states=0, path=HERE), INVALID, "states"),
    (dict(_BITS), INVALID, "state_pool"),
    (dict(_BITS, state_pool=HERE), INVALID, "state_pool"),
    (dict(_BITS, path=HERE, write_back=1), INVALID, "write_back"),
    (dict(write_back=1), INVALID, "write_back"),
    (dict(next_out=HERE), INVALID, "next_out"),
    (dict(_BITS, path=HERE, tok_next=HERE, next_out=HERE), INVALID, "next_out"),
    (dict(batch=0, src=None), OK, ""),  # nothing to do
])
def test_verify_entry(fields: dict, code: int, words: str) -> None:
    rc, message = _verify(**fields)
    assert rc == code and (rc == OK or words in message), (rc, message)


def test_verify_null() -> None:
    assert _capi.lib().bpd_verify_drafts(None, None) == INVALID


_PROJECT = dict(x=HERE, x_stride=64, weight=HERE, weight_stride=64, dtype=1, rows=3,
                in_features=64, out_features=32, a=HERE, b=HERE, scale=HERE, num_adapters=2,
                rank=16, ids=HERE, ids_int64=0, out=HERE, out_dtype=1, out_stride=32,
                workspace=HERE, stream=None)


@pytest.mark.parametrize("fields, code, words", [
    (dict(rows=-1), INVALID, "bad sizes"),
    (dict(in_features=0), INVALID, "bad sizes"),
    (dict(out_features=0), INVALID, "bad sizes"),
    (dict(num_adapters=-1), INVALID, "bad sizes"),
    (dict(dtype=0), INVALID, "dtype"),
    (dict(out_dtype=2), INVALID, "output dtype"),
    (dict(x=None), INVALID, "null pointer"),
    (dict(weight=None), INVALID, "null pointer"),
    (dict(out=None), INVALID, "null pointer"),
    (dict(a=None), INVALID, "null pointer"),
    (dict(b=None), INVALID, "null pointer"),
    (dict(scale=None), INVALID, "null pointer"),
    (dict(workspace=None), INVALID, "null pointer"),
    (dict(in_features=60), INVALID, "multiple of 8"),
    (dict(x=HERE + 2), INVALID, "16-byte"),
    (dict(weight=HERE + 8), INVALID, "16-byte"),
    (dict(x_stride=68), INVALID, "16-byte"),
    (dict(weight_stride=65), INVALID, "16-byte"),
    (dict(x_stride=56), INVALID, "stride"),
    (dict(weight_stride=56), INVALID, "stride"),
    (dict(out_stride=31), INVALID, "stride"),
    (dict(rank=0), INVALID, "rank"),
    (dict(rank=8), INVALID, "rank"),
    (dict(rank=144), INVALID, "rank"),
    (dict(b=HERE + 4), INVALID, "16-byte"),
    (dict(workspace=HERE + 4), INVALID, "16-byte"),
    (dict(num_adapters=(1 << 28) + 1), CAPACITY, ""),
    (dict(rows=0, x=None), OK, ""),  # nothing to do
])
def test_project_entry(fields: dict, code: int, words: str) -> None:
    L = _capi.lib()
    rc = L.bpd_lora_project(*dict(_PROJECT, **fields).values())
    assert rc == code and (rc == OK or words in L.bpd_last_error().decode()), (
        rc, L.bpd_last_error())


def test_sizes() -> None:
    L = _capi.lib()
    assert L.bpd_lora_take_error(None) == INVALID
    assert L.bpd_verify_workspace_bytes(0, 0) >= 0
    # more requests or rows never need less
    for K in (0, 1, 31):
        sizes = [L.bpd_verify_workspace_bytes(b, K) for b in (1, 7, 64, 1024)]
        assert sizes == sorted(sizes) and sizes[0] > 0
    for rank in (16, 128):
        sizes = [L.bpd_lora_workspace_bytes(t, rank, 8, 1) for t in (1, 16, 215, 4096)]
        assert sizes == sorted(sizes) and sizes[0] > 0


def test_adapter_bank_arguments() -> None:
    from bpdecode_b200.adapters import MAX_RANK, AdapterBank

    for bad in (dict(in_features=60), dict(in_features=0), dict(out_features=0),
                dict(max_adapters=0), dict(max_rank=0), dict(max_rank=MAX_RANK + 1)):
        with pytest.raises(ValueError):
            AdapterBank(**{**dict(in_features=64, out_features=40, max_adapters=2, max_rank=8,
                                  device="cpu"), **bad})
    with pytest.raises(RuntimeError, match="dtype"):
        AdapterBank(64, 40, 2, 8, dtype=torch.float32, device="cpu")
    bank = AdapterBank(64, 40, 2, 8, device="cpu")
    a, b = torch.randn(8, 64), torch.randn(40, 8)
    with pytest.raises(IndexError):
        bank.load(2, a, b)
    with pytest.raises(IndexError):
        bank.unload(-1)
    for x, y in ((a[:, :32], b), (a, b[:39]), (a[:7], b), (torch.randn(9, 64), torch.randn(40, 9)),
                 (a[0], b), (a[:0], b[:, :0])):
        with pytest.raises(ValueError):
            bank.load(0, x, y)
    for what in (float("inf"), float("nan")):
        bad_b = b.clone()
        bad_b[3, 1] = what
        with pytest.raises(ValueError, match="infinities"):
            bank.load(0, a, bad_b)
    assert bank.loaded == set()
    bank.load(1, a, b, scaling=0.5)
    assert bank.loaded == {1} and float(bank._scale[1]) == 0.5
    bank.unload(1)
    assert bank.loaded == set() and not bank._a.any() and not bank._b.any()


@pytest.mark.parametrize("rank, max_rank", [(1, 1), (5, 8), (16, 16), (17, 40)])
def test_adapter_bank_layout(rank: int, max_rank: int) -> None:
    """What the kernels read: A padded with zero rows, B as tiles of 128 outputs,
    in blocks of 8 of the rank for each output."""
    from bpdecode_b200.adapters import AdapterBank

    K, N = 24, 300
    bank = AdapterBank(K, N, 2, max_rank, device="cpu")
    bank.load(0, torch.randn(max_rank, K), torch.randn(N, max_rank))  # replaced below
    a, b = torch.randn(rank, K).bfloat16(), torch.randn(N, rank).bfloat16()
    bank.load(0, a, b)
    assert torch.equal(bank._a[0, :rank], a) and not bank._a[0, rank:].any()
    for n, r in ((0, 0), (127, rank - 1), (128, 0), (299, rank - 1), (200, rank // 2)):
        assert bank._b[0, n // 128, r // 8, n % 128, r % 8] == b[n, r]
    full = bank._b[0].transpose(1, 2).reshape(-1, bank.rank_pad)
    assert torch.equal(full[:N, :rank], b)
    assert not full[N:].any() and not full[:, rank:].any()


def test_host_tensors_are_refused() -> None:
    from bpdecode_b200.adapters import project
    from bpdecode_b200.speculative import verify_drafts

    with pytest.raises(RuntimeError, match="CUDA"):
        project(torch.zeros(2, 8).bfloat16(), torch.zeros(4, 8).bfloat16())
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_drafts(torch.zeros(2, 8), noise=torch.ones(2, 8))
