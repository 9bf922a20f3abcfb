"""Verification of drafted tokens under a grammar, and sampling.

A draft model (or a lookup in the text so far) proposes a few tokens for each
request, the target model computes the rows of logits of all of them in one
pass, and :func:`verify_drafts` decides how many to keep, so that the tokens
are distributed as if the target had sampled them one by one under the
request's grammar. All randomness is given: a uniform number for each draft
and a row of exponential noise for each request, so a step can be repeated,
and tested, exactly. Without drafts it samples one token for each request.

:meth:`ConstraintBatch.verify_drafts <bpdecode_b200.batch.ConstraintBatch.verify_drafts>`
and :meth:`CFGConstraintBatch.verify_drafts
<bpdecode_b200.grammar.device.CFGConstraintBatch.verify_drafts>` do the same on
the states that a batch keeps, and commit them.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi
from .ops import _DTYPE_CODE, FsaTensors, _as_i32, _ptr, _require_cuda, _stream, on_device

MAX_DRAFTS = 31  # BPD_MAX_DRAFTS


class VerifyResult(NamedTuple):
    """What :func:`verify_drafts` returns for requests with up to K drafts."""

    tokens: torch.Tensor  # int64 [B, K + 1]: accepted drafts, the token behind them, then -1
    counts: torch.Tensor  # int32 [B]: how many tokens those are
    logprobs: torch.Tensor  # float32 [B, K + 1]: their log-probabilities, then 0
    states: torch.Tensor | None  # int32 [B]: the grammar state behind the last one


def _matrix(t: torch.Tensor, what: str, rows: int, cols: int, dtypes: tuple,
            device: torch.device) -> torch.Tensor:
    if t.dim() != 2 or t.shape[0] < rows or t.shape[1] < cols:
        raise RuntimeError(f"bpdecode_b200: {what} must be [{rows}, {cols}] or larger, got "
                           f"{tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise RuntimeError(f"bpdecode_b200: unsupported {what} dtype {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"bpdecode_b200: {what} must be on {device}")
    if cols and (t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < cols):
        raise RuntimeError(f"bpdecode_b200: {what} needs contiguous columns and rows that do not "
                           f"overlap (strides {t.stride()})")
    return t


def _stride(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.stride(0) if t.shape[0] > 1 else max(int(t.shape[1]), 1)


def _vector(t: torch.Tensor | None, what: str, n: int, dtype: torch.dtype,
            device: torch.device) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype != dtype or t.shape != (n,) or t.device != device:
        raise RuntimeError(f"bpdecode_b200: {what} must be {dtype} [{n}] on {device}")
    return t.contiguous()


def _launch(src, drafts, uniforms, noise, draft_lens, draft_probs, temperature, src_rows,
            prob_rows, batch, vocab, pool, slot_ptr, path, bits, tok_next, num_states,
            states, write_back) -> VerifyResult:
    """Check the arguments that every form shares and enqueue the kernel."""
    _require_cuda(src, "src")
    dev, B, V = src.device, batch, vocab
    _matrix(src, "src", 0, V, tuple(_DTYPE_CODE), dev)
    if drafts is None:
        K = 0
    else:
        if drafts.dim() != 2:
            raise RuntimeError("bpdecode_b200: drafts must be [batch, drafts]")
        K = int(drafts.shape[1])
        _matrix(drafts, "drafts", B, K, (torch.int32, torch.int64), dev)
    if K > MAX_DRAFTS:
        raise RuntimeError(f"bpdecode_b200: at most {MAX_DRAFTS} drafts ({K})")
    src_rows = _vector(src_rows, "src_rows", B, torch.int64, dev)
    if src_rows is None and src.shape[0] < B * (K + 1):
        raise RuntimeError("bpdecode_b200: src has fewer rows than the requests' drafts + 1")
    draft_lens = _vector(draft_lens, "draft_lens", B, torch.int32, dev)
    heat, everywhere = None, 1.0
    if isinstance(temperature, torch.Tensor):
        heat = _vector(temperature, "temperature", B, torch.float32, dev)
    else:
        everywhere = float(temperature)
        if not 0.0 <= everywhere < float("inf"):
            raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    if heat is not None or everywhere > 0.0:
        if noise is None or (uniforms is None and K):
            raise RuntimeError("bpdecode_b200: sampling needs noise, and uniforms for drafts")
    f32 = (torch.float32,)
    if noise is not None:
        _matrix(noise, "noise", B, V, f32, dev)
    if uniforms is not None:
        _matrix(uniforms, "uniforms", B, K, f32, dev)
    if K == 0:
        draft_probs = prob_rows = None
    if draft_probs is not None:
        _matrix(draft_probs, "draft_probs", 0, V, tuple(_DTYPE_CODE), dev)
        prob_rows = _vector(prob_rows, "prob_rows", B, torch.int64, dev)
        if prob_rows is None and draft_probs.shape[0] < B * K:
            raise RuntimeError("bpdecode_b200: draft_probs has fewer rows than the drafts")
    elif prob_rows is not None:
        raise RuntimeError("bpdecode_b200: prob_rows without draft_probs")
    tokens = torch.empty((B, K + 1), dtype=torch.int64, device=dev)
    counts = torch.empty(B, dtype=torch.int32, device=dev)
    logprobs = torch.empty((B, K + 1), dtype=torch.float32, device=dev)
    L = _capi.lib()
    work = torch.empty(L.bpd_verify_workspace_bytes(B, K), dtype=torch.uint8, device=dev)
    with on_device(dev):
        L.check(L.bpd_verify_drafts(
            src.data_ptr(), _DTYPE_CODE[src.dtype], max(_stride(src), V), src.shape[0],
            _ptr(src_rows), _ptr(drafts) if K else None, int(K > 0 and drafts.dtype == torch.int64),
            _stride(drafts), _ptr(draft_lens), _ptr(draft_probs),
            0 if draft_probs is None else _DTYPE_CODE[draft_probs.dtype],
            0 if draft_probs is None else max(_stride(draft_probs), V),
            0 if draft_probs is None else draft_probs.shape[0], _ptr(prob_rows),
            _ptr(uniforms), _stride(uniforms), _ptr(noise),
            0 if noise is None else max(_stride(noise), V), _ptr(heat), everywhere, B, K, V,
            _ptr(pool), slot_ptr, _ptr(path), _ptr(bits), 0 if bits is None else bits.shape[1],
            _ptr(tok_next), num_states, tokens.data_ptr(), counts.data_ptr(),
            logprobs.data_ptr(), _ptr(states), int(write_back),
            work.data_ptr(), _stream(src)))
    return VerifyResult(tokens, counts, logprobs, states)


def verify_drafts(
    src: torch.Tensor,
    drafts: torch.Tensor | None = None,
    uniforms: torch.Tensor | None = None,
    noise: torch.Tensor | None = None,
    *,
    draft_lens: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
    temperature: float | torch.Tensor = 1.0,
    fsa: FsaTensors | None = None,
    states: torch.Tensor | None = None,
    src_rows: torch.Tensor | None = None,
    prob_rows: torch.Tensor | None = None,
) -> VerifyResult:
    """Verify up to K drafted tokens for each of B requests.

    ``src`` [rows, >= vocab] (any float dtype): the target's logits; request b
    has rows ``src_rows[b] ..`` (int64 [B]; b * (K + 1) when None), one for each
    draft and one behind the last. ``drafts`` int32 or int64 [B, K] (None: no
    drafts), of which ``draft_lens[b]`` (int32, None: K) count. ``draft_probs``
    [rows, >= vocab]: the distributions that the drafts were drawn from, request
    b's at rows ``prob_rows[b] ..`` (b * K when None); without it the drafts
    were not drawn (looked up, say). ``uniforms`` float32 [B, >= K] in [0, 1),
    ``noise`` float32 [B, >= vocab] exponential. ``temperature``: one number, or
    float32 [B]; 0 is greedy, and a call with the number 0 needs neither noise
    nor uniforms. ``fsa`` with ``states`` [B]: the grammar, walked along the
    drafts; ``states`` is not modified.

    Draft d is accepted when ``u * q[d] < p[d]``; the first that is not is
    replaced by ``argmax(max(p - q, 0) / noise)``, behind the last one comes
    ``argmax(p / noise)``; equal scores go to the lowest index, NaN logits count
    as -inf. Where nothing is allowed a request ends without a token and its
    state is BROKEN. A request whose length or rows are out of range is idle:
    count 0, state unchanged. Tokens behind an accepted end-of-sequence token
    are the caller's to drop. Launches on torch's current stream without
    synchronising."""
    if (fsa is None) != (states is None):
        raise RuntimeError("bpdecode_b200: fsa and states come together")
    _require_cuda(src, "src")
    if src.dim() != 2:
        raise RuntimeError("bpdecode_b200: src must be [rows, vocab]")
    if states is not None:
        B = int(states.numel())
    elif drafts is not None:
        B = int(drafts.shape[0])
    elif src_rows is not None:
        B = int(src_rows.shape[0])
    else:
        B = int(src.shape[0])
    if drafts is not None and int(drafts.shape[0]) != B:
        raise RuntimeError(f"bpdecode_b200: one row of drafts per request ({drafts.shape[0]} != {B})")
    if fsa is None:
        return _launch(src, drafts, uniforms, noise, draft_lens, draft_probs, temperature,
                       src_rows, prob_rows, B, int(src.shape[1]), None, None, None, None, None,
                       0, None, False)
    tok_next, bits = fsa.dense_tables()
    if fsa.device != src.device:
        raise RuntimeError("bpdecode_b200: src and tables live on different devices")
    st = _as_i32(states, B, fsa.device)
    nxt = torch.empty(B, dtype=torch.int32, device=src.device)
    return _launch(src, drafts, uniforms, noise, draft_lens, draft_probs, temperature, src_rows,
                   prob_rows, B, fsa.vocab_size, st, None, None, bits, tok_next, fsa.num_states,
                   nxt, False)


__all__ = ["MAX_DRAFTS", "VerifyResult", "verify_drafts"]
