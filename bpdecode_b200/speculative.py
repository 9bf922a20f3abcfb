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

import ctypes
import struct
from typing import NamedTuple

import torch

from . import _capi
from .ops import _DTYPE_CODE, FsaTensors, _as_i32, _require_cuda, _stream, on_device

MAX_DRAFTS = 31  # BPD_MAX_DRAFTS

_FLOATS = tuple(_DTYPE_CODE)
_INTS = (torch.int32, torch.int64)
_F32 = (torch.float32,)
_INF = float("inf")


class VerifyResult(NamedTuple):
    """What :func:`verify_drafts` returns for requests with up to K drafts."""

    tokens: torch.Tensor  # int64 [B, K + 1]: accepted drafts, the token behind them, then -1
    counts: torch.Tensor  # int32 [B]: how many tokens those are
    logprobs: torch.Tensor  # float32 [B, K + 1]: their log-probabilities, then 0
    states: torch.Tensor | None  # int32 [B]: the grammar state behind the last one


_ARGS = struct.Struct("=26q9if")  # bpd_verify_args: 26 pointers and strides, then the rest
assert _ARGS.size == ctypes.sizeof(_capi.VerifyArgs)


def _bad(what: str, why: str, t: torch.Tensor) -> RuntimeError:
    return RuntimeError(f"bpdecode_b200: {what} {why}, got {tuple(t.shape)} {t.dtype} on "
                        f"{t.device}, strides {t.stride()}")


def _matrix(t: torch.Tensor, what: str, rows: int, cols: int, dtypes: tuple,
            device: torch.device) -> tuple[int, int]:
    """(pointer, row stride) of a matrix of at least [rows, cols]."""
    if t.dim() != 2:
        raise _bad(what, f"must be [{rows}, {cols}] or larger", t)
    (have, width), (stride, step) = t.shape, t.stride()
    if have < rows or width < cols:
        raise _bad(what, f"must be [{rows}, {cols}] or larger", t)
    if t.dtype not in dtypes or t.device != device:
        raise _bad(what, f"must be one of {dtypes} on {device}", t)
    if have <= 1:
        stride = max(width, 1)
    if cols and (step != 1 and width > 1 or stride < cols):
        raise _bad(what, "needs contiguous columns and rows that do not overlap", t)
    return t.data_ptr(), stride


def _vector(t: torch.Tensor, what: str, n: int, dtype: torch.dtype,
            device: torch.device) -> torch.Tensor:
    if t.dtype != dtype or t.shape != (n,) or t.device != device:
        raise _bad(what, f"must be {dtype} [{n}] on {device}", t)
    return t.contiguous()


def _launch(src, drafts, uniforms, noise, draft_lens, draft_probs, temperature, src_rows,
            prob_rows, batch, vocab, pool, slot_ptr, path, bits, tok_next, num_states,
            states, write_back) -> VerifyResult:
    """Check the arguments that every form shares and enqueue the kernels."""
    dev, B, V = src.device, batch, vocab
    src_ptr, src_stride = _matrix(src, "src", 0, V, _FLOATS, dev)
    K = draft_ptr = draft_stride = drafts64 = 0
    if drafts is not None:
        if drafts.dim() != 2:
            raise RuntimeError("bpdecode_b200: drafts must be [batch, drafts]")
        K = drafts.shape[1]
        draft_ptr, draft_stride = _matrix(drafts, "drafts", B, K, _INTS, dev)
        drafts64 = int(drafts.dtype is torch.int64)
        if K > MAX_DRAFTS:
            raise RuntimeError(f"bpdecode_b200: at most {MAX_DRAFTS} drafts ({K})")
    rows_ptr = lens_ptr = heat_ptr = prows_ptr = 0
    if src_rows is not None:
        src_rows = _vector(src_rows, "src_rows", B, torch.int64, dev)
        rows_ptr = src_rows.data_ptr()
    elif src.shape[0] < B * (K + 1):
        raise RuntimeError("bpdecode_b200: src has fewer rows than the requests' drafts + 1")
    if draft_lens is not None:
        draft_lens = _vector(draft_lens, "draft_lens", B, torch.int32, dev)
        lens_ptr = draft_lens.data_ptr()
    everywhere = 1.0
    if isinstance(temperature, torch.Tensor):
        temperature = _vector(temperature, "temperature", B, torch.float32, dev)
        heat_ptr = temperature.data_ptr()
    else:
        everywhere = float(temperature)
        if not 0.0 <= everywhere < _INF:
            raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    if (heat_ptr or everywhere > 0.0) and (noise is None or (uniforms is None and K)):
        raise RuntimeError("bpdecode_b200: sampling needs noise, and uniforms for drafts")
    noise_ptr = noise_stride = uni_ptr = uni_stride = 0
    if noise is not None:
        noise_ptr, noise_stride = _matrix(noise, "noise", B, V, _F32, dev)
    if uniforms is not None:
        uni_ptr, uni_stride = _matrix(uniforms, "uniforms", B, K, _F32, dev)
    probs_ptr = probs_stride = probs_rows = probs_code = 0
    if draft_probs is not None:
        probs_ptr, probs_stride = _matrix(draft_probs, "draft_probs", 0, V, _FLOATS, dev)
        probs_rows, probs_code = draft_probs.shape[0], _DTYPE_CODE[draft_probs.dtype]
        if prob_rows is not None:
            prob_rows = _vector(prob_rows, "prob_rows", B, torch.int64, dev)
            prows_ptr = prob_rows.data_ptr()
        elif probs_rows < B * K:
            raise RuntimeError("bpdecode_b200: draft_probs has fewer rows than the drafts")
    elif prob_rows is not None:
        raise RuntimeError("bpdecode_b200: prob_rows without draft_probs")
    # sizes one by one: a tuple of them costs a microsecond more
    tokens = torch.empty(B, K + 1, dtype=torch.int64, device=dev)
    counts = torch.empty(B, dtype=torch.int32, device=dev)
    logprobs = torch.empty(B, K + 1, dtype=torch.float32, device=dev)
    L = _capi.lib()
    work = torch.empty(L.bpd_verify_workspace_bytes(B, K), dtype=torch.uint8, device=dev)
    args = _ARGS.pack(
        src_ptr, src_stride, src.shape[0], rows_ptr, draft_ptr, draft_stride, lens_ptr, probs_ptr,
        probs_stride, probs_rows, prows_ptr, uni_ptr, uni_stride, noise_ptr, noise_stride,
        heat_ptr, 0 if pool is None else pool.data_ptr(), slot_ptr or 0,
        0 if path is None else path.data_ptr(), 0 if bits is None else bits.data_ptr(),
        0 if tok_next is None else tok_next.data_ptr(), tokens.data_ptr(), counts.data_ptr(),
        logprobs.data_ptr(), 0 if states is None else states.data_ptr(), work.data_ptr(),
        _DTYPE_CODE[src.dtype], drafts64, probs_code, B, K, V,
        0 if bits is None else bits.shape[1], num_states, write_back, everywhere)
    with on_device(dev):
        L.check(L.bpd_verify_drafts(args, _stream(src)))
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
        B = states.numel()
    elif drafts is not None:
        B = drafts.shape[0]
    elif src_rows is not None:
        B = src_rows.shape[0]
    else:
        B = src.shape[0]
    if drafts is not None and drafts.shape[0] != B:
        raise RuntimeError(f"bpdecode_b200: one row of drafts per request ({drafts.shape[0]} != {B})")
    if fsa is None:
        return _launch(src, drafts, uniforms, noise, draft_lens, draft_probs, temperature,
                       src_rows, prob_rows, B, src.shape[1], None, None, None, None, None,
                       0, None, False)
    tok_next, bits = fsa.dense_tables()
    if fsa.device != src.device:
        raise RuntimeError("bpdecode_b200: src and tables live on different devices")
    st = states
    if (st.dtype is not torch.int32 or st.dim() != 1 or not st.is_contiguous()
            or st.device != src.device):
        st = _as_i32(states, B, fsa.device)
    nxt = torch.empty(B, dtype=torch.int32, device=src.device)
    return _launch(src, drafts, uniforms, noise, draft_lens, draft_probs, temperature, src_rows,
                   prob_rows, B, fsa.vocab_size, st, None, None, bits, tok_next, fsa.num_states,
                   nxt, False)


__all__ = ["MAX_DRAFTS", "VerifyResult", "verify_drafts"]
