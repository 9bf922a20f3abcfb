"""Low-rank adapters of many requests beside a projection that they share.

A served batch whose requests carry their own adapter multiplies its hidden
rows with one weight and adds each row's own low-rank part:

    y[t] = W x[t] + scaling_a * B_a (A_a x[t])        a = adapter_ids[t]

:class:`AdapterBank` holds the adapters of one projection in device memory, in
the layout that the kernels read; :func:`project` runs the whole batch in one
pass over the weight, whatever mix of adapters its rows have. Its rows of
logits are what the constrained steps (:class:`~bpdecode_b200.batch.ConstraintBatch`)
and :func:`~bpdecode_b200.speculative.verify_drafts` take. There is no
backward pass: adapters are served here, not trained.
"""

from __future__ import annotations

import ctypes

import torch

from . import _capi
from .ops import _DTYPE_CODE, _require_cuda, _stream, on_device

MAX_RANK = 128  # BPD_LORA_MAX_RANK
_TYPES = (torch.bfloat16, torch.float16)
_TILE = 128  # outputs of one tile of the packed B


class AdapterBank:
    """The adapters of one projection ``[out_features, in_features]``.

    ``max_adapters`` slots of up to ``max_rank`` each, allocated once: every
    slot takes ``ceil(max_rank / 16) * 16 * (in_features + out_features)``
    elements. A slot is filled by :meth:`load` and emptied by :meth:`unload`;
    an empty slot adds nothing. Loads are ordered with the steps by the stream
    they run on.
    """

    def __init__(self, in_features: int, out_features: int, max_adapters: int, max_rank: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda") -> None:
        if dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError(f"bpdecode_b200: unsupported adapter dtype {dtype}")
        if in_features < 1 or in_features % 8 or out_features < 1 or max_adapters < 1:
            raise ValueError("AdapterBank: in_features must be a positive multiple of 8, "
                             "out_features and max_adapters positive")
        if not 1 <= max_rank <= MAX_RANK:
            raise ValueError(f"AdapterBank: max_rank must be in 1..{MAX_RANK}")
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.in_features, self.out_features = in_features, out_features
        self.max_adapters, self.max_rank, self.dtype, self.device = (
            max_adapters, max_rank, dtype, device)
        self.rank_pad = (max_rank + 15) // 16 * 16
        tiles = (out_features + _TILE - 1) // _TILE
        self._a = torch.zeros(max_adapters, self.rank_pad, in_features, dtype=dtype, device=device)
        self._b = torch.zeros(max_adapters, tiles, self.rank_pad // 8, _TILE, 8, dtype=dtype,
                              device=device)
        self._scale = torch.zeros(max_adapters, dtype=torch.float32, device=device)
        self.loaded: set[int] = set()

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.max_adapters:
            raise IndexError(f"AdapterBank: slot {slot} is outside 0..{self.max_adapters - 1}")
        return slot

    def load(self, slot: int, a: torch.Tensor, b: torch.Tensor, scaling: float = 1.0) -> None:
        """Put the adapter ``A = a`` [rank, in_features], ``B = b`` [out_features,
        rank] into ``slot``, replacing what was there. ``b`` must be finite: the
        rows of other adapters pass over it with a factor of zero. (That check
        waits for the device; loading is not part of a step.)"""
        self._slot(slot)
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1]:
            raise ValueError("AdapterBank.load: a is [rank, in_features], b [out_features, rank]")
        r = int(a.shape[0])
        if (int(a.shape[1]), int(b.shape[0])) != (self.in_features, self.out_features):
            raise ValueError(f"AdapterBank.load: the adapter is {tuple(a.shape)}, "
                             f"{tuple(b.shape)}, the projection "
                             f"[{self.out_features}, {self.in_features}]")
        if not 1 <= r <= self.max_rank:
            raise ValueError(f"AdapterBank.load: rank {r} is outside 1..{self.max_rank}")
        a, b = (t.detach().to(device=self.device, dtype=self.dtype) for t in (a, b))
        if not bool(torch.isfinite(b).all()):
            raise ValueError("AdapterBank.load: b has infinities or NaN")
        tiles = self._b.shape[1]
        packed = torch.zeros(tiles * _TILE, self.rank_pad, dtype=self.dtype, device=self.device)
        packed[: self.out_features, :r] = b
        self._b[slot].copy_(packed.view(tiles, _TILE, self.rank_pad // 8, 8).transpose(1, 2))
        self._a[slot, :r].copy_(a)
        self._a[slot, r:].zero_()
        self._scale[slot] = float(scaling)
        self.loaded.add(slot)

    def unload(self, slot: int) -> None:
        """Empty ``slot``: rows that still name it get the shared projection alone."""
        self._slot(slot)
        for t in (self._a, self._b, self._scale):
            t[slot].zero_()
        self.loaded.discard(slot)


def _check_rows(t: torch.Tensor, what: str, cols: int, dtype: torch.dtype) -> int:
    """The row stride of a matrix whose rows start on 16-byte boundaries."""
    stride, step = t.stride()
    if t.shape[0] <= 1:
        stride = (cols + 7) // 8 * 8
    if t.shape[1] != cols or t.dtype != dtype:
        raise RuntimeError(f"bpdecode_b200: {what} must be [rows, {cols}] {dtype}, got "
                           f"{tuple(t.shape)} {t.dtype}")
    if step != 1 or stride < cols or stride % 8 or t.data_ptr() % 16:
        raise RuntimeError(f"bpdecode_b200: {what} needs contiguous columns and rows that start "
                           f"on 16-byte boundaries (strides {t.stride()})")
    return stride


def project(
    x: torch.Tensor,
    weight: torch.Tensor,
    bank: AdapterBank | None = None,
    adapter_ids: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``x @ weight.T`` plus each row's own adapter, in one pass.

    ``x`` [rows, in_features] and ``weight`` [out_features, in_features] are
    bf16 or fp16 (``in_features`` a multiple of 8); ``adapter_ids`` (int32 or
    int64 [rows]) names each row's slot of ``bank``, any id outside the bank
    (such as -1) none. The result [rows, out_features] is of ``x``'s type, or
    fp32 (``out_dtype``), rounded once from fp32 sums; ``out`` receives it
    (contiguous columns, any row stride). In fp16, ``scaling * A x`` must stay
    below 65504, and what is below 2^-25 of it is lost. No autograd graph is
    recorded, whether inputs require gradients or not. With a bank a call takes
    a workspace from torch's allocator: up to ``256 * rank`` bytes for each row
    (384 for fp32 results of bf16), less where the bank has fewer than 64 slots.
    Launches on torch's current stream without synchronising."""
    _require_cuda(x, "x")
    dtype, dev = x.dtype, x.device
    if dtype not in _TYPES:
        raise RuntimeError(f"bpdecode_b200: unsupported dtype {dtype}")
    if weight.device != dev:
        raise RuntimeError("bpdecode_b200: x and weight live on different devices")
    if x.dim() != 2 or weight.dim() != 2:
        raise RuntimeError("bpdecode_b200: x and weight are matrices")
    T, K = x.shape
    N = weight.shape[0]
    if K % 8:
        raise RuntimeError("bpdecode_b200: in_features must be a multiple of 8")
    xs = _check_rows(x, "x", K, dtype)
    ws = _check_rows(weight, "weight", K, dtype)
    if (bank is None) != (adapter_ids is None):
        raise RuntimeError("bpdecode_b200: bank and adapter_ids come together")
    if out is None:
        out = torch.empty(T, N, dtype=out_dtype or dtype, device=dev)
    elif (out.shape != (T, N) or out.device != dev
          or (out_dtype is not None and out.dtype != out_dtype) or (N > 1 and out.stride(1) != 1)
          or (T > 1 and out.stride(0) < N)):
        raise RuntimeError(f"bpdecode_b200: out must be [{T}, {N}] with contiguous columns")
    if out.dtype is not dtype and out.dtype is not torch.float32:
        raise RuntimeError(f"bpdecode_b200: the result is {dtype} or fp32, not {out.dtype}")
    L = _capi.lib()
    a = b = scale = ids_ptr = work_ptr = None
    n = rank = ids64 = 0
    if bank is not None:
        if bank.device != dev or bank.dtype != dtype:
            raise RuntimeError(f"bpdecode_b200: the bank is {bank.dtype} on {bank.device}")
        if (bank.in_features, bank.out_features) != (K, N):
            raise RuntimeError(f"bpdecode_b200: the bank is for [{bank.out_features}, "
                               f"{bank.in_features}], the weight is [{N}, {K}]")
        ids64 = int(adapter_ids.dtype is torch.int64)
        if ((not ids64 and adapter_ids.dtype is not torch.int32) or adapter_ids.shape != (T,)
                or adapter_ids.device != dev):
            raise RuntimeError("bpdecode_b200: adapter_ids must be int32 or int64 [rows] on the "
                               "device")
        adapter_ids = adapter_ids.contiguous()
        ids_ptr = adapter_ids.data_ptr()
        a, b, scale = bank._a.data_ptr(), bank._b.data_ptr(), bank._scale.data_ptr()
        n, rank = bank.max_adapters, bank.rank_pad
        work = torch.empty(L.bpd_lora_workspace_bytes(T, rank, n, _DTYPE_CODE[out.dtype]),
                           dtype=torch.uint8, device=dev)
        work_ptr = work.data_ptr()
    with on_device(dev):
        L.check(L.bpd_lora_project(
            x.data_ptr(), xs, weight.data_ptr(), ws, _DTYPE_CODE[dtype], T, K, N, a, b, scale,
            n, rank, ids_ptr, ids64, out.data_ptr(), _DTYPE_CODE[out.dtype],
            out.stride(0) if T > 1 else max(N, 1), work_ptr, _stream(x)))
    return out


def check_device() -> None:
    """Wait for the current device and raise if a projection on it gave up
    waiting for its own loads since the last call (its result is then not
    complete). The kernels end with that mark, instead of hanging, should the
    device ever misbehave; a step need not ask."""
    error = ctypes.c_int32(0)
    L = _capi.lib()
    L.check(L.bpd_lora_take_error(ctypes.byref(error)))
    if error.value:
        raise RuntimeError("bpdecode_b200: a projection gave up waiting for its loads")


__all__ = ["MAX_RANK", "AdapterBank", "check_device", "project"]
