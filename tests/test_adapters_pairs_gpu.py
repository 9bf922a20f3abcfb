"""project where two CTAs share the instructions of a tile: adapters whose rows
are runs of every width, ranks that end in half a step, rows far apart. Inputs
are small whole numbers, so every sum is exact and results are compared as they
are."""

from __future__ import annotations

import os
import re

import pytest
import torch

from conftest import ROOT

BF16, F16 = torch.bfloat16, torch.float16


def test_arrivals_in_another_cta_are_ordered() -> None:
    """What one CTA of a cluster says to another about memory is a release, and
    what the other waits for is an acquire: neither is relaxed."""
    folder = os.path.join(ROOT, "bpdecode_b200", "csrc")
    for name in sorted(os.listdir(folder)):
        with open(os.path.join(folder, name), encoding="utf-8") as f:
            text = f.read()
        assert not re.search(r"mbarrier\.[a-z_.]*\.relaxed", text), name


def _runs(*widths: int) -> torch.Tensor:
    """Runs of 32 rows times each width, an adapter each."""
    return torch.cat([torch.full((32 * w,), i) for i, w in enumerate(widths)])


def _spread(apart: int) -> torch.Tensor:
    """Adapters whose rows stand `apart` rows from each other, with none between."""
    ids = torch.full((256,), -1)
    for i in range(3):
        ids[7 * i::apart] = i
    return ids


PLANS = {"1 2 5": _runs(1, 2, 5), "3 4 1": _runs(3, 4, 1), "7 1": _runs(7, 1), "8": _runs(8),
         "6 2": _runs(6, 2), "every 40th": _spread(40), "every 100th": _spread(100),
         "in turn": torch.arange(256) % 11}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rank", [16, 32, 48, 64, 112, 128])
@pytest.mark.parametrize("plan", PLANS)
def test_every_width_of_an_adapters_rows(plan: str, rank: int, dtype: torch.dtype) -> None:
    from bpdecode_b200.adapters import AdapterBank, project

    K, N = 72, 19201  # 151 tiles of outputs, the last of one output: more than SMs
    ids = PLANS[plan].cuda()
    T, n = len(ids), int(ids.max()) + 1
    g = torch.Generator(device="cuda").manual_seed(rank)

    def whole(*shape: int) -> torch.Tensor:
        return torch.randint(-1, 2, shape, generator=g, device="cuda").to(dtype)

    x, w = whole(T, K), torch.zeros(N, K, dtype=dtype, device="cuda")
    # |S| <= 72, and one of them is a result: exact in any type
    a = whole(n, rank, K)
    at = torch.randint(0, rank, (n, N), generator=g, device="cuda")
    b = torch.zeros(n, N, rank, dtype=dtype, device="cuda").scatter_(2, at[:, :, None], 1.0)
    bank = AdapterBank(K, N, n, rank, dtype=dtype)
    for i in range(n):
        bank.load(i, a[i], b[i])
    want = torch.zeros(T, N, device="cuda")
    for i in range(n):
        mine = (ids == i).nonzero()[:, 0]
        want[mine] = (x[mine].float() @ a[i].float().T)[:, at[i]]
    for _ in range(4):
        assert torch.equal(project(x, w, bank, ids).float(), want)


@pytest.mark.gpu
def test_prompts_give_the_same_bits_each_time() -> None:
    """Whatever else is in the caches, and however the CTAs of a pair are placed."""
    from bpdecode_b200.adapters import AdapterBank, project

    T, K, N, n, rank = 1024, 1024, 8192, 8, 64
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device="cuda").bfloat16()

    x, w = normal(T, K), normal(N, K)
    bank = AdapterBank(K, N, n, rank)
    for i in range(n):
        bank.load(i, normal(rank, K), normal(N, rank), scaling=0.1)
    ids = torch.arange(T, device="cuda") * n // T
    first = project(x, w, bank, ids)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for i in range(30):
        if i % 2:
            flush.fill_(i)
        assert torch.equal(project(x, w, bank, ids), first)
