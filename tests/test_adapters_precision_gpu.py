"""How exact project is. With positive numbers a sum that is cut off at every step
drifts, which an fp32 result must not show."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# A step of 16 inner elements is cut off by at most 2^-23 of the sum so far. A group of 512 has
# 32 of them, whose sums grow evenly where all terms are positive: 2^-23 * 33 / 2 of the group's
# at most. Groups are then added with rounding, 2^-24 each of up to 16 (and parts of a cluster, 8);
# what S passes on loses 2^-22.
DRIFT = 2.0**-23 * 16.5 + 24 * 2.0**-24 + 2.0**-22


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K", [(5, 4096), (64, 8192), (300, 4096), (700, 8192), (2500, 8192),
                                 (12000, 4096)])
def test_an_fp32_results_adapters_do_not_drift(T: int, K: int, dtype: torch.dtype) -> None:
    """y = S[j] alone, where the rows leave few CTAs for each and where they leave many."""
    from bpdecode_b200.adapters import AdapterBank, project

    n, rank, N = 3, 16, 130
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.rand(T, K, generator=g, device="cuda").to(dtype)
    a = torch.rand(n, rank, K, generator=g, device="cuda").to(dtype)
    j = torch.randint(0, rank, (n, N), generator=g, device="cuda")
    b = torch.zeros(n, N, rank, device="cuda").scatter_(2, j[:, :, None], 1.0)
    bank = AdapterBank(K, N, n, rank, dtype=dtype)
    for i in range(n):
        bank.load(i, a[i], b[i])
    ids = torch.arange(T, device="cuda") % n
    got = project(x, torch.zeros(N, K, dtype=dtype, device="cuda"), bank, ids, out_dtype=F32)
    for i in range(n):
        want = (x[ids == i].double() @ a[i].double().T)[:, j[i]]
        assert float(((got[ids == i].double() - want).abs() / want).max()) <= DRIFT
