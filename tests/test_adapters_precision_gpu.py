"""How exact project is. With small whole numbers every sum is exact, so results
are compared as they are: S = A x needs all of its 16-bit parts for that. With
positive numbers a sum that is cut off at every step drifts, which an fp32
result must not show."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
PAIRS = [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


def _ids(T: int, n: int, order: str, g: torch.Generator) -> torch.Tensor:
    if order == "runs":
        return torch.arange(T, device="cuda") * (n + 1) // T - 1
    return torch.randint(-1, n, (T,), generator=g, device="cuda")


def _whole(g: torch.Generator, low: int, high: int, *shape: int) -> torch.Tensor:
    return torch.randint(low, high, shape, generator=g, device="cuda").float()


@pytest.mark.parametrize("dtype,out", PAIRS)
@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("T,K,N,n,rank", [
    (1, 4096, 200, 2, 16), (20, 4104, 130, 3, 16), (64, 2048, 300, 24, 16),
    (129, 4096, 19300, 5, 32), (256, 2048, 700, 6, 48), (300, 2048, 130, 8, 16),
    (300, 4104, 300, 3, 128), (700, 4096, 260, 9, 64), (700, 2048, 130, 40, 16),
    (2000, 4096, 130, 8, 64), (2000, 4104, 260, 7, 112), (5000, 2056, 130, 5, 32)])
def test_whole_numbers_are_exact(T, K, N, n, rank, order, dtype, out) -> None:
    """y = W x + S[j] - S[k] for two ranks of each output. S has up to 16 bits, which
    one part does not hold; sums of all tiles, groups and parts are exact."""
    from bpdecode_b200.adapters import AdapterBank, project

    g = torch.Generator(device="cuda").manual_seed(T + K + rank)
    ids = _ids(T, n, order, g)
    x, w = _whole(g, 0, 16, T, K), _whole(g, 0, 2, N, K)
    w *= _whole(g, 0, 2, N, K)  # a quarter of ones
    a = _whole(g, 0, 2, n, rank, K)  # S is below 16 K <= 65,664 / 1.06
    a[:, :, -8:] = 0
    j, k = (torch.randint(0, rank, (n, N), generator=g, device="cuda") for _ in range(2))
    b = torch.zeros(n, N, rank, device="cuda")
    b.scatter_add_(2, j[:, :, None], torch.ones(n, N, 1, device="cuda"))
    b.scatter_add_(2, k[:, :, None], -torch.ones(n, N, 1, device="cuda"))
    bank = AdapterBank(K, N, n, rank, dtype=dtype)
    for i in range(n):
        bank.load(i, a[i], b[i])
    want = (x.double() @ w.double().T)
    for i in range(n):
        mine = (ids == i).nonzero()[:, 0]
        s = x[mine].double() @ a[i].double().T
        assert not len(mine) or float(s.max()) < 65504
        want[mine] += s[:, j[i]] - s[:, k[i]]
    got = project(x.to(dtype), w.to(dtype), bank, ids, out_dtype=out)
    assert torch.equal(got, want.to(out))


@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("T,K,N,n,rank", [(7, 256, 130, 2, 16), (64, 256, 300, 6, 16),
                                          (200, 248, 19300, 5, 64), (300, 256, 130, 4, 128),
                                          (1500, 256, 260, 8, 48)])
def test_three_parts_of_a_sum_keep_24_bits(T, K, N, n, rank, order) -> None:
    """bf16 to fp32: S of up to 24 bits is all there."""
    from bpdecode_b200.adapters import AdapterBank, project

    g = torch.Generator(device="cuda").manual_seed(T)
    ids = _ids(T, n, order, g)
    x, a = _whole(g, 0, 256, T, K), _whole(g, 0, 256, n, rank, K)  # below 2^24
    j = torch.randint(0, rank, (n, N), generator=g, device="cuda")
    b = torch.zeros(n, N, rank, device="cuda").scatter_(2, j[:, :, None], 1.0)
    bank = AdapterBank(K, N, n, rank, dtype=BF16)
    for i in range(n):
        bank.load(i, a[i], b[i])
    want = torch.zeros(T, N, dtype=torch.float64, device="cuda")
    for i in range(n):
        mine = (ids == i).nonzero()[:, 0]
        want[mine] = (x[mine].double() @ a[i].double().T)[:, j[i]]
    w = torch.zeros(N, K, dtype=BF16, device="cuda")
    got = project(x.to(BF16), w, bank, ids, out_dtype=F32)
    assert torch.equal(got.double(), want)


# A step of 16 inner elements is cut off by at most 2^-23 of the sum so far. A group of 512 has
# 32 of them, whose sums grow evenly where all terms are positive: 2^-23 * 33 / 2 of the group's
# at most. Groups are then added with rounding, 2^-24 each of up to 16 (and parts of a cluster, 8);
# what S passes on loses 2^-22.
DRIFT = 2.0**-23 * 16.5 + 24 * 2.0**-24 + 2.0**-22


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K", [(5, 4096), (64, 8192), (128, 4104), (300, 4096), (700, 8192),
                                 (2500, 4096)])
def test_an_fp32_result_does_not_drift(T: int, K: int, dtype: torch.dtype) -> None:
    from bpdecode_b200.adapters import project

    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.rand(T, K, generator=g, device="cuda").to(dtype)
    w = torch.rand(300, K, generator=g, device="cuda").to(dtype)
    got = project(x, w, out_dtype=F32).double()
    want = x.double() @ w.double().T
    assert float(((got - want).abs() / want).max()) <= DRIFT


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


@pytest.mark.parametrize("T", [9, 200, 700])
@pytest.mark.parametrize("scaling", [1.0, 1e-3, 1e-5])
def test_small_sums_in_fp16_keep_what_its_parts_can_hold(scaling: float, T: int) -> None:
    """Two parts hold 2^-22 of S, and nothing below 2^-25."""
    from bpdecode_b200.adapters import AdapterBank, project

    K, N, rank = 512, 130, 16
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.rand(T, K, generator=g, device="cuda").half()
    a = (torch.rand(rank, K, generator=g, device="cuda") / 256).half()
    j = torch.randint(0, rank, (N,), generator=g, device="cuda")
    b = torch.zeros(N, rank, device="cuda").scatter_(1, j[:, None], 1.0)
    bank = AdapterBank(K, N, 1, rank, dtype=F16)
    bank.load(0, a, b, scaling=scaling)
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    got = project(x, torch.zeros(N, K, dtype=F16, device="cuda"), bank, ids, out_dtype=F32)
    scale = float(torch.tensor(scaling, dtype=F32))
    want = scale * (x.double() @ a.double().T)[:, j]
    assert bool(((got.double() - want).abs() <= DRIFT * want + 2.0**-25).all())


@pytest.mark.parametrize("T", [9, 200, 700])
@pytest.mark.parametrize("out", [F16, F32])
def test_sums_beyond_fp16_stay_in_their_rows(out: torch.dtype, T: int) -> None:
    """S of 65504 and more is no fp16 number: such a row has no finite result where
    its adapter's B is not zero, and no other row notices."""
    from bpdecode_b200.adapters import AdapterBank, project

    K, N, rank = 128, 130, 16
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.rand(T, K, generator=g, device="cuda").half()
    w = torch.rand(N, K, generator=g, device="cuda").half()
    bank = AdapterBank(K, N, 2, rank, dtype=F16)
    for i in range(2):
        bank.load(i, torch.rand(rank, K, generator=g, device="cuda"), torch.ones(N, rank))
    ids = torch.arange(T, dtype=torch.int32, device="cuda") % 3 - 1
    large = x.clone()
    large[4] = 2048.0  # adapter 0: sums of about 130,000
    clean, got = (project(t, w, bank, ids, out_dtype=out) for t in (x, large))
    rest = torch.arange(T, device="cuda") != 4
    assert torch.equal(got[rest], clean[rest])
    assert not bool(torch.isfinite(got[4]).any())
