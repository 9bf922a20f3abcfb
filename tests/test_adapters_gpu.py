"""project (a shared projection with each row's own low-rank adapter) against
the formula in 64 bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {BF16: 2.0**-8, F16: 2.0**-11, F32: 2.0**-24}


def make(T, K, N, n, r, dtype, seed, ids=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    x, w = normal(T, K), normal(N, K, std=K**-0.5)
    a, b = normal(n, r, K, std=K**-0.5), normal(n, N, r)
    scale = torch.rand(n, generator=g, device="cuda") + 0.5
    if ids is None:
        ids = torch.randint(-1, n, (T,), generator=g, device="cuda")
    return x, w, a, b, scale, ids


def bank_of(a, b, scale, max_rank=None, slots=None):
    from bpdecode_b200.adapters import AdapterBank

    n, r, K = a.shape
    bank = AdapterBank(K, b.shape[1], max_adapters=slots or n, max_rank=max_rank or r,
                       dtype=a.dtype, device="cuda")
    for i in range(n):
        bank.load(i, a[i], b[i], scaling=float(scale[i]))
    return bank


def formula(x, w, a, b, scale, ids):
    """y and a bound on the error of 32-bit sums, both in 64 bits."""
    x, w = x.double(), w.double()
    y, size = x @ w.T, x.abs() @ w.abs().T
    low_size = torch.zeros_like(y)
    for i in range(a.shape[0]):
        mine = (ids == i).nonzero()[:, 0]
        if len(mine):
            s, ai, bi = float(scale[i]), a[i].double(), b[i].double()
            y[mine] += s * (x[mine] @ ai.T @ bi.T)
            low_size[mine] += s * (x[mine].abs() @ ai.abs().T @ bi.abs().T)
    return y, size, low_size


def check(got, x, w, a, b, scale, ids) -> None:
    y, size, low = formula(x, w, a, b, scale, ids)
    K, r = x.shape[1], a.shape[1]
    # sums of K (and K + r) products, each addition off by 2^-23 at most (the matrix unit cuts
    # off); the inner sums are passed on in two 16-bit parts that keep 2^-16 of them
    bound = (UNIT[got.dtype] * y.abs() + K * 2.0**-23 * size + ((K + r) * 2.0**-23 + 2.0**-16) * low
             + (2.0**-24 if got.dtype == F16 or x.dtype == F16 else 0.0) * (1 + r))
    off = (got.double() - y).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((off <= bound * 1.01).all()), float((off / bound.clamp(min=1e-30)).max())


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("T,K,N,n,r", [
    (1, 64, 128, 1, 16), (1, 2048, 4099, 3, 8), (7, 8, 1, 2, 1), (16, 200, 127, 4, 16),
    (17, 512, 129, 20, 5), (33, 1608, 1000, 43, 12), (64, 1024, 2048, 24, 16),
    (130, 264, 515, 7, 40), (257, 512, 640, 9, 64), (300, 136, 384, 300, 16),
    (515, 320, 1030, 5, 128), (1000, 64, 77, 2, 100), (2048, 256, 512, 8, 32)])
def test_against_the_formula(dtype, out, T, K, N, n, r) -> None:
    from bpdecode_b200.adapters import project

    c = make(T, K, N, n, r, dtype, seed=T + K + N)
    got = project(c[0], c[1], bank_of(*c[2:5]), c[5], out_dtype=out)
    assert got.dtype == out and got.shape == (T, N)
    check(got, *c)


@pytest.mark.parametrize("kind", ["none", "all", "one", "runs", "outside", "int32"])
@pytest.mark.parametrize("T", [40, 600])
def test_mixes_of_adapters(kind, T) -> None:
    from bpdecode_b200.adapters import project

    n = 6
    ids = {"none": torch.full((T,), -1), "all": torch.arange(T) % n,
           "one": torch.where(torch.arange(T) == T - 3, 4, -1), "runs": torch.arange(T) * n // T,
           "outside": torch.arange(T) % 9 - 1, "int32": (torch.arange(T) % 7 - 1).int()}[kind]
    c = make(T, 512, 700, n, 16, BF16, seed=T, ids=ids.cuda())
    got = project(c[0], c[1], bank_of(*c[2:5]), c[5], out_dtype=F32)
    check(got, *c)


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("T,K,N,n,r,order", [
    (129, 72, 19201, 3, 16, "mixed"), (140, 264, 19100, 20, 16, "runs"),
    (165, 64, 19072, 9, 40, "mixed"), (215, 200, 19500, 43, 12, "runs"),
    (256, 136, 20000, 24, 16, "mixed"), (257, 328, 9999, 30, 16, "runs"),
    (300, 64, 9730, 6, 128, "mixed"), (321, 128, 9600, 40, 16, "runs"),
    (700, 136, 6500, 50, 16, "mixed"), (1025, 200, 4000, 8, 64, "runs"),
    (33, 136, 9601, 5, 16, "mixed"), (50, 1608, 9733, 43, 12, "runs"),
    (64, 64, 9728, 1, 16, "all"), (65, 320, 10240, 70, 33, "mixed"),
    (100, 520, 19000, 9, 48, "runs"), (128, 8, 9610, 128, 8, "mixed"),
    (200, 200, 9733, 43, 12, "runs"), (256, 768, 9857, 24, 16, "mixed"),
    (290, 136, 6500, 300, 16, "mixed"), (600, 264, 4999, 8, 128, "runs"),
    (1030, 512, 2049, 11, 64, "runs")])
def test_tiles_for_every_sm(dtype, out, T, K, N, n, r, order) -> None:
    """More tiles than SMs, or nearly: large tiles' products are then shared by two CTAs."""
    from bpdecode_b200.adapters import project

    t = torch.arange(T)
    ids = {"mixed": None, "all": torch.zeros(T).long(), "runs": t * (n + 1) // T - 1}[order]
    c = make(T, K, N, n, r, dtype, seed=T + N, ids=ids if ids is None else ids.cuda())
    bank = bank_of(*c[2:5])
    got = project(c[0], c[1], bank, c[5], out_dtype=out)
    check(got, *c)
    assert torch.equal(got, project(c[0], c[1], bank, c[5], out_dtype=out))
    alone = torch.full_like(c[5], -1)
    check(project(c[0], c[1], out_dtype=out), *c[:5], alone)


@pytest.mark.parametrize("T,K,N", [(1, 64, 19000), (16, 200, 38000), (64, 72, 60000),
                                   (100, 136, 37889), (128, 520, 18945)])
def test_one_two_and_more_tiles_for_an_sm(T, K, N) -> None:
    from bpdecode_b200.adapters import project

    c = make(T, K, N, 5, 24, BF16, seed=N)
    bank = bank_of(*c[2:5])
    for out in (BF16, F32):
        got = project(c[0], c[1], bank, c[5], out_dtype=out)
        check(got, *c)


def test_no_bank_is_the_projection_alone() -> None:
    from bpdecode_b200.adapters import project

    c = make(50, 256, 300, 1, 16, F16, seed=1, ids=torch.full((50,), -1, device="cuda"))
    check(project(c[0], c[1]), *c)
    bank = bank_of(*c[2:5])
    assert torch.equal(project(c[0], c[1]), project(c[0], c[1], bank, c[5]))


def test_smaller_ranks_reloading_and_unloading() -> None:
    from bpdecode_b200.adapters import project

    x, w, a, b, scale, ids = make(20, 128, 260, 3, 16, BF16, seed=3)
    bank = bank_of(a, b, scale, max_rank=50, slots=5)
    check(project(x, w, bank, ids, out_dtype=F32), x, w, a, b, scale, ids)
    bank.load(1, a[0, :4], b[0, :, :4], scaling=2.0)  # a smaller rank over a larger one
    bank.unload(2)
    a2, b2, s2 = a.clone(), b.clone(), scale.clone()
    a2[1], b2[1], s2[1] = a[0], b[0], 2.0
    a2[1, 4:] = 0
    s2[2] = 0.0
    check(project(x, w, bank, ids, out_dtype=F32), x, w, a2, b2, s2, ids)
    assert bank.loaded == {0, 1}


def test_one_row_does_not_touch_another() -> None:
    """NaN and infinities in one row's input stay in that row, and a row's result
    does not depend on the rows beside it."""
    from bpdecode_b200.adapters import project

    x, w, a, b, scale, ids = make(48, 256, 384, 4, 16, BF16, seed=6)
    bank = bank_of(a, b, scale)
    ids[7], ids[20] = 1, 2
    clean = project(x, w, bank, ids)
    bad = x.clone()
    bad[7], bad[20, 5] = float("nan"), float("inf")
    got = project(bad, w, bank, ids)
    rest = torch.tensor([t for t in range(48) if t not in (7, 20)], device="cuda")
    assert torch.equal(got[rest], clean[rest])
    assert bool(torch.isnan(got[7]).all()) and not bool(torch.isfinite(got[20]).any())
    again = project(x, w, bank, ids)
    assert torch.equal(again, clean)


def test_strides_and_out() -> None:
    from bpdecode_b200.adapters import project

    x, w, a, b, scale, ids = make(30, 128, 333, 2, 16, BF16, seed=8)
    wide_x = torch.zeros(30, 160, dtype=BF16, device="cuda")
    wide_w = torch.zeros(333, 136, dtype=BF16, device="cuda")
    wide_x[:, 8:136], wide_w[:, :128] = x, w
    out = torch.full((30, 341), 5.0, device="cuda")
    bank = bank_of(a, b, scale)
    got = project(wide_x[:, 8:136], wide_w[:, :128], bank, ids, out=out[:, 3:336])
    assert got.data_ptr() == out[:, 3:].data_ptr()
    check(got, x, w, a, b, scale, ids)
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 336:] == 5).all())
    empty = project(x[:0], w, bank, ids[:0])
    assert empty.shape == (0, 333)


def test_another_stream() -> None:
    from bpdecode_b200.adapters import project

    c = make(70, 512, 900, 5, 16, BF16, seed=10)
    bank = bank_of(*c[2:5])
    one = project(c[0], c[1], bank, c[5])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        two = project(c[0], c[1], bank, c[5])
    side.synchronize()
    assert torch.equal(one, two)


def test_refusals() -> None:
    from bpdecode_b200.adapters import AdapterBank, project

    x, w, a, b, scale, ids = make(12, 64, 96, 2, 16, BF16, seed=2)
    bank = bank_of(a, b, scale)
    flat = torch.zeros(64 * 12 + 8, dtype=BF16, device="cuda")
    for args in ((x.cpu(), w), (x, w.cpu()), (x.float(), w.float()), (x, w.half()),
                 (x[:, :63], w[:, :63]), (x, w[:, :56]), (x[:, ::2], w[:, :32]),
                 (flat[1:769].view(12, 64), w), (x, w, bank), (x, w, None, ids),
                 (x, w[:90], bank, ids), (x, w, bank, ids[:5]), (x, w, bank, ids.float()),
                 (x, w, bank, ids.cpu()), (x, w, None, None, torch.empty(12, 95, device="cuda")),
                 (x, w, None, None, None, F16)):
        with pytest.raises((RuntimeError, ValueError)):
            project(*args)
    bad = b[0].clone()
    bad[3, 1] = float("nan")
    for load in ((2, a[0], b[0]), (-1, a[0], b[0]), (0, a[0], b[0, :, :8]), (0, a[0, :, :8], b[0]),
                 (0, a[0], b[0, :90]), (0, a[0], bad), (0, a[0].repeat(2, 1), b[0].repeat(1, 2))):
        with pytest.raises((ValueError, IndexError)):
            bank.load(*load)
    for size in ((60, 96, 2, 16), (64, 0, 2, 16), (64, 96, 0, 16), (64, 96, 2, 0), (64, 96, 2, 129)):
        with pytest.raises(ValueError):
            AdapterBank(*size)


def test_no_projection_gave_up_waiting() -> None:
    from bpdecode_b200.adapters import AdapterBank, check_device, project

    g = torch.Generator().manual_seed(1)
    x = torch.randn(33, 256, generator=g).bfloat16().cuda()
    w = torch.randn(300, 256, generator=g).bfloat16().cuda()
    bank = AdapterBank(256, 300, 2, 16)
    bank.load(1, torch.randn(16, 256, generator=g), torch.randn(300, 16, generator=g))
    project(x, w, bank, torch.arange(33, device="cuda") % 3)
    check_device()
    check_device()


@pytest.mark.parametrize("T,N,out", [(200, 19500, BF16), (800, 700, BF16), (800, 700, F32),
                                     (1100, 9000, BF16)])
def test_one_row_does_not_touch_another_in_large_tiles(T, N, out) -> None:
    from bpdecode_b200.adapters import project

    x, w, a, b, scale, ids = make(T, 200, N, 5, 40, BF16, seed=T)
    bank = bank_of(a, b, scale)
    bad_rows = [0, 31, 130, T - 1]
    ids[torch.tensor(bad_rows, device="cuda")] = torch.tensor([1, 2, -1, 3], device="cuda")
    clean = project(x, w, bank, ids, out_dtype=out)
    bad = x.clone()
    bad[0], bad[31, 5], bad[130], bad[T - 1, 7] = float("nan"), float("inf"), float("nan"), 3e38
    got = project(bad, w, bank, ids, out_dtype=out)
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[bad_rows] = False
    assert torch.equal(got[rest], clean[rest])
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isnan(got[130]).all())
    assert not bool(torch.isfinite(got[31]).any())


@pytest.mark.parametrize("T,N", [(3, 500), (200, 19500), (800, 700)])
def test_captured_in_a_graph(T, N) -> None:
    from bpdecode_b200.adapters import project

    x, w, a, b, scale, ids = make(T, 136, N, 4, 16, F16, seed=T + 1)
    bank = bank_of(a, b, scale)
    out = torch.empty(T, N, dtype=F16, device="cuda")
    project(x, w, bank, ids, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        project(x, w, bank, ids, out=out)
    for seed in (5, 6):
        y = make(T, 136, N, 4, 16, F16, seed=seed)
        x.copy_(y[0])
        ids.copy_(y[5])
        want = project(x, w, bank, ids)
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
