"""The gradients of lora_tn where a loose bound would hide an error: small inner products, many rows, exact sums.

Tolerances are derived beside each test.
"""
import pytest
import torch

from tests.test_gpu_rows import BF16, F16, F32, Lora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e3, 1.0, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("rank", [8, 24, 64, 128])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_f16_gradients_of_small_inner_products(lib, gpu, m, rank, size):
    """Every row has an adapter of its own, and each of its inner products is a single product of two f16 numbers, so that U
    and T are exact in f32 and dA = U x^T, dB = dY T^T are products of two numbers.  What is left is how U and T are carried:
    22 bits, half a step 2^-22, down to 2^-14 and 2^-36 below (half the smallest step of a remainder times 2^11); the two
    products' sum in f32 adds 2 steps of 2^-23, the scaling back none."""
    n, k = 136, 264
    p = Lora(lib, m, n, k, rank, m, F16, F32, torch.arange(m))
    p.scale.fill_(1.0)
    part = size ** 0.5
    one = lambda *s: torch.where(torch.rand(*s, device="cuda", generator=p.gen) < 0.5, -1.0, 1.0) * (torch.rand(*s, device="cuda", generator=p.gen) + 0.5)
    p.a.zero_()
    p.b.zero_()
    j = torch.arange(rank, device="cuda")
    p.a[:, j, j * 2] = (one(m, rank) * part).to(F16)
    p.b[:, j, j] = (one(m, rank) * part).to(F16)
    p.x.copy_((one(m, k) * part).to(F16))
    p.dy.copy_((one(m, n) * part).to(F16))
    for tuning in [(0, 0), (2, 0)] + ([(1, 0)] if m <= 128 else []):
        p.run(tuning)
        _, da, db = p.back()
        x, dy = p.x.double(), p.dy.double()
        t = torch.einsum("irk,ik->ir", p.a.double(), x)
        u = torch.einsum("inr,in->ir", p.b.double(), dy)
        assert torch.equal(t, t.float().double()) and torch.equal(u, u.float().double())
        carried = lambda v: v.abs() * 2.0 ** -22 + 2.0 ** -36
        for name, got, low, v in (("dA", da, u, x), ("dB", db.transpose(1, 2), t, dy)):
            want = low[:, :, None] * v[:, None, :]
            bound = carried(low)[:, :, None] * v.abs()[:, None, :] + want.abs() * 2.0 ** -22
            off = (got.double() - want).abs()
            assert (off <= bound).all(), f"{name} off by {(off / bound).max():.3g} of the bound"


@pytest.mark.parametrize("rank", [16, 24, 64, 128])
@pytest.mark.parametrize("m,adapters,share", [(262144, 1, 1.0), (131072, 16, 0.9)])
def test_gradients_of_long_row_lists(lib, gpu, m, adapters, share, rank):
    """All operands are small integers of one sign, U and T exact as their two numbers, and the sum over any 4096 rows of
    an adapter stays below 2^24, where f32 is exact (asserted below), while the sum over all of them passes it.  Sums of 4096
    rows can thus be taken in one accumulator, and adding them up in f32 costs half a step, 2^-24 of the total, per
    addition that is added on: m / 4096 of them, and within 4096 rows up to 8 CTAs, 4 accumulators and 2 numbers."""
    n, k = 256, 64
    ids = torch.zeros(m, dtype=torch.int64)
    if adapters > 1:
        gen = torch.Generator().manual_seed(rank)
        ids = torch.where(torch.rand(m, generator=gen) < share, 3, torch.randint(0, adapters, (m,), generator=gen))
    p = Lora(lib, m, n, k, rank, adapters, BF16, BF16, ids)
    draw = lambda t, lo, hi: t.copy_(torch.randint(lo, hi, t.shape, device="cuda", generator=p.gen))
    p.scale.fill_(1.0)
    draw(p.x, 0, 65)
    draw(p.dy, 0, 2)
    draw(p.a, 0, 4)
    draw(p.b, 0, 2)
    p.run()
    _, da, db = p.back()
    allowed = (m / 4096 + 8 + 4 + 2) * 2.0 ** -24
    past = False
    for i in range(adapters):
        r = p.rows(i)
        x, dy = p.x[r].double(), p.dy[r].double()
        t, u = x @ p.a[i].double().t(), dy @ p.b[i].double()
        assert u.max() <= 256 and t.max() < 2 ** 16
        for name, got, low, v in (("dA", da[i], u, x), ("dB", db[i].t(), t, dy)):
            for piece in range(0, r.numel(), 4096):
                assert (low[piece:piece + 4096].t() @ v[piece:piece + 4096]).max() < 2 ** 24
            want = low.t() @ v
            past |= bool(want.max() > 2 ** 25)
            off = (got.double() - want).abs()
            assert (off <= allowed * want).all(), f"{name}[{i}] off by {(off / want).max():.3g}, {allowed:.3g} allowed"
    assert past
