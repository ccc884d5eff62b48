"""The gradients of lora_tn where a loose bound would hide an error: small inner products, many rows, exact sums, differences,
isolation, graphs and streams.

Tolerances are derived beside each test.
"""
import pytest
import torch

from tests.test_gpu_rows import BACK, BF16, F16, F32, Lora, variants

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


@pytest.mark.parametrize("ab", [BF16, F16])
@pytest.mark.parametrize("m,n,k,rank,adapters,ids", BACK)
def test_gradients_of_integers_are_exact(lib, gpu, m, n, k, rank, adapters, ids, ab):
    # |T| <= 4 k and |U| <= 4 n are exact as two 16-bit numbers of either type; the sums are exact in f32 below 2^24.
    p = Lora(lib, m, n, k, rank, adapters, ab, F32, ids, integers=True)
    for tuning in variants(m):
        p.run(tuning)
        dx, da, db = p.back(tuning=(0 if tuning[0] == 1 else tuning[0], 0))
        want = p.expect(p.dy, p.w.t(), p.b.transpose(1, 2), p.a.transpose(1, 2))[0]
        assert want.abs().max() < 2 ** 22 and torch.equal(dx[:m].double(), want)
        for i in range(adapters):
            r = p.rows(i)
            x, dy = p.x[r].double(), p.dy[r].double()
            for got, low, v in ((da[i], dy @ p.b[i].double(), x), (db[i].t(), x @ p.a[i].double().t(), dy)):
                want = low.t() @ v
                assert (low.abs().t() @ v.abs()).max() < 2 ** 24 if r.numel() else True
                assert torch.equal(got.double(), want)


@pytest.mark.parametrize("ab", [BF16, F16])
@pytest.mark.parametrize("m", [40, 200])
def test_gradients_are_differences_of_the_forward_product(lib, gpu, m, ab):
    # f(X, A, B) = <dY, Y> is linear in each of X, A, B, and with small integers Y and f are exact: so is every difference.
    p = Lora(lib, m, 64, 128, 16, 3, ab, F32, integers=True)
    for tuning in variants(m):
        f = lambda: float((p.dy.double() * p.run(tuning)[:m].double()).sum())
        base = f()
        grads = p.back(tuning=(0 if tuning[0] == 1 else tuning[0], 0))
        gen = torch.Generator().manual_seed(m)
        for t, grad in zip((p.x, p.a, p.b), grads):
            grad = grad[:m, :p.k] if t is p.x else grad
            seen = 0
            for _ in range(12):
                at = tuple(int(torch.randint(0, n, (1,), generator=gen)) for n in t.shape)
                old = t[at].clone()
                t[at] = old + 3
                diff = f() - base
                t[at] = old
                assert diff == 3 * float(grad[at])
                seen += diff != 0
            assert seen >= 6


@pytest.mark.parametrize("m", [3, 100, 128, 1000])
def test_gradients_keep_to_their_adapter(lib, gpu, m):
    # Infinities and NaNs in rows without an adapter and in those of some adapters: the others' gradients have the same bits.
    ids = torch.arange(m) % 5 - 1
    for tuning in variants(m):
        back = (0 if tuning[0] == 1 else tuning[0], 0)
        p = Lora(lib, m, 304, 264, 24, 4, BF16, F32, ids)
        p.run(tuning)
        dx, da, db = p.back(tuning=back)
        q = Lora(lib, m, 304, 264, 24, 4, BF16, F32, ids)
        q.x[::5] = float("nan")
        q.dy[::5] = float("inf")
        q.a[1, :, 0] = float("inf")
        q.b[2] = float("nan")
        q.run(tuning)
        dx2, da2, db2 = q.back(tuning=back)
        for i in (0, 3):
            assert torch.equal(da[i], da2[i]) and torch.equal(db[i], db2[i])
            assert torch.equal(dx[i + 1:m:5], dx2[i + 1:m:5])
        assert torch.equal(da[1], da2[1]) and torch.equal(db[2], db2[2])  # U needs B alone, T needs A alone
        if m >= 5:
            assert not db2[1].isfinite().any() and not da2[2].isfinite().any()


class Step:
    """Forward and backward on buffers of their own, as a training program keeps them."""

    def __init__(self, lib, p):
        self.lib, self.p, d = lib, p, p.desc()
        self.inputs = [t.contiguous().clone() for t in (p.x, p.w, p.a, p.b, p.ids, p.scale, p.dy)]
        self.wt = self.inputs[1].t().contiguous()
        self.y = torch.zeros(p.m, p.n, device="cuda", dtype=p.c)
        self.dx = torch.zeros(p.m, p.k, device="cuda", dtype=p.c)
        self.da, self.db = torch.zeros(p.a.shape, device="cuda"), torch.zeros(p.b.shape, device="cuda")
        self.fwd, self.bwd = p.workspace(lib.lora_workspace(d)), p.workspace(lib.lora_backward_workspace(d))

    def load(self, q):
        """Other values into the same buffers, by kernels on the current stream."""
        for dst, src in zip(self.inputs, (q.x, q.w, q.a, q.b, q.ids, q.scale, q.dy)):
            torch.add(src, 0, out=dst)
        torch.add(q.w.t(), 0, out=self.wt)

    def __call__(self):
        x, w, a, b, ids, scale, dy = (t.data_ptr() for t in self.inputs)
        s, d = torch.cuda.current_stream().cuda_stream, self.p.desc()
        self.lib.lora_tn(d, x, w, a, b, ids, scale, self.y.data_ptr(), self.fwd.data_ptr(), s)
        self.lib.lora_tn_backward(d, x, self.wt.data_ptr(), a, b, ids, scale, dy, self.fwd.data_ptr(), self.dx.data_ptr(),
                                  self.da.data_ptr(), self.db.data_ptr(), self.bwd.data_ptr(), s)

    def results(self):
        return [t.clone() for t in (self.y, self.dx, self.da, self.db)]


STEPS = [(1, 16, BF16), (24, 16, BF16), (24, 72, F16), (100, 32, BF16), (300, 16, F16), (700, 128, BF16)]  # m, rank, operands


def problems(lib, m, rank, ab, count):
    ps = [Lora(lib, m, 520, 264, rank, 6, ab, F32, ids, seed=s) for s, ids in zip(range(count), ["mixed", "packed"] * count)]
    want = []
    for p in ps:
        step = Step(lib, p)
        step()
        torch.cuda.synchronize()
        want.append(step.results())
    return ps, want


@pytest.mark.parametrize("m,rank,ab", STEPS)
def test_a_training_step_captured_and_replayed(lib, gpu, m, rank, ab):
    """Two steps back to back on one workspace in a graph; replays follow the buffers' contents, ids among them."""
    ps, want = problems(lib, m, rank, ab, 4)
    step = Step(lib, ps[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
        step()
    for _ in range(3):
        for p, w in zip(ps, want):
            step.load(p)
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(step.results(), w))


@pytest.mark.parametrize("m,rank,ab", STEPS)
def test_operands_written_just_before_the_call(lib, gpu, m, rank, ab):
    """Kernels that write every operand, then the step, over and over without a wait: what a kernel loads ahead of the one before
    it must be the new values."""
    ps, want = problems(lib, m, rank, ab, 4)
    step = Step(lib, ps[0])
    got = []
    for _ in range(10):
        for p in ps:
            step.load(p)
            step()
            got.append(step.results())
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 4]))


def test_training_steps_on_several_streams_at_once(lib, gpu):
    jobs = []
    for m, rank, ab in STEPS:
        ps, want = problems(lib, m, rank, ab, 1)
        jobs.append((Step(lib, ps[0]), want[0], torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for _ in range(10):
        for (step, _, stream), g in zip(jobs, got):
            with torch.cuda.stream(stream):
                step()
                g.append(step.results())
    torch.cuda.synchronize()
    for (_, want, _), g in zip(jobs, got):
        for r in g:
            assert all(torch.equal(a, b) for a, b in zip(r, want))
    assert lib.device_status() == (0, 0, 0, 0)
