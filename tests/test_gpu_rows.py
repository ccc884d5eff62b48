"""The products whose weights are chosen row by row (lora_tn, lora_tn_backward, moe_tn) against their definitions in 64 bits.

Tolerances, from the operators' arithmetic (every bound is per element):
* a sum of K products of 16-bit numbers in f32: 2 K 2^-23 sum|a b|, the bound the tensor-core GEMM is held to;
* the inner product T is carried as two 16-bit numbers where the result is f32 and in the gradients: half a step of half a
  step, 2^-16 |T| (bf16) or 2^-22 |T| plus half the smallest f16 step, 2^-25 (f16); towards a 16-bit result it is rounded
  once, half a step: 2^-8 |T| (bf16) or 2^-11 |T| plus 2^-25 (f16);
* one rounding to the result's type: half a step, eps / 2, and 2^-25 for f16 below its normal range.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def kind(lib, t):
    return {F16: lib.F16, BF16: lib.BF16, F32: lib.F32}[t]


def acc(count):
    return 2.0 * count * 2.0 ** -23


def randn(gen, *shape, std=1.0, dtype=F32):
    return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)


class Lora:
    """One problem: its inputs, the library's call, the definition in 64 bits and the allowed error."""

    def __init__(self, lib, m, n, k, rank, adapters, ab, c, ids=None, seed=0, pad_x=0, pad_y=0, integers=False):
        self.lib, self.m, self.n, self.k, self.rank, self.adapters, self.ab, self.c = lib, m, n, k, rank, adapters, ab, c
        gen = self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.ldx, self.ldy = k + pad_x, n + pad_y
        if integers:  # small integers: every product and sum is exact
            draw = lambda *s, std=1.0: torch.randint(-2, 3, s, device="cuda", generator=gen).to(ab)
        else:
            draw = lambda *s, std=1.0: randn(gen, *s, std=std, dtype=ab)
        self.x_all = torch.full((m, self.ldx), float("nan"), device="cuda", dtype=ab)
        self.x_all[:, :k] = draw(m, k)
        self.x = self.x_all[:, :k]
        self.w, self.a = draw(n, k, std=k ** -0.5), draw(adapters, rank, k, std=k ** -0.5)
        self.b = draw(adapters, n, rank, std=rank ** -0.5)
        self.scale = torch.ones(adapters, device="cuda") if integers else torch.rand(adapters, device="cuda", generator=gen) + 0.5
        if ids is None or ids == "mixed":
            ids = torch.randint(-1, adapters, (m,), device="cuda", generator=gen)
        elif ids == "packed":
            ids = torch.arange(m, device="cuda") * (2 * adapters - 1) // max(m, 1) % adapters
        self.ids = ids.to(device="cuda", dtype=torch.int32).contiguous()
        self.dy_all = torch.full((m, self.ldy), float("nan"), device="cuda", dtype=ab)
        self.dy_all[:, :n] = draw(m, n, std=0.5)
        self.dy = self.dy_all[:, :n]

    def desc(self, tuning=(0, 0)):
        d = self.lib.lora_desc(self.m, self.n, self.k, self.rank, self.adapters, kind(self.lib, self.ab), kind(self.lib, self.c),
                               self.ldx if self.ldx != self.k else 0, self.ldy if self.ldy != self.n else 0)
        d.tuning[0], d.tuning[1] = tuning
        return d

    def workspace(self, size):
        return torch.full((size,), 255, device="cuda", dtype=torch.uint8)  # NaNs of every type

    def run(self, tuning=(0, 0), stream=None):
        """Y with two guard rows behind it, all of it preset to 7."""
        d = self.desc(tuning)
        y = torch.full((self.m + 2, self.ldy), 7.0, device="cuda", dtype=self.c)
        self.work = self.workspace(self.lib.lora_workspace(d))
        s = stream if stream is not None else torch.cuda.current_stream()
        self.lib.lora_tn(d, self.x.data_ptr(), self.w.data_ptr(), self.a.data_ptr(), self.b.data_ptr(), self.ids.data_ptr(),
                         self.scale.data_ptr(), y.data_ptr(), self.work.data_ptr(), s.cuda_stream)
        return y

    def rows(self, i):
        return torch.nonzero(self.ids == i).flatten()

    def inner(self, x, a, whole=True):
        """T and its bound for every row, 64 bits; whole: as two 16-bit numbers."""
        t = torch.zeros(self.m, self.rank, device="cuda", dtype=torch.float64)
        e = torch.zeros_like(t)
        x = x.double()
        for i in range(self.adapters):
            r = self.rows(i)
            if r.numel():
                s = float(self.scale[i])
                t[r] = s * (x[r] @ a[i].double().t())
                e[r] = abs(s) * acc(x.shape[1]) * (x[r].abs() @ a[i].double().abs().t()) + t[r].abs() * 2.0 ** -23
        split = HALF[self.ab] ** 2 if whole else HALF[self.ab]
        return t, e + (t.abs() + e) * split + (2.0 ** -25 if self.ab == F16 else 0.0)

    def expect(self, x, w, a, b):
        """(result, bound) of the forward operator in 64 bits."""
        t, et = self.inner(x, a, whole=self.c == F32)
        xd, wd = x.double(), w.double()
        y = xd @ wd.t()
        mag = xd.abs() @ wd.abs().t()
        err = torch.zeros_like(y)
        for i in range(self.adapters):
            r = self.rows(i)
            if r.numel():
                bd = b[i].double()
                y[r] += t[r] @ bd.t()
                mag[r] += 2 * (t[r].abs() @ bd.abs().t())
                err[r] += et[r] @ bd.abs().t()
        err += acc(x.shape[1] + 2 * self.rank) * mag
        return y, err + (y.abs() + err) * HALF[self.c] + TINY[self.c]

    def check(self, y):
        assert (y[self.m:] == 7).all() and (y[:, self.n:] == 7).all(), "wrote behind its rows or columns"
        want, bound = self.expect(self.x, self.w, self.a, self.b)
        off = (y[:self.m, :self.n].double() - want).abs()
        assert (off <= bound).all(), f"off by {(off / bound).max():.3g} of the bound"

    def back(self, with_dx=True, with_dw=True, tuning=(0, 0)):
        d = self.desc(tuning)
        dx = torch.full((self.m + 2, self.ldx), 7.0, device="cuda", dtype=self.c) if with_dx else None
        da = torch.full((self.adapters, self.rank, self.k), float("nan"), device="cuda") if with_dw else None
        db = torch.full((self.adapters, self.n, self.rank), float("nan"), device="cuda") if with_dw else None
        work = self.workspace(self.lib.lora_backward_workspace(d))
        wt = self.w.t().contiguous()
        p = lambda t: 0 if t is None else t.data_ptr()
        self.lib.lora_tn_backward(d, p(self.x), p(wt), p(self.a), p(self.b), p(self.ids), p(self.scale), p(self.dy), p(self.work),
                                  p(dx), p(da), p(db), p(work), torch.cuda.current_stream().cuda_stream)
        return dx, da, db

    def check_back(self, dx, da, db):
        u, eu = self.inner(self.dy, self.b.transpose(1, 2))
        t, et = self.inner(self.x, self.a)
        if dx is not None:
            assert (dx[self.m:] == 7).all() and (dx[:, self.k:] == 7).all(), "wrote behind its rows or columns"
            want, bound = self.expect(self.dy, self.w.t(), self.b.transpose(1, 2), self.a.transpose(1, 2))
            off = (dx[:self.m, :self.k].double() - want).abs()
            assert (off <= bound).all(), f"dX off by {(off / bound).max():.3g} of the bound"
        if da is None:
            return
        for i in range(self.adapters):
            r = self.rows(i)
            if r.numel() == 0:
                assert not da[i].any() and not db[i].any()
                continue
            x, dy = self.x[r].double(), self.dy[r].double()
            for name, got, low, elow, v in (("dA", da[i], u[r], eu[r], x), ("dB", db[i].t(), t[r], et[r], dy)):
                want = low.t() @ v
                bound = elow.t() @ v.abs() + acc(2 * r.numel()) * 2 * (low.abs().t() @ v.abs())
                off = (got.double() - want).abs()
                assert (off <= bound).all(), f"{name}[{i}] off by {(off / bound).max():.3g} of the bound"


def variants(m):
    return [(0, 0), (2, 0), (3, 0), (4, 0), (5, 0), (6, 0)] + ([(1, 0)] if m <= 128 else [])


SHAPES = [  # m, n, k, rank, adapters, ids
    (1, 1, 8, 8, 1, "packed"), (1, 300, 1000, 16, 3, "packed"), (2, 7, 72, 24, 5, "mixed"), (17, 128, 512, 16, 17, "mixed"),
    (64, 500, 264, 64, 64, "mixed"), (127, 130, 136, 40, 9, "packed"), (128, 257, 520, 128, 4, "mixed"),
    (129, 130, 72, 8, 2, "packed"), (300, 520, 1000, 32, 6, "mixed"), (513, 1025, 264, 72, 40, "mixed"),
    (1025, 384, 640, 16, 3, "packed"), (2050, 264, 4104, 128, 2, "packed"), (600, 2050, 64, 112, 600, "mixed"),
    (300, 264, 4104, 16, 100, "mixed"), (530, 513, 2056, 48, 90, "mixed"),
]


@pytest.mark.parametrize("ab,c", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("m,n,k,rank,adapters,ids", SHAPES)
def test_lora(lib, gpu, m, n, k, rank, adapters, ids, ab, c):
    p = Lora(lib, m, n, k, rank, adapters, ab, c, ids)
    for tuning in variants(m):
        p.check(p.run(tuning))
    assert lib.device_status() == (0, 0, 0, 0)


@pytest.mark.parametrize("m,n,k,rank,adapters,ids", SHAPES)
def test_lora_integers_are_exact(lib, gpu, m, n, k, rank, adapters, ids):
    # |T| <= 4 k: exact as two bf16 numbers below 2^16; |y| <= 4 k + 2 rank |T|, exact in f32 below 2^24
    p = Lora(lib, m, n, min(k, 1000), rank, adapters, BF16, F32, ids, integers=True)
    want = p.expect(p.x, p.w, p.a, p.b)[0]
    for tuning in variants(m):
        assert torch.equal(p.run(tuning)[:m].double(), want)


@pytest.mark.parametrize("ab,c", [(BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("m", [1, 20, 200])
def test_lora_result_in_the_other_16_bit_type(lib, gpu, m, ab, c):
    p = Lora(lib, m, 264, 520, 16, 5, ab, c)
    for tuning in variants(m):
        p.check(p.run(tuning))
    p.check_back(*p.back())


def test_lora_no_rows(lib, gpu):
    p = Lora(lib, 0, 64, 64, 16, 2, BF16, BF16)
    assert (p.run() == 7).all()
    dx, da, db = p.back()
    assert (dx == 7).all() and not da.any() and not db.any()


@pytest.mark.parametrize("m", [5, 128, 700])
def test_lora_ids_outside_the_table_mean_none(lib, gpu, m):
    ids = torch.tensor([-1, 3, 2 ** 31 - 1, -2 ** 31, 0, 4, 1 << 20])[torch.arange(m) % 7]
    p = Lora(lib, m, 200, 128, 16, 3, BF16, F32, ids)
    none = Lora(lib, m, 200, 128, 16, 3, BF16, F32, torch.full((m,), -1))
    for tuning in variants(m):
        y = p.run(tuning)
        p.check(y)
        none.check(none.run(tuning))
    p.check_back(*p.back())


@pytest.mark.parametrize("ab,c", [(BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("rank", [8, 16, 24])
@pytest.mark.parametrize("n,k", [(4104, 4104), (40, 64), (20000, 520), (8, 8)])
def test_lora_of_a_single_row(lib, gpu, n, k, rank, ab, c):
    for id in (0, 4, -1, 5):
        p = Lora(lib, 1, n, k, rank, 5, ab, c, torch.tensor([id]), seed=id + 1)
        p.a[2], p.b[3] = float("nan"), float("inf")  # adapters that the row does not name
        p.check(p.run())
        p.check_back(*p.back())


@pytest.mark.parametrize("m", [3, 100, 128, 1000])
def test_lora_rows_do_not_touch_one_another(lib, gpu, m):
    # Infinities and NaNs in a row, or in another row's adapter, stay there: every other row has the same bits as without.
    ids = torch.arange(m) % 5 - 1
    p = Lora(lib, m, 300, 264, 24, 4, BF16, F32, ids)
    for tuning in variants(m):
        clean = p.run(tuning)
        p.work_clean = p.work
        da_clean = p.back(tuning=tuning)[1:] if p.n % 8 == 0 else None
        q = Lora(lib, m, 300, 264, 24, 4, BF16, F32, ids)
        q.x[::5] = float("nan")       # rows without an adapter
        q.x[1::10, 3] = float("inf")  # some rows of adapter 0
        q.a[1, :, 0] = float("inf")
        q.b[2] = float("nan")
        dirty = q.run(tuning)
        same = torch.ones(m, dtype=torch.bool)
        same[::5] = False
        same[1::10] = False
        same[2::5] = False
        same[3::5] = False
        same = same.cuda()
        assert torch.equal(clean[:m][same], dirty[:m][same])
        if m >= 5:
            assert dirty[0].isnan().all() and not dirty[3].isfinite().any()


@pytest.mark.parametrize("rank", [16, 40, 128])
def test_lora_adapters_side_by_side_do_not_touch_one_another(lib, gpu, rank):
    # Many adapters per tile share T's accumulators: only the rows of the bad ones differ.
    m, adapters = 260, 90
    ids = torch.arange(m) % (adapters + 1) - 1
    bad = (ids % 7 == 3).cuda()
    p = Lora(lib, m, 264, 520, rank, adapters, BF16, F32, ids)
    q = Lora(lib, m, 264, 520, rank, adapters, BF16, F32, ids)
    q.a[3::7] = float("nan")
    q.b[3::7] = float("inf")
    for tuning in variants(m):
        clean, dirty = p.run(tuning)[:m], q.run(tuning)[:m]
        assert torch.equal(clean[~bad], dirty[~bad])
        assert not dirty[bad].isfinite().any()
        dx, dx_bad = p.back(tuning=tuning)[0][:m], q.back(tuning=tuning)[0][:m]
        assert torch.equal(dx[~bad], dx_bad[~bad])


def test_gradients_leave_masked_rows_out(lib, gpu):
    m = 500
    ids = torch.arange(m) // 7 % 5 - 1
    p = Lora(lib, m, 136, 264, 24, 4, BF16, F32, ids)
    p.run()
    _, da, db = p.back()
    q = Lora(lib, m, 136, 264, 24, 4, BF16, F32, ids)
    none = (q.ids == -1)
    q.x[none] = float("nan")
    q.dy[none] = float("inf")
    bad = (q.ids == 2)
    q.x[bad] = float("inf")
    q.run()
    _, da2, db2 = q.back()
    for i in (0, 1, 3):
        assert torch.equal(da[i], da2[i]) and torch.equal(db[i], db2[i])
    assert not da2[2].isfinite().all()


@pytest.mark.parametrize("ab,c", [(BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("m", [9, 400])
def test_lora_pitches(lib, gpu, m, ab, c):
    p = Lora(lib, m, 200, 136, 16, 3, ab, c, pad_x=24, pad_y=8)
    for tuning in variants(m):
        p.check(p.run(tuning))
    p.check_back(*p.back())
    odd = Lora(lib, m, 201, 136, 16, 3, ab, c, pad_y=6)  # rows of Y on odd addresses
    for tuning in variants(m):
        odd.check(odd.run(tuning))


BACK = [
    (1, 8, 8, 8, 1, "packed"), (3, 72, 136, 16, 2, "mixed"), (64, 264, 520, 64, 9, "mixed"), (127, 128, 64, 40, 3, "packed"),
    (129, 520, 72, 128, 2, "mixed"), (777, 264, 1000, 24, 5, "packed"), (1500, 1032, 648, 16, 70, "mixed"),
    (2050, 136, 128, 8, 1, "packed"), (300, 4104, 264, 16, 100, "mixed"), (530, 1032, 520, 96, 90, "mixed"),
]


@pytest.mark.parametrize("ab,c", [(BF16, BF16), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("m,n,k,rank,adapters,ids", BACK)
def test_lora_backward(lib, gpu, m, n, k, rank, adapters, ids, ab, c):
    p = Lora(lib, m, n, k, rank, adapters, ab, c, ids)
    p.check(p.run())
    first = p.back()
    p.check_back(*first)
    again = p.back()
    assert all(torch.equal(a, b) for a, b in zip(first, again)), "the same call gave other bits"
    for tuning in variants(m)[2:]:
        p.check_back(*p.back(tuning=tuning))
    dx, _, _ = p.back(with_dw=False)
    assert torch.equal(dx, first[0])
    _, da, db = p.back(with_dx=False)
    assert torch.equal(da, first[1]) and torch.equal(db, first[2])
    assert lib.device_status() == (0, 0, 0, 0)


def test_gradients_against_differences(lib, gpu):
    # f(X, A, B) = <dY, Y> is linear in each of X, A, B: a difference over a step of the argument's own grid is exact up to
    # the rounding of Y, whose bound is known.
    p = Lora(lib, 200, 64, 128, 16, 3, F16, F32)
    base = p.run()[:p.m].double()
    _, bound = p.expect(p.x, p.w, p.a, p.b)
    dx, da, db = p.back()
    weight = p.dy.double()
    slack = 2 * (weight.abs() * bound).sum()
    for name, t, grad, at in (("x", p.x, dx, (5, 17)), ("a", p.a, da, (1, 3, 9)), ("b", p.b, db, (2, 40, 7))):
        old = t[at].clone()
        t[at] = old + 4.0
        step = float(t[at].double() - old.double())
        f = (weight * (p.run()[:p.m].double() - base)).sum()
        # with A changed the bound of Y grows with T: measure it again
        _, b2 = p.expect(p.x, p.w, p.a, p.b)
        t[at] = old
        allowed = (slack + 2 * (weight.abs() * b2).sum()) / step + 1e-3 * abs(float(grad[at]))
        assert abs(float(f) / step - float(grad[at])) <= float(allowed), name


def test_lora_captured_and_replayed_with_other_rows(lib, gpu):
    for m in (1, 24, 300):
        p, q = (Lora(lib, m, 264, 136, 16, 6, BF16, F32, seed=s) for s in (1, 2))
        d = p.desc()
        y, work = torch.zeros(m, p.n, device="cuda"), p.workspace(lib.lora_workspace(d))
        y2, work2 = torch.zeros(m, p.n, device="cuda"), p.workspace(lib.lora_workspace(d))
        x, ids = p.x.contiguous().clone(), p.ids.clone()
        def call(out, w):
            lib.lora_tn(d, x.data_ptr(), p.w.data_ptr(), p.a.data_ptr(), p.b.data_ptr(), ids.data_ptr(), p.scale.data_ptr(),
                        out.data_ptr(), w.data_ptr(), torch.cuda.current_stream().cuda_stream)
        graphs = []
        for out, w in ((y, work), (y2, work2)):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call(out, w)
                call(out, w)  # back to back on one workspace
            graphs.append(g)
        for src in (p, q):
            x.copy_(src.x)
            ids.copy_(src.ids)
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            now = Lora(lib, m, 264, 136, 16, 6, BF16, F32, seed=1)
            now.x.copy_(src.x)
            now.ids.copy_(src.ids)
            want = now.run()[:m]
            assert torch.equal(y, want) and torch.equal(y2, want)


def test_lora_on_several_streams_at_once(lib, gpu):
    ps = [Lora(lib, m, 520, 264, 16, 6, BF16, F32, seed=i) for i, m in enumerate((40, 340, 1))]
    want = [p.run() for p in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    got = [[] for _ in ps]
    for _ in range(20):
        for i, (p, s) in enumerate(zip(ps, streams)):
            with torch.cuda.stream(s):
                got[i].append(p.run(stream=s))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)


def test_lora_offsets_past_32_bits(lib, gpu):
    # B holds more than 2^31 numbers; the rows name the last adapters.
    n, rank, adapters = 4096, 128, 4200
    p = Lora(lib, 1, 8, 8, 8, 1, BF16, F32)
    p.m, p.n, p.k, p.rank, p.adapters = 150, n, 64, rank, adapters
    p.ldx, p.ldy = 64, n
    p.x = randn(p.gen, 150, 64, dtype=BF16)
    p.w = randn(p.gen, n, 64, std=0.1, dtype=BF16)
    p.a = randn(p.gen, adapters, rank, 64, std=0.1, dtype=BF16)
    p.b = torch.empty(adapters, n, rank, device="cuda", dtype=BF16)
    p.b[-3:] = randn(p.gen, 3, n, rank, std=0.1, dtype=BF16)
    p.scale = torch.ones(adapters, device="cuda")
    p.ids = (adapters - 1 - torch.arange(150, device="cuda") % 3).to(torch.int32)
    for m in (150, 100):
        p.m, p.x, p.ids = m, p.x[:m], p.ids[:m]
        p.check(p.run())


def test_lora_result_past_32_bits(lib, gpu):
    m, n = 66000, 33000
    p = Lora(lib, m, n, 8, 8, 1, BF16, BF16, ids="packed")
    y = p.run()
    for lo in (0, 65072, m - 64):
        q = Lora(lib, 1, 8, 8, 8, 1, BF16, BF16)
        q.m, q.n, q.k, q.rank, q.adapters, q.w, q.a, q.b, q.scale = 64, n, 8, 8, 1, p.w, p.a, p.b, p.scale
        q.x, q.ids = p.x[lo:lo + 64], p.ids[lo:lo + 64]
        want, bound = q.expect(q.x, q.w, q.a, q.b)
        assert ((y[lo:lo + 64].double() - want).abs() <= bound).all()
    assert (y[m:] == 7).all()


# ---- mixture of experts ------------------------------------------------------------


class Moe:
    def __init__(self, lib, tokens, experts, top, d, f, dtype, renorm=True, seed=0, spread=3.0):
        self.lib, self.tokens, self.experts, self.top, self.d, self.f, self.dtype, self.renorm = lib, tokens, experts, top, d, f, dtype, renorm
        gen = self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.x = randn(gen, tokens, d, dtype=dtype)
        self.r = randn(gen, experts, d, std=spread * d ** -0.5, dtype=dtype)
        self.g, self.u = (randn(gen, experts, f, d, std=d ** -0.5, dtype=dtype) for _ in range(2))
        self.dn = randn(gen, experts, d, f, std=f ** -0.5, dtype=dtype)

    def desc(self):
        return self.lib.moe_desc(self.tokens, self.experts, self.top, self.d, self.f, kind(self.lib, self.dtype), self.renorm)

    def run(self, stream=None, tuning=0):
        y = torch.full((self.tokens + 2, self.d), 7.0, device="cuda", dtype=self.dtype)
        desc = self.desc()
        desc.tuning[1] = tuning
        work = torch.full((self.lib.moe_workspace(desc),), 255, device="cuda", dtype=torch.uint8)
        s = stream if stream is not None else torch.cuda.current_stream()
        self.lib.moe_tn(desc, self.x.data_ptr(), self.r.data_ptr(), self.g.data_ptr(), self.u.data_ptr(), self.dn.data_ptr(),
                        y.data_ptr(), work.data_ptr(), s.cuda_stream)
        return y

    def expect(self):
        """y and its bound in 64 bits.  Where two logits at the border of the choice lie closer than their bound the choice
        would be open; the tests' inputs are checked not to do that (equal logits go to the lower index)."""
        x, r = self.x.double(), self.r.double()
        logits = x @ r.t()
        # The router's sums run in f32 by 32 lanes side by side and a tree: no more than d / 32 + 16 additions in a row, each off
        # by half a step (of any logit of the token).
        el = (self.d / 32 + 16) * 2.0 ** -24 * (x.abs() @ r.abs().t()).amax(1)
        order = torch.sort(logits, dim=1, descending=True, stable=True)
        if self.top < self.experts and self.tokens:
            gap = order.values[:, self.top - 1] - order.values[:, self.top]
            assert ((gap > 2 * el) | (gap == 0)).all(), "the inputs leave the choice open"
        chosen = order.indices[:, :self.top]
        p = torch.softmax(logits, 1).gather(1, chosen)
        rel = torch.expm1(2 * el) + 2.0 ** -19  # exp, sums of up to 512, division
        if self.renorm:
            p, rel = p / p.sum(1, keepdim=True), 2 * rel + 2.0 ** -20
        y = torch.zeros(self.tokens, self.d, device="cuda", dtype=torch.float64)
        err, mag = torch.zeros_like(y), torch.zeros_like(y)
        for e in torch.unique(chosen).tolist():
            t, slot = torch.nonzero(chosen == e, as_tuple=True)
            g, u = self.g[e].double(), self.u[e].double()
            xv = x[t]
            gv, uv = xv @ g.t(), xv @ u.t()
            eg, eu = acc(self.d) * (xv.abs() @ g.abs().t()), acc(self.d) * (xv.abs() @ u.abs().t())
            w = p[t, slot][:, None]
            s = gv * torch.sigmoid(gv)
            h = w * s * uv
            eh = w * (1.1 * eg * (uv.abs() + eu) + s.abs() * eu) + h.abs() * (rel[t][:, None] + 2.0 ** -20)  # |silu'| < 1.1
            eh = eh + (h.abs() + eh) * HALF[self.dtype] + TINY[self.dtype]
            dn = self.dn[e].double()
            y[t] += h @ dn.t()
            err[t] += eh @ dn.abs().t()
            mag[t] += (h.abs() + eh) @ dn.abs().t()
        err += acc(self.f * self.top) * mag
        return y, err + (y.abs() + err) * HALF[self.dtype] + TINY[self.dtype]

    def check(self, y):
        assert (y[self.tokens:] == 7).all()
        want, bound = self.expect()
        off = (y[:self.tokens].double() - want).abs()
        assert (off <= bound).all(), f"off by {(off / bound).max():.3g} of the bound"


MOE = [  # tokens, experts, top, d, f, renorm
    (1, 1, 1, 8, 8, True), (1, 8, 2, 1024, 520, True), (2, 3, 3, 72, 24, False), (3, 512, 16, 136, 8, True),
    (5, 10, 3, 520, 328, True), (8, 64, 6, 264, 72, False), (17, 16, 1, 640, 136, True), (33, 130, 8, 128, 200, False),
    (64, 4, 2, 2056, 264, True), (64, 128, 8, 256, 64, True), (63, 2, 1, 64, 1032, False), (64, 300, 16, 64, 40, True),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,experts,top,d,f,renorm", MOE)
def test_moe(lib, gpu, tokens, experts, top, d, f, renorm, dtype):
    p = Moe(lib, tokens, experts, top, d, f, dtype, renorm)
    y = p.run()
    p.check(y)
    assert torch.equal(y, p.run()), "the same call gave other bits"
    assert lib.device_status() == (0, 0, 0, 0)


def test_moe_no_tokens(lib, gpu):
    assert (Moe(lib, 0, 4, 2, 64, 64, BF16).run() == 7).all()


@pytest.mark.parametrize("top", [1, 3])
def test_moe_equal_logits_go_to_the_lower_index(lib, gpu, top):
    p = Moe(lib, 20, 40, top, 128, 64, BF16)
    p.r[:] = p.r[torch.arange(40) // 5 * 5].clone()  # groups of five equal experts' rows
    p.check(p.run())
    p.r.zero_()  # all equal: experts 0 .. top - 1
    p.check(p.run())


def test_moe_everybody_chooses_the_same_experts(lib, gpu):
    p = Moe(lib, 64, 32, 2, 256, 136, BF16)
    p.x[:, 0] = 8.0
    p.r.zero_()
    p.r[7, 0] = 4.0
    p.r[31, 0] = 2.0
    p.check(p.run())


def test_moe_tokens_do_not_touch_one_another(lib, gpu):
    p = Moe(lib, 30, 16, 3, 264, 136, BF16)
    clean = p.run()
    p.x[4] = float("nan")
    p.x[17, 5] = float("inf")
    p.x[20, 0] = float("-inf")
    y = p.run()
    rest = [t for t in range(30) if t not in (4, 17, 20)]
    assert torch.equal(clean[rest], y[rest])
    assert not y[4].isfinite().any() and not y[17].isfinite().any()


def test_moe_unchosen_experts_are_not_read(lib, gpu):
    p = Moe(lib, 6, 12, 2, 128, 72, BF16)
    clean = p.run()
    chosen = torch.unique(torch.sort(p.x.double() @ p.r.double().t(), dim=1, descending=True, stable=True).indices[:, :2])
    left = [e for e in range(12) if e not in chosen.tolist()]
    assert left
    for t in (p.g, p.u, p.dn):
        t[left] = float("nan")
    assert torch.equal(clean, p.run())


def test_moe_captured_and_replayed(lib, gpu):
    p, q = Moe(lib, 12, 24, 4, 256, 136, BF16, seed=1), Moe(lib, 12, 24, 4, 256, 136, BF16, seed=2)
    desc = p.desc()
    outs = []
    x = p.x.clone()
    for _ in range(2):
        y, work = torch.zeros(12, 256, device="cuda", dtype=BF16), torch.full((lib.moe_workspace(desc),), 255, device="cuda", dtype=torch.uint8)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(2):
                lib.moe_tn(desc, x.data_ptr(), p.r.data_ptr(), p.g.data_ptr(), p.u.data_ptr(), p.dn.data_ptr(), y.data_ptr(),
                           work.data_ptr(), torch.cuda.current_stream().cuda_stream)
        outs.append((g, y, work))
    for src in (p, q):
        x.copy_(src.x)
        for g, _, _ in outs:
            g.replay()
        torch.cuda.synchronize()
        now = Moe(lib, 12, 24, 4, 256, 136, BF16, seed=1)
        now.x.copy_(src.x)
        want = now.run()[:12]
        assert all(torch.equal(y, want) for _, y, _ in outs)


def test_moe_on_two_streams_at_once(lib, gpu):
    ps = [Moe(lib, 3 + 40 * i, 24, 4, 256, 136, BF16, seed=i) for i in range(2)]
    want = [p.run() for p in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    got = [[], []]
    for _ in range(20):
        for i, (p, s) in enumerate(zip(ps, streams)):
            with torch.cuda.stream(s):
                got[i].append(p.run(stream=s))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)


# ---- bounded waits -------------------------------------------------------------------


def test_waits_that_run_out_are_reported(lib, gpu):
    """The producers issue nothing (a test knob): every wait gives up after 20 ms, the kernels return, the report names it,
    and the next call on the same device is right."""
    one = Lora(lib, 1, 264, 520, 16, 6, BF16, F32)
    few, tiled, moe = Lora(lib, 20, 264, 136, 72, 6, BF16, F32), Lora(lib, 700, 264, 136, 16, 6, BF16, F32), Moe(lib, 12, 24, 4, 256, 136, BF16)
    calls = [lambda: one.run((1, 12)), lambda: few.run((1, 12))] + [lambda c=c: tiled.run((c, 12)) for c in (3, 4, 5, 6)] + [lambda: moe.run(tuning=12)]
    for call in calls:
        call()
        with pytest.raises(lib.CuteB200Error) as e:
            lib.synchronize()
        assert e.value.status == lib.ERR_DEVICE_TIMEOUT
        assert lib.device_status() == (0, 0, 0, 0)
    one.check(one.run())
    few.check(few.run())
    tiled.check(tiled.run())
    d = tiled.desc((0, 12))
    da, db, work = torch.empty_like(tiled.a, dtype=F32), torch.empty_like(tiled.b, dtype=F32), tiled.workspace(lib.lora_backward_workspace(d))
    wt = tiled.w.t().contiguous()
    lib.lora_tn_backward(d, tiled.x.data_ptr(), wt.data_ptr(), tiled.a.data_ptr(), tiled.b.data_ptr(), tiled.ids.data_ptr(),
                         tiled.scale.data_ptr(), tiled.dy.data_ptr(), tiled.work.data_ptr(), 0, da.data_ptr(), db.data_ptr(),
                         work.data_ptr(), torch.cuda.current_stream().cuda_stream)
    with pytest.raises(lib.CuteB200Error) as e:
        lib.synchronize()
    assert e.value.status == lib.ERR_DEVICE_TIMEOUT
    tiled.check_back(*tiled.back())
    moe.check(moe.run())
    assert lib.device_status() == (0, 0, 0, 0)


# ---- together ------------------------------------------------------------------------


def test_a_block_of_them_as_a_model_runs_them(lib, gpu):
    """gemm_tn -> lora_tn -> moe_tn -> lora_tn on one stream, each reading what the one before wrote, no waits between."""
    tokens, d = 24, 256
    one, two = Lora(lib, tokens, d, d, 16, 5, BF16, BF16, seed=3), Lora(lib, tokens, 136, d, 32, 4, BF16, F32, seed=4)
    moe = Moe(lib, tokens, 12, 3, d, 136, BF16, seed=5)
    x0, w0 = randn(one.gen, tokens, d, dtype=BF16), randn(one.gen, d, d, std=d ** -0.5, dtype=BF16)
    for _ in range(3):
        s = torch.cuda.current_stream().cuda_stream
        lib.gemm_tn(lib.gemm_desc(tokens, d, d, lib.BF16, lib.BF16), x0.data_ptr(), w0.data_ptr(), one.x_all.data_ptr(), s)
        y1 = torch.empty(tokens, d, device="cuda", dtype=BF16)
        w1 = one.workspace(lib.lora_workspace(one.desc()))
        lib.lora_tn(one.desc(), one.x.data_ptr(), one.w.data_ptr(), one.a.data_ptr(), one.b.data_ptr(), one.ids.data_ptr(),
                    one.scale.data_ptr(), y1.data_ptr(), w1.data_ptr(), s)
        moe.x = y1
        wm = torch.empty(lib.moe_workspace(moe.desc()), device="cuda", dtype=torch.uint8)
        lib.moe_tn(moe.desc(), y1.data_ptr(), moe.r.data_ptr(), moe.g.data_ptr(), moe.u.data_ptr(), moe.dn.data_ptr(),
                   two.x_all.data_ptr(), wm.data_ptr(), s)
        y2 = two.run()
    torch.cuda.synchronize()
    one.check(torch.cat([y1, torch.full((2, d), 7.0, device="cuda", dtype=BF16)]))
    moe.check(torch.cat([two.x, torch.full((2, d), 7.0, device="cuda", dtype=BF16)]))
    two.check(y2)
