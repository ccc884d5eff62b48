"""moe_tn at the edges of what its router may meet, and on operands written just before the call."""
import pytest
import torch

from tests.test_gpu_rows import BF16, F16, Moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("renorm", [True, False])
def test_a_logit_of_minus_infinity_is_a_probability_of_zero(lib, gpu, dtype, renorm):
    # Experts 1, 5 and 6 of eight get the logit -inf from every token; five are chosen, so none of them is.  The same bits as with
    # a logit so low that its exponential is zero.
    p = Moe(lib, 9, 8, 5, 136, 72, dtype, renorm)
    p.x[:, 0] = 1.0
    low = torch.tensor([1, 5, 6])
    p.r[low] = 0.0
    p.r[low, 0] = -30000.0
    want = p.run()
    p.check(want)
    p.r[low, 0] = float("-inf")
    assert torch.equal(p.run(), want)
    # With all eight chosen, theirs count with weight zero, whatever is finite in their weights.
    p.top = 8
    p.r[low, 0] = -30000.0
    want = p.run()
    p.r[low, 0] = float("-inf")
    assert want.isfinite().all() and torch.equal(p.run(), want)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_logits_without_a_softmax_give_nans_to_their_token_alone(lib, gpu, value):
    p = Moe(lib, 12, 8, 3, 136, 72, BF16)
    p.x[:, 0] = 0.0
    p.r[:, 0] = 1.0
    clean = p.run()
    p.x[7, 0] = value
    y = p.run()
    assert y[7].isnan().all()
    rest = [t for t in range(12) if t != 7]
    assert torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("tokens", [1, 12, 64])
def test_moe_operands_written_just_before_the_call(lib, gpu, tokens):
    """Kernels that write every operand, then the layer, over and over without a wait: what a kernel loads ahead of the one before
    it must be the new values."""
    ps = [Moe(lib, tokens, 24, 4, 256, 136, BF16, seed=s) for s in range(4)]
    want = [p.run() for p in ps]
    torch.cuda.synchronize()
    own = Moe(lib, tokens, 24, 4, 256, 136, BF16, seed=9)
    got = []
    for _ in range(10):
        for p in ps:
            for dst, src in zip((own.x, own.r, own.g, own.u, own.dn), (p.x, p.r, p.g, p.u, p.dn)):
                torch.add(src, 0, out=dst)
            got.append(own.run())
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4])
