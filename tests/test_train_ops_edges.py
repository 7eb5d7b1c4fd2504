"""The training operators at their edges: what the documentation allows and tests/test_train_ops.py does not call."""
import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs an MI355X"
    from videoitg_amd import ops as o
    return o


def interleave(gate, up):
    return torch.stack([gate.unflatten(-1, (-1, 32)), up.unflatten(-1, (-1, 32))], -2).flatten(-3)


# rows few enough for one pass; ring kernel with a join; 256x256 tiles whole, with ragged edges too; tiles split over the rows; 256x384 tiles whole
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [(20, 1088, 2048), (300, 256, 832), (2100, 1024, 16384), (1100, 1088, 16448), (7000, 1088, 2048), (4100, 3584, 9472)])
def test_weight_gradient_is_added_once_on_every_route(ops, dtype, m, k, n):
    """gate = 0 (sigmoid 1/2, dU = 0), up 1 or 2 and whole x and dout: dGU and every partial sum are exact, so that one rounding is left - that of old + sum.  A route
    that carries the large old value through the sum rounds once per step"""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    whole = lambda *s: torch.randint(-4, 5, s, generator=g, device="cuda", dtype=torch.int32).to(dtype)      # noqa: E731
    x, dout, w = whole(m, k), whole(m, n // 2), whole(n, k)
    up = torch.randint(1, 3, (m, n // 2), generator=g, device="cuda").to(dtype)
    gu = interleave(torch.zeros_like(up), up)
    old = torch.randn(n, k, generator=g, device="cuda") * 1e5
    dgu = interleave(dout.double() * up.double() / 2, torch.zeros_like(up, dtype=torch.float64))
    want = (old.double() + dgu.t() @ x.double()).float()
    for dx in (None, torch.empty_like(x)):
        dw = old.clone()
        ops.swiglu_backward(dout, gu, x, w, dx=dx, dw=dw, accumulate=True)
        assert torch.equal(dw, want), f"{int((dw != want).sum())} of {dw.numel()} rounded more than once"
