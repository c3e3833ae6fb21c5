"""8-bit operators at the ends of their ranges: gates of every size under SiLU, and what is no number there."""
import pytest
import torch

from tilelang_moe_b200 import kernels

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = 2.0 ** -100                     # the largest magnitude of a group counts as at least this


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("I", [256, 250, 129])
def test_silu_mul_of_gates_of_every_size(cuda, lib, I, dtype):
    """The fp32 scale shows what the 8-bit values do not.  exp is off by 2 units of 2^-23 at most, and by as much or less once 1
    is added; that sum, the quotient and the product are rounded once each: 2^-22 + 3 * 2^-24 < 2^-21.  The scale's own division
    adds 2^-24."""
    g = torch.Generator().manual_seed(I)
    ends = [-88.7, -85.0, -80.0, -60.0, -40.0, -20.0, -10.0, -5.0, -1.0, -1e-3, 0.0, 1e-3, 1.0, 20.0, 88.0, 1e4]
    rows = []
    for lo, hi in zip(ends, ends[1:]):           # a row for each range: its groups' largest products come from there
        rows.append(lo + (hi - lo) * torch.rand(8, I, generator=g))
    gate = torch.cat(rows)
    if dtype != torch.float32:                   # rounded towards zero: no gate below the lowest end
        gate = torch.where(gate.to(dtype).float().abs() > gate.abs(), gate * (1 - 2 * torch.finfo(dtype).eps), gate)
    gate = gate.to(dtype)
    up = torch.randn(gate.shape, generator=g)
    up = ((up * 8192).clamp(-6e4, 6e4) if dtype == torch.float16 else up * 2.0 ** 60).to(dtype)
    want = gate.double() * torch.sigmoid(gate.double()) * up.double()
    q, scale = (t.cpu() for t in kernels.fp8_silu_mul(gate.to(cuda), up.to(cuda)))
    slack = 2.0 ** -21
    for j in range(scale.shape[1]):
        x, got = want[:, j * 128:(j + 1) * 128], q[:, j * 128:(j + 1) * 128].float().double()
        top = x.abs().amax(1, keepdim=True).clamp(min=TINY)
        assert torch.all((scale[:, j:j + 1].double() - top / 448).abs() <= (slack + 2.0 ** -24) * top / 448)
        v = x * (448 / top)
        big = torch.maximum(v.abs(), got.abs())
        step = 2.0 ** (torch.floor(torch.log2(big.clamp(min=2.0 ** -6))) - 3)
        assert torch.all((got - v).abs() <= step / 2 + v.abs() * (2 * slack + 2.0 ** -22))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("I", [256, 250])
def test_silu_mul_of_what_is_no_number(cuda, lib, I, dtype):
    nan, inf = float("nan"), float("inf")
    gate, up = torch.ones(11, I), torch.ones(11, I)
    gate[0, 3], up[1, 4], gate[2, 5], up[3, 6] = nan, nan, -inf, -nan       # -inf * sigmoid(-inf) is -inf * 0
    gate[4, 7], up[5, 8], up[6, 9] = inf, inf, -inf
    gate[7, 10], up[7, 10] = 0.0, inf                                       # 0 * inf
    gate[8, :128], gate[9, :128] = -89.0, -1e4 if dtype != torch.float16 else -6e4      # exp overflows: nothing is left
    gate[10, 0] = -0.0
    q, scale = (t.cpu() for t in kernels.fp8_silu_mul(gate.to(dtype).to(cuda), up.to(dtype).to(cuda)))
    q = q.float()
    back = q[:, :128] * scale[:, :1]
    assert torch.isnan(back[[0, 1, 2, 3, 7]]).all()
    assert torch.all(scale[[4, 5, 6], 0] == inf) and torch.isnan(q[4, 7]) and torch.isnan(q[5, 8]) and torch.isnan(q[6, 9])
    assert torch.all(q[[8, 9], :128] == 0) and torch.all((scale[[8, 9], 0].double() * 448 / TINY - 1).abs() <= 2.0 ** -24)
    assert q[10, 0] == 0 and torch.all(q[10, 1:128] == 448)
    assert torch.all(q[:, 128:] == 448)                                     # the group beside them is as it should be
    one = torch.sigmoid(torch.ones((), dtype=torch.float64)) / 448
    assert torch.all((scale[:, 1].double() / one - 1).abs() <= 2.0 ** -21 + 2.0 ** -24)
