"""The step sizes of the scan by themselves: softplus over its whole range."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_softplus_error_bound():
    """One token from a zero state with one state of B = C = 1 and x = 1 returns d = softplus(dt) exactly.

    u = exp(-|v|) is off by |v| (1 + 0.25) 2^-24 of itself (the rounding of the exponent and of log2 e) and 4 roundings
    of the hardware's 2^x; the quotient, the polynomial and the products add at most 8.  A result below the smallest
    normal number is 0."""
    from boa_b200 import ops
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.linspace(-95, 95, 3000), torch.randn(1000, generator=g), torch.tensor([0.0, -0.0, 1e-30, -1e-30]),
                   torch.linspace(-87.4, -87.2, 92)])
    n = v.numel()
    one = torch.zeros(1, 1, 16, device="cuda")
    one[..., 0] = 1.0
    x, dt, A = torch.ones(1, 1, n, device="cuda"), v.cuda().view(1, 1, n), torch.zeros(n, 16, device="cuda")
    want = torch.logaddexp(v.double(), torch.zeros(n).double())
    bound = (12 + 1.25 * (-v.double()).clamp(min=0)) * 2.0 ** -24 * want + torch.finfo(torch.float32).tiny
    with torch.no_grad():
        whole = ops.ssm_scan(x, dt, A, one, one)[0, 0]
        odd = ops.ssm_scan(x[..., :n - 1], dt[..., :n - 1], A[:n - 1], one, one)[0, 0]      # element by element
        step = ops.ssm_step(x[:, 0], dt[:, 0], torch.zeros(1, n, 16, device="cuda"), A, one[:, 0], one[:, 0])[0]
    for got in (whole, odd, step):
        off = (got.double().cpu() - want[:got.numel()]).abs()
        assert (off <= bound[:got.numel()]).all(), (off / bound[:got.numel()]).max()
    assert (whole[v.cuda() < -88] == 0).all()
