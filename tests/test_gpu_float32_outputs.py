"""float32 results of the gated activations are the same numbers whichever tiles a product runs on."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob

pytestmark = pytest.mark.gpu

F64 = torch.float64


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("m,n,k", [(1, 300, 192), (3, 8192, 192), (40, 513, 160), (100, 2000, 192),
                                   (300, 1001, 320), (1500, 2304, 192)])
def test_float32_activations(cuda, act, codes, m, n, k):
    """Whole-number codes and a power-of-two scale: the sums are exact in fp32 in every order, so all
    tensor-core tiles (one K block, blocks of 128) have to return the same bits. Against 64 bits, in
    units of 2^-24 of the value: z is exact for silu and off by 6 |z| at most for gelu (two rounded
    constants, four operations), which moves the exponential by as much, expf itself by 4, both
    weighted by 1 - sigmoid; the sum, the quotient (2) and the residual's addition round. A sigmoid
    below 2^-126, fp32's last normal number, may come out as zero (|x| < 16)."""
    gen = torch.Generator().manual_seed(m + n)
    hi = 8
    a = torch.randint(-hi, hi + 1, (m, k), generator=gen).float().to(codes).to(cuda)
    b = torch.randint(-hi, hi + 1, (n, k), generator=gen).float().to(codes).to(cuda)
    bias = (torch.randint(-64, 65, (n,), generator=gen) / 64).to(cuda)
    res = torch.randn(m, n, generator=gen).to(cuda)
    op = (tob.w8a8_block_int8_matmul_bias_act if codes == torch.int8
          else tob.w8a8_block_fp8_matmul_bias_act)

    def run(bn, bk, residual):
        a_s = torch.full((m, -(-k // bk)), 2.0 ** -4, device=cuda)
        b_s = torch.full((-(-n // bn), -(-k // bk)), 2.0 ** -3, device=cuda)
        return op(a, b, a_s, b_s, [bn, bk], bias, act=act, residual=residual,
                  output_dtype=torch.float32)

    x = (a.float().to(F64) @ b.float().to(F64).t()) * 2.0 ** -7 + bias.to(F64)
    z = {"silu": x, "gelu": (8 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)}.get(act)
    for residual in (None, res):
        want = x if act is None else x.clamp(min=0) if act == "relu" else x * torch.sigmoid(z)
        unit = 0.0 if z is None else 3 + 4 * (1 - torch.sigmoid(z))
        if act == "gelu":
            unit = unit + 6 * z.abs() * (1 - torch.sigmoid(z))
        tol = unit * want.abs() * 2.0 ** -24 * (1 + 1e-6) + 2.0 ** -122
        if residual is not None:
            want = want + res.to(F64)
            tol = tol + want.abs() * 2.0 ** -24 * (1 + 1e-6)
        first = run(1, k, residual)
        for bn, bk in ((1, k), (n, k), (1, 128), (128, 128), (1, 64)):
            y = run(bn, bk, residual)
            assert bool(((y.to(F64) - want).abs() <= tol).all()), (bn, bk)
            assert bk == 64 or torch.equal(y, first), (bn, bk)  # 64: the SIMT tiles


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_float32_limits(cuda, act, m):
    """Far arguments: the value itself above, zero below, NaN for NaN and -inf as x sigmoid(x) is."""
    n, k = 4096, 64
    a = torch.ones(m, k, dtype=torch.int8, device=cuda)
    b = torch.zeros(n, k, dtype=torch.int8, device=cuda)
    bias = torch.zeros(n, device=cuda)
    vals = [float("inf"), float("-inf"), float("nan"), 1e30, -1e30, 200.0, -200.0, -0.0, 1e-40]
    bias[:9] = torch.tensor(vals)
    y = tob.w8a8_block_int8_matmul_bias_act(
        a, b, torch.ones(m, 1, device=cuda), torch.ones(n, 1, device=cuda), [1, k], bias, act=act,
        output_dtype=torch.float32)
    want = [float("inf"), float("nan"), float("nan"), float(torch.tensor(1e30)), 0.0, 200.0, 0.0, 0.0]
    torch.testing.assert_close(y[:, :8], torch.tensor(want, device=cuda).expand(m, 8), rtol=0,
                               atol=1e-36, equal_nan=True)
    assert bool((y[:, 8].abs() <= 1e-40).all()) and bool((y[:, 9:] == 0).all())
