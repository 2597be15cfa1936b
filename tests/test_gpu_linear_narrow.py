"""Products with an epilogue whose rows end inside 16 bytes, written into and read from aligned rows
that are wider: nothing past the last column is written, or read into a sum."""

from __future__ import annotations

import pytest
import torch

import tileops_b200 as tob

pytestmark = pytest.mark.gpu

F64 = torch.float64


@pytest.mark.parametrize("kind", ["dense", "channel", "block", "odd_block"])
@pytest.mark.parametrize("m", [70, 9601, 19001])
@pytest.mark.parametrize("n", [1, 3, 8, 31, 33, 70])
def test_narrow_results(cuda, kind, m, n):
    k = 160
    gen = torch.Generator(device=cuda).manual_seed(m + n)

    def ri(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=gen, device=cuda)

    a, b, bias = ri(-3, 3, m, k), ri(-2, 2, n, k), ri(-8, 8, n).half()
    pitch = -(-n // 8) * 8 + 8
    wide_r, wide_o = ri(-8, 8, m, pitch).half(), torch.full((m, pitch), 7, device=cuda).half()
    res, out = wide_r[:, :n], wide_o[:, :n]
    want = ((a.to(F64) @ b.to(F64).t() + bias.to(F64)).clamp(min=0) + res.to(F64)).half()

    def run(residual, dst):
        if kind == "dense":
            return tob.gemm_bias_act(a.half(), b.half().t().contiguous(), bias, act="relu",
                                     residual=residual, out=dst)
        bn, bk = {"channel": (1, k), "block": (128, 128), "odd_block": (48, 128)}[kind]
        return tob.w8a8_block_int8_matmul_bias_act(
            a.to(torch.int8), b.to(torch.int8), torch.ones(m, -(-k // bk), device=cuda),
            torch.ones(-(-n // bn), -(-k // bk), device=cuda), [bn, bk], bias, act="relu",
            residual=residual, out=dst)

    assert run(res, out) is out
    assert torch.equal(out, want) and bool((wide_o[:, n:] == 7).all())
    rest = wide_r[:, n:].clone()
    run(res, res)
    assert torch.equal(res, want) and torch.equal(wide_r[:, n:], rest)


@pytest.mark.parametrize("m,n,k", [(4, 64, 61), (70, 136, 1001), (300, 1000, 333), (2000, 2048, 77)])
def test_rows_of_a_that_end_inside_16_bytes(cuda, m, n, k):
    """A as the first k columns of aligned rows whose other columns are NaN: none of those is read
    into the sums."""
    gen = torch.Generator(device=cuda).manual_seed(m)
    pitch = -(-k // 8) * 8 + 8
    wide = torch.full((m, pitch), float("nan"), device=cuda).half()
    wide[:, :k] = torch.randint(-3, 4, (m, k), generator=gen, device=cuda).half()
    b = torch.randint(-2, 3, (k, n), generator=gen, device=cuda).half()
    want = (wide[:, :k].to(F64) @ b.to(F64)).half()
    assert torch.equal(tob.gemm_bias_act(wide[:, :k], b), want)


@pytest.mark.parametrize("m,n,k", [(400, 6001, 64), (1000, 2049, 136)])
@pytest.mark.parametrize("kind", ["dense", "channel", "block"])
def test_wide_results_that_end_inside_16_bytes(cuda, kind, m, n, k):
    gen = torch.Generator(device=cuda).manual_seed(n)
    a = torch.randint(-3, 4, (m, k), generator=gen, device=cuda)
    b = torch.randint(-2, 3, (n, k), generator=gen, device=cuda)
    want = (a.to(F64) @ b.to(F64).t()).half()
    wide = torch.full((m, n + 15), 7, device=cuda).half()
    out = wide[:, :n]
    if kind == "dense":
        tob.gemm_bias_act(a.half(), b.half().t().contiguous(), out=out)
    else:
        bn, bk = (1, k) if kind == "channel" else (128, 128)
        tob.w8a8_block_int8_matmul_bias_act(
            a.to(torch.int8), b.to(torch.int8), torch.ones(m, -(-k // bk), device=cuda),
            torch.ones(-(-n // bn), -(-k // bk), device=cuda), [bn, bk], out=out)
    assert torch.equal(out, want) and bool((wide[:, n:] == 7).all())
