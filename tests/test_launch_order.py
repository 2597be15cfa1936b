"""Order of the stream with programmatic dependent launches. A kernel that lets its successor start
before its own predecessor has completed puts three kernels in flight, and with launch overlap on
the third may read weights that the first still writes; set_launch_overlap promises that only the
launch immediately before a call matters."""

from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

import tileops_b200 as tob

CSRC = Path(tob.__file__).resolve().parent / "csrc"
F64 = torch.float64


def code(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


@pytest.mark.parametrize("path", sorted(p for p in CSRC.glob("*.cu")
                                        if "grid_dependents_launch()" in p.read_text()),
                         ids=lambda p: p.name)
def test_successors_start_after_the_wait(path):
    """In every kernel, the wait for the previous kernel stands before the successor's start."""
    for body in code(path).split("__global__")[1:]:
        start = body.find("grid_dependents_launch()")
        if start >= 0:
            assert 0 <= body.find("grid_dependency_wait()") < start


def ints(gen, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=gen)


@pytest.fixture
def overlap():
    prev = tob.set_launch_overlap(True)
    yield
    tob.set_launch_overlap(prev)


@pytest.mark.gpu
@pytest.mark.parametrize("between", ["norm", "copies", "few_tokens", "pairs", "block_scaled"])
@pytest.mark.parametrize("reader", ["gemv", "product"])
def test_weights_written_two_launches_back(cuda, overlap, between, reader):
    """An update of w, one operator, then a product that reads w. Whole numbers: every sum is exact
    in fp32, so the result is that of the updated w, rounded once."""
    gen = torch.Generator().manual_seed(1)
    n = 4096
    w0 = ints(gen, -2, 2, n, n).half().to(cuda)
    la, lb = ints(gen, -1, 1, n, 16).half().to(cuda), ints(gen, -1, 1, 16, n).half().to(cuda)
    x = ints(gen, -1, 1, 1, n).half().to(cuda)
    m, k = {"norm": (8, 512), "copies": (4, 333), "few_tokens": (4, 512), "pairs": (2048, 64),
            "block_scaled": (2048, 256)}[between]
    y = ints(gen, -1, 1, m, k).half().to(cuda)
    v = ints(gen, -1, 1, k, 2048).half().to(cuda)
    y8, v8 = y.to(torch.int8), v.t().contiguous().to(torch.int8)
    y_s, v_s = torch.ones(m, -(-k // 128), device=cuda), torch.ones(16, -(-k // 128), device=cuda)
    ones = torch.ones(k, device=cuda).half()

    def step():
        if between == "norm":
            tob.add_rms_norm_group_quant(y, ones, 128)
        elif between == "block_scaled":
            tob.w8a8_block_int8_matmul_bias_act(y8, v8, y_s, v_s, [128, 128])
        else:
            tob.gemm_bias_act(y, v)

    w64 = w0.to(F64) + la.to(F64) @ lb.to(F64)
    want = (w64 @ x[0].to(F64) if reader == "gemv" else x.to(F64) @ w64).half()
    for _ in range(10):
        w = w0.clone()
        tob.gemm_bias_act(la, lb, residual=w, out=w)
        step()
        got = tob.gemv(w, x[0]) if reader == "gemv" else tob.gemm_bias_act(x, w)
        assert torch.equal(got, want)


@pytest.mark.parametrize("path", sorted(CSRC.glob("linear_*")) + [CSRC / "norm_quant.cu"],
                         ids=lambda p: p.name)
def test_products_with_an_epilogue_read_nothing_ahead(path):
    """No wait of these kernels is conditional on the launch-overlap switch."""
    text = code(path)
    assert "launch_overlap" not in text and "early_weights" not in text


@pytest.mark.parametrize("name", ["linear_nt_sm100.cu", "linear_pair_sm100.cu",
                                  "linear_bs_sm100.cu"])
def test_bounded_waits_start_after_the_previous_kernel(name):
    """Every role of a product's blocks waits for the previous kernel before its first bounded wait,
    so that a predecessor which runs longer than the limit does not use it up."""
    body = (CSRC / name).read_text().split("__global__")[1]
    waits = ("mbar_wait_polled(", "mbar_wait_warp(", "mbar_wait(")
    roles = [re.sub(r"//[^\n]*", "", r) for r in re.split(r"// -{20,}", body)[1:]]
    roles = [r for r in roles if any(w in r for w in waits)]
    assert len(roles) >= 3
    for r in roles:
        assert 0 <= r.find("grid_dependency_wait()") < min(r.find(w) for w in waits if w in r)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1, 4096, 4096), (40, 2048, 1000), (1000, 1024, 2048),
                                   (4, 1001, 3001)])
def test_weights_written_by_the_launch_before(cuda, overlap, m, k, n):
    """A weight handed over transposed (the call copies it first), or written by the launch just
    before the call, through the few-token and pair tiles and the aligned copies."""
    gen = torch.Generator().manual_seed(m)
    a = ints(gen, -2, 2, m, k).half().to(cuda)
    wt = ints(gen, -2, 2, n, k).half().to(cuda)
    want = (a.to(F64) @ wt.to(F64).t()).half()
    want2 = (a.to(F64) @ (wt.to(F64) + 1).t()).half()
    for _ in range(10):
        assert torch.equal(tob.gemm_bias_act(a, wt.t()), want)
        w = wt.t().contiguous()
        w.add_(1)
        assert torch.equal(tob.gemm_bias_act(a, w), want2)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("block", [[1, 4096], [128, 128]])
@pytest.mark.parametrize("m", [1, 40, 600])
def test_codes_written_by_the_launch_before(cuda, overlap, codes, block, m):
    gen = torch.Generator().manual_seed(m)
    k, n = 4096, 1536
    a, w = ints(gen, -2, 2, m, k).to(codes).to(cuda), ints(gen, -3, 3, n, k).to(codes).to(cuda)
    a_s = torch.ones(m, -(-k // block[1]), device=cuda)
    b_s = torch.ones(-(-n // block[0]), -(-k // block[1]), device=cuda)
    op = (tob.w8a8_block_int8_matmul_bias_act if codes == torch.int8
          else tob.w8a8_block_fp8_matmul_bias_act)
    want = (a.to(torch.float32).to(F64) @ w.to(torch.float32).to(F64).t()).float()
    for _ in range(10):
        v = torch.zeros_like(w)
        v.copy_(w)
        assert torch.equal(op(a, v, a_s, b_s, block, output_dtype=torch.float32), want)
