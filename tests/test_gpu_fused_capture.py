"""The fused operators captured as a process's first calls, captured across forked streams, and called
from several threads at once."""

from __future__ import annotations

import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import tileops_b200 as tob

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
F64 = torch.float64

FIRST = """
import torch, tileops_b200 as tob
d = torch.device("cuda", 0)
m, n, k = {shape}
x = torch.randint(-3, 4, (m, k), device=d).to({dt})
w = torch.randint(-2, 3, (n, k), device=d).to({dt})
one_m = torch.ones(m, -(-k // {bk}), device=d)
one_n = torch.ones(-(-n // {bn}), -(-k // {bk}), device=d)
wt = w.t().contiguous() if {dt} == torch.float16 else w
gain = torch.ones(k, device=d).half()
want = (x.double() @ w.double().t()).half()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    {call}
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
{check}
print("captured")
"""


@pytest.mark.parametrize("call,dt,shape", [
    ("y = tob.gemm_bias_act(x, wt)", "torch.float16", (3, 512, 1024)),
    ("y = tob.gemm_bias_act(x, wt)", "torch.float16", (3, 513, 1001)),
    ("y = tob.gemm_bias_act(x, wt)", "torch.float16", (1000, 2048, 256)),
    ("y = tob.w8a8_block_int8_matmul_bias_act(x, w, one_m, one_n, [{bn}, {bk}])", "torch.int8",
     (3, 512, 1024)),
    ("y = tob.w8a8_block_int8_matmul_bias_act(x, w, one_m, one_n, [{bn}, {bk}])", "torch.int8",
     (2000, 1280, 512)),
    ("q, s = tob.add_rms_norm_group_quant(x, gain, 8, dtype=torch.int8)", "torch.float16",
     (300, 64, 512)),
])
def test_first_call_is_captured(cuda, call, dt, shape):
    check = ("assert torch.equal(y, want)" if call.startswith("y")
             else "assert torch.equal(s, tob.add_rms_norm_group_quant(x, gain, 8, dtype=torch.int8)[1])")
    code = FIRST.format(shape=shape, dt=dt, bn=128, bk=128, check=check,
                        call=call.format(bn=128, bk=128))
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                         timeout=120)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


def ints(gen, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=gen)


def test_forked_capture(cuda):
    """Two branches of a capture, each with its own operand copies, joined by a product of both."""
    gen = torch.Generator().manual_seed(2)
    a = [ints(gen, -3, 3, 20, 333).half().to(cuda) for _ in range(2)]
    b = [ints(gen, -2, 2, 333, 257).half().to(cuda) for _ in range(2)]
    want = sum(x.to(F64) @ y.to(F64) for x, y in zip(a, b)).half()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            first = tob.gemm_bias_act(a[0], b[0])
        tob.gemm_bias_act(b[1].t().contiguous(), b[1])  # work beside it
        main.wait_stream(side)
        y = tob.gemm_bias_act(a[1], b[1], residual=first)
    for _ in range(5):
        g.replay()
        assert torch.equal(y, want)


def test_threads(cuda):
    """Four threads, a stream each, through every kind of tiles at the same time."""
    gen = torch.Generator().manual_seed(3)
    w = ints(gen, -2, 2, 640, 1024)
    wh, w8 = w.half().to(cuda), w.t().contiguous().to(torch.int8).to(cuda)
    one_n = torch.ones(8, 5, device=cuda)
    xs = {m: ints(gen, -3, 3, m, 640) for m in (1, 30, 300, 2000)}
    data = {m: (x.half().to(cuda), x.to(torch.int8).to(cuda), torch.ones(m, 5, device=cuda),
                (x.double() @ w.double()).half().to(cuda)) for m, x in xs.items()}
    gain = torch.ones(640, device=cuda).half()
    norm = {m: tob.add_rms_norm_group_quant(d[0], gain, 128)[1] for m, d in data.items()}
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                for m, (xh, x8, one_m, want) in data.items():
                    ys = (tob.gemm_bias_act(xh, wh),
                          tob.w8a8_block_int8_matmul_bias_act(x8, w8, one_m, one_n, [128, 128]))
                    s = tob.add_rms_norm_group_quant(xh, gain, 128)[1]
                    if not all(torch.equal(y, want) for y in ys) or not torch.equal(s, norm[m]):
                        bad.append(m)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
