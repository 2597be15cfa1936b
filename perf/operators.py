"""Cases of the fused norm + quantiser and of the matrix products with an epilogue, each in two
forms: elementary torch operations in fp32 (``own`` false) and this library's calls (``own`` true).

  norm   h = x + r;  y = h / sqrt(mean(h^2) + eps) * w;  per group of columns s = max|y| / qmax and
         the 8-bit codes of y / s; h is returned as the next residual
  dense  C = act(A @ B + bias) + residual                     A [M, K], B [K, N], 16-bit
  w8a8   C = act(sum_kb (A_kb @ B_kb^T) * a_s * b_s + bias) + residual
         A [M, K], B [N, K] in int8 or e4m3, per-token x per-channel or 128 x 128 block scales
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}
_EPS, _QEPS = 1e-6, 1e-10


# ------------------------------------------------------------------ cases
def _norm(name, rows, cols, group, dt, codes, residual=True):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "group": group, "dt": dt,
            "codes": codes, "residual": residual}


def _dense(name, m, n, k, dt, bias=False, act="none", residual=False):
    return {"name": name, "op": "dense", "m": m, "n": n, "k": k, "dt": dt, "bias": bias,
            "act": act, "residual": residual}


def _w8a8(name, m, n, k, codes, scales, dt, bias=False, act="none", residual=False):
    return {"name": name, "op": "w8a8", "m": m, "n": n, "k": k, "codes": codes, "scales": scales,
            "dt": dt, "bias": bias, "act": act, "residual": residual}


def listed():
    return [
        # one token of a decode step entering a layer of width 4096: latency
        _norm("norm_token", 1, 4096, 128, "bf16", "e4m3"),
        # a batch of decode tokens, int8 with one scale per token (the INT8 layer's input form)
        _norm("norm_batch_int8", 256, 11008, 11008, "f16", "int8"),
        # a prefill of 8192 tokens at width 8192: bandwidth
        _norm("norm_prefill", 8192, 8192, 128, "bf16", "e4m3"),
        # one token through an unquantised 4096 x 4096 linear
        _dense("dense_token", 1, 4096, 4096, "f16", bias=True, act="silu"),
        # a decode batch through a down projection added to the residual stream
        _dense("dense_batch", 16, 4096, 14336, "bf16", residual=True),
        # a prefill through the 28672-wide up projection
        _dense("dense_prefill", 2048, 28672, 8192, "bf16", bias=True, act="gelu"),
        # odd sizes in every dimension: an adapter or head whose widths are no multiples of anything
        _dense("dense_odd", 777, 2049, 1531, "f16", bias=True, act="relu", residual=True),
        # one token, block-scaled FP8 weights
        _w8a8("fp8_block_token", 1, 7168, 7168, "e4m3", "block", "bf16", residual=True),
        # the INT8 layer at 256 tokens
        _w8a8("int8_layer", 256, 11008, 4096, "int8", "channel", "bf16", bias=True, act="silu"),
        # block-scaled FP8 prefill
        _w8a8("fp8_block_prefill", 4096, 7168, 7168, "e4m3", "block", "bf16", residual=True),
        # the FP8 layer at 8192 tokens, everything in the epilogue
        _w8a8("fp8_layer", 8192, 8192, 8192, "e4m3", "channel", "bf16", bias=True, act="gelu",
              residual=True),
        # a small ragged int8 product
        _w8a8("int8_odd", 37, 1003, 2049, "int8", "channel", "f16", bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    """Log-uniform in [lo, hi]; a multiple of `step` two times out of three, else any value."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 1 / 3 else max(step, v // step * step)


def draw(rng):
    op = rng.choice(["norm", "dense", "w8a8"])
    dt = rng.choice(["bf16", "f16"])
    if op == "norm":
        codes = rng.choice(["e4m3", "int8"])
        rows = _log(rng, 1, 8192)
        group = rng.choice([64, 128, 128, 0])  # 0: one scale per token
        cols = _size(rng, 256, 16384, 128) if group == 0 else _log(rng, 256, 16384) // group * group
        while rows * cols > 8192 * 8192:
            rows = rows // 2
        return {k: v for k, v in _norm("", rows, cols, group or cols, dt, codes,
                                       residual=rng.random() < 0.75).items() if k != "name"}
    m = _log(rng, 1, 8192)
    n, k = _size(rng, 64, 28672, 64), _size(rng, 64, 14336, 128)
    while 2.0 * m * n * k > 1.0e12:
        m = m // 2
    epi = {"bias": rng.random() < 0.5, "act": rng.choice(["none", "relu", "silu", "gelu"]),
           "residual": rng.random() < 0.5}
    if op == "dense":
        c = _dense("", m, n, k, dt, **epi)
    else:
        c = _w8a8("", m, n, k, rng.choice(["e4m3", "int8"]), rng.choice(["channel", "block"]), dt,
                  **epi)
    return {key: v for key, v in c.items() if key != "name"}


# ------------------------------------------------------------------ inputs
def _blocks(n):
    return -(-n // 128)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(*shape, generator=g, device="cuda")

    dt = _DT[case["dt"]]
    st = {"case": dict(case)}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # activations with a few loud channels, as a residual stream has them
        loud = 1.0 + 15.0 * (torch.rand(cols, generator=g, device="cuda") < 0.004)
        st["x"] = normal(rows, cols).to(dt)
        st["r"] = (normal(rows, cols) * 2.0 * loud).to(dt) if case["residual"] else None
        st["w"] = (1.0 + 0.2 * normal(cols)).to(dt)
        return st
    m, n, k = case["m"], case["n"], case["k"]
    st["bias"] = normal(n).to(dt) if case["bias"] else None
    st["res"] = normal(m, n).to(dt) if case["residual"] else None
    if case["op"] == "dense":
        st["a"] = normal(m, k).to(dt)
        st["b"] = normal(k, n).mul_(k ** -0.5).to(dt)
        return st

    def codes(rows):
        v = normal(rows, k)
        if case["codes"] == "int8":
            return v.mul_(40.0).round_().clamp_(-127, 127).to(torch.int8)
        return v.mul_(100.0).clamp_(-448, 448).to(torch.float8_e4m3fn)

    std = 40.0 if case["codes"] == "int8" else 100.0
    kt = 1 if case["scales"] == "channel" else _blocks(k)
    nt = n if case["scales"] == "channel" else _blocks(n)
    st["a"], st["b"] = codes(m), codes(n)
    st["a_s"] = uniform(0.5, 1.5, m, kt) / std
    st["b_s"] = uniform(0.5, 1.5, nt, kt) / (std * k ** 0.5)
    st["block"] = [1, k] if case["scales"] == "channel" else [128, 128]
    return st


# ------------------------------------------------------------------ plain forms
def _act(v, act):
    if act == "relu":
        return torch.clamp(v, min=0.0)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    return v


def _epilogue(acc, st):
    if st["bias"] is not None:
        acc = acc + st["bias"].float()
    acc = _act(acc, st["case"]["act"])
    if st["res"] is not None:
        acc = acc + st["res"].float()
    return acc.to(_DT[st["case"]["dt"]])


def _plain_norm(st):
    c = st["case"]
    h = st["x"].float()
    if st["r"] is not None:
        h = h + st["r"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS) * st["w"].float()
    yg = y.view(c["rows"], c["cols"] // c["group"], c["group"])
    qmax = 448.0 if c["codes"] == "e4m3" else 127.0
    s = torch.clamp(yg.abs().amax(-1, keepdim=True), min=_QEPS) / qmax
    z = yg / s
    if c["codes"] == "e4m3":
        q = torch.clamp(z, -448.0, 448.0).to(torch.float8_e4m3fn)
    else:
        q = torch.clamp(torch.round(z), -128.0, 127.0).to(torch.int8)
    out = (q.view(c["rows"], c["cols"]), s.squeeze(-1))
    return out if st["r"] is None else (*out, h.to(_DT[c["dt"]]))


def _spread(s, block, size, dim):
    """Block scales repeated over their blocks, cut to `size`."""
    return s.repeat_interleave(block, dim).narrow(dim, 0, size)


def _plain_w8a8(st):
    c = st["case"]
    a, b = st["a"].float(), st["b"].float()
    if c["scales"] == "channel":
        acc = (a @ b.t()) * (st["a_s"] * st["b_s"].t())
    else:
        a = a * _spread(st["a_s"], 128, c["k"], 1)
        b = b * _spread(_spread(st["b_s"], 128, c["n"], 0), 128, c["k"], 1)
        acc = a @ b.t()
    return _epilogue(acc, st)


# ------------------------------------------------------------------ one pass
def _values(outs, case):
    """int8 codes as the numbers they are; e4m3 tensors are numbers already."""
    q = outs[0] if case["codes"] == "e4m3" else outs[0].to(_DT[case["dt"]])
    return {"q": q, "s": outs[1], **({"h": outs[2]} if len(outs) > 2 else {})}


def _own(st):
    import tileops_b200 as tob

    c = st["case"]
    if c["op"] == "norm":
        codes = torch.float8_e4m3fn if c["codes"] == "e4m3" else torch.int8
        return tob.add_rms_norm_group_quant(st["x"], st["w"], c["group"], st["r"], eps=_EPS,
                                            dtype=codes, quant_eps=_QEPS)
    act = None if c["act"] == "none" else c["act"]
    if c["op"] == "dense":
        return tob.gemm_bias_act(st["a"], st["b"], st["bias"], act=act, residual=st["res"])
    op = (tob.w8a8_block_int8_matmul_bias_act if c["codes"] == "int8"
          else tob.w8a8_block_fp8_matmul_bias_act)
    return op(st["a"], st["b"], st["a_s"], st["b_s"], st["block"], st["bias"], act=act,
              residual=st["res"], output_dtype=_DT[c["dt"]])


def run(st):
    c = st["case"]
    if own:
        out = _own(st)
    elif c["op"] == "norm":
        out = _plain_norm(st)
    elif c["op"] == "dense":
        out = _epilogue(st["a"].float() @ st["b"].float(), st)
    else:
        out = _plain_w8a8(st)
    return _values(out, c) if c["op"] == "norm" else out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "norm":
        e = case["rows"] * case["cols"]
        io = 2 * (3 if case["residual"] else 1) + 1
        scales = 4 * case["rows"] * (case["cols"] // case["group"])
        return {"bytes": e * io + scales + 2 * case["cols"], "flops": 8 * e}
    m, n, k = case["m"], case["n"], case["k"]
    b = 2 * m * n * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0)
    if case["op"] == "dense":
        b += 2 * (m * k + k * n)
    else:
        b += m * k + n * k
        b += 4 * (m + n) if case["scales"] == "channel" else 4 * _blocks(k) * (m + _blocks(n))
    return {"bytes": b, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_codes(y, qmax, kind):
    s = y.abs().amax(-1, keepdim=True).clamp(min=_QEPS) / qmax
    z = (y / s).clamp(-qmax, qmax)
    if kind == "int8":
        return torch.round(z), s
    # e4m3: 3 mantissa bits above 2^-6, steps of 2^-9 below; ties to even
    e = torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3.0)
    return torch.round(z / step) * step, s


def exact(case, seed):
    st = prepare(case, seed)
    d = {k: v.double() for k, v in st.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "norm":
        h = d["x"] + d["r"] if case["residual"] else d["x"]
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + _EPS) * d["w"]
        y = y.reshape(case["rows"], -1, case["group"])
        q, s = _exact_codes(y, 448.0 if case["codes"] == "e4m3" else 127.0, case["codes"])
        out = {"q": q.reshape(case["rows"], case["cols"]), "s": s.squeeze(-1)}
        return {**out, "h": h} if case["residual"] else out
    if case["op"] == "dense":
        v = d["a"] @ d["b"]
    elif case["scales"] == "channel":
        v = (d["a"] @ d["b"].T) * d["a_s"] * d["b_s"].T
    else:
        ka = torch.arange(case["k"], device="cuda") // 128
        nb = torch.arange(case["n"], device="cuda") // 128
        v = (d["a"] * d["a_s"][:, ka]) @ (d["b"] * d["b_s"][nb][:, ka]).T
    if case["bias"]:
        v = v + d["bias"]
    if case["act"] == "relu":
        v = v.clamp(min=0)
    elif case["act"] == "silu":
        v = v * torch.sigmoid(v)
    elif case["act"] == "gelu":
        v = 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v + d["res"] if case["residual"] else v
