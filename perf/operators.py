"""Cases, inputs and plain forms of the 8-bit training operators in ``elf_b200.ops.fp8``.

A block-scaled tensor holds e4m3 values and one power-of-two scale per block of 128 columns,
stored as its biased exponent: ``value = data * 2^(scale - 127)``.  Activations and gradients
have a scale for each row and 128 columns, weights one for each 128 x 128 tile.  The scale is
the smallest power of two that brings the block's largest finite magnitude to at most 448;
what is not finite becomes NaN and has no part in it.

Operators (``case["op"]``):

``checkpoint``  an activation kept in 8 bits from the forward to the backward pass: quantised,
                then restored to 16 bits
``norm``        RMSNorm, with or without the residual's addition, whose output is block-scaled
``linear``      the products of a linear layer on block-scaled operands (``case["pass"]``):
                ``forward`` Y = X W^T, ``input_grad`` dX = dY W, ``weight_grad`` dW = dY^T X
``ffn``         gated feed-forward block, y = (silu(x Wg^T) * (x Wu^T)) Wd^T, forward alone or
                with its backward pass from 8-bit checkpoints
"""

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------- cases


def listed():
    return [
        # one micro-batch of the smallest decoder configuration: launch latency
        {"name": "checkpoint 128x256", "op": "checkpoint", "rows": 128, "cols": 256, "dtype": "bf16"},
        # hidden width of the 1.3B configuration, a last token dropped: ragged rows, fp16 training
        {"name": "checkpoint 2047x5504 fp16", "op": "checkpoint", "rows": 2047, "cols": 5504, "dtype": "fp16"},
        # gate and up activations of one 8B micro-batch, the largest tensor a layer keeps
        {"name": "checkpoint 4096x28672", "op": "checkpoint", "rows": 4096, "cols": 28672, "dtype": "bf16"},
        # a single token
        {"name": "norm 1x4096", "op": "norm", "rows": 1, "dim": 4096, "residual": True},
        # second norm of a decoder layer, 8B shape
        {"name": "norm 4096x4096 residual", "op": "norm", "rows": 4096, "dim": 4096, "residual": True},
        # first norm of a layer, 13B width, ragged micro-batch
        {"name": "norm 1000x5120", "op": "norm", "rows": 1000, "dim": 5120, "residual": False},
        # down projection of a few tokens: bound by the weight's bytes
        {"name": "linear forward 16 rows", "op": "linear", "pass": "forward", "m": 16, "n": 4096, "k": 14336},
        # down projection of one 8B micro-batch
        {"name": "linear forward 4096 rows", "op": "linear", "pass": "forward", "m": 4096, "n": 4096, "k": 14336},
        # input gradient of the 1.3B gate/up projection, ragged tokens
        {"name": "linear input grad 2047 rows", "op": "linear", "pass": "input_grad", "m": 2047, "n": 11008, "k": 2048},
        # weight gradient of the 1.3B down projection, ragged tokens
        {"name": "linear weight grad 2047 rows", "op": "linear", "pass": "weight_grad", "m": 2047, "n": 2048, "k": 5504},
        # the smallest decoder configuration's block, forward alone (validation)
        {"name": "ffn forward 128 tokens", "op": "ffn", "m": 128, "d": 256, "f": 512, "train": False},
        # one 8B micro-batch, forward and backward
        {"name": "ffn train 4096 tokens", "op": "ffn", "m": 4096, "d": 4096, "f": 14336, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("checkpoint", "norm", "linear", "ffn"))
    if op == "checkpoint":
        cols = _log(rng, 1, 28672)
        rows = _log(rng, 1, min(16384, 4096 * 28672 // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 16384), "dim": 8 * _log(rng, 2, 1024), "residual": rng.random() < 0.5}
    if op == "linear":
        m, n = _log(rng, 1, 8192), _log(rng, 16, 28672)
        k = _log(rng, 16, min(14336, 4096 * 28672 * 4096 // (m * n)))
        return {"op": op, "pass": rng.choice(("forward", "input_grad", "weight_grad")), "m": m, "n": n, "k": k}
    return {"op": op, "m": _log(rng, 1, 4096), "d": 16 * _log(rng, 2, 256), "f": 128 * _log(rng, 1, 112), "train": rng.random() < 0.6}


# ---------------------------------------------------------------------------------- inputs


def _activations(gen, rows, cols, dtype=torch.float32):
    """Normal values with a few large channels, as the residual stream of a decoder has them."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    loud = torch.rand(cols, device="cuda", generator=gen) < 0.005
    return (x * (1 + 19 * loud)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    op = case["op"]
    state = {"case": dict(case)}
    if op == "checkpoint":
        state["x"] = _activations(gen, case["rows"], case["cols"], DTYPES[case["dtype"]])
    elif op == "norm":
        state["x"] = _activations(gen, case["rows"], case["dim"], torch.bfloat16)
        state["residual"] = _activations(gen, case["rows"], case["dim"], torch.bfloat16) if case["residual"] else None
        state["gain"] = (1 + 0.1 * randn(case["dim"])).to(torch.bfloat16)
    elif op == "linear":
        # block-scaled operands are what a program has in hand here: the norm, the forward pass
        # or the optimizer step before left them
        m, n, k = case["m"], case["n"], case["k"]
        if case["pass"] != "input_grad":
            state["x"] = _quantize(_activations(gen, m, k, torch.bfloat16), 1)
        if case["pass"] != "forward":
            state["dy"] = _quantize((1e-3 * randn(m, n)).to(torch.bfloat16), 1)
        if case["pass"] != "weight_grad":
            state["w"] = _quantize((0.02 * randn(n, k)).to(torch.bfloat16), BLOCK)
    else:
        m, d, f = case["m"], case["d"], case["f"]
        state["x"] = randn(m, d).to(torch.bfloat16)
        # the weights and the 8-bit copies made of them after the last optimizer step
        for name, rows, cols in (("gate_up", 2 * f, d), ("down", d, f)):
            w = (0.02 * randn(rows, cols)).to(torch.bfloat16)
            state[name], state[name + "_q"] = w, _quantize(w, BLOCK)
        if case["train"]:
            state["dy"] = (1e-3 * randn(m, d)).to(torch.bfloat16)
            for name in ("x", "gate_up", "down"):
                state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------------- plain forms


def _blocks(x, block_rows):
    """``[rows, cols]`` padded with zeros and seen as ``[row blocks, block_rows, col blocks, 128]``."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    return x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // BLOCK, BLOCK)


def _spread(scale, rows, cols, block_rows):
    """The factor of every element for a matrix of exponents."""
    factor = torch.ldexp(torch.ones_like(scale, dtype=torch.float32), scale.to(torch.int32) - 127)
    return factor.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _quantize(x, block_rows):
    rows, cols = x.shape
    x = x.float()
    amax = torch.where(torch.isfinite(x), x.abs(), 0.0)
    amax = _blocks(amax, block_rows).amax((1, 3))
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    scale = exponent - 9 + (mantissa > 0.875).to(exponent.dtype) + 127  # 448 = 0.875 * 2^9
    scale = torch.where(amax > 0, scale, 1).clamp(1, 254).to(torch.uint8)
    v = x / _spread(scale, rows, cols, block_rows)
    v = torch.where(torch.isfinite(x), v.clamp(-448.0, 448.0), float("nan"))
    return v.to(torch.float8_e4m3fn), scale, block_rows


def _values(q):
    data, scale, block_rows = q
    return data.float() * _spread(scale, data.shape[0], data.shape[1], block_rows)


def _plain_norm(x, residual, gain, eps=1e-5):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + eps)
    return h, hf * rstd * gain.float()


def _plain_ffn(x, gate_up_q, down_q, dy):
    f = down_q[0].shape[1]
    wgu, wd = _values(gate_up_q), _values(down_q)
    xv = _values(_quantize(x, 1))
    gu = xv @ wgu.T
    sig = 1 / (1 + torch.exp(-gu[:, :f]))
    act = _values(_quantize(gu[:, :f] * sig * gu[:, f:], 1))
    y = (act @ wd.T).to(x.dtype)
    if dy is None:
        return {"y": y}
    gu = _values(_quantize(gu, 1))  # what is kept for the backward pass
    gate, up = gu[:, :f], gu[:, f:]
    dact = _values(_quantize(dy, 1)) @ wd
    sig = 1 / (1 + torch.exp(-gate))
    dgu = torch.cat([dact * up * sig * (1 + gate * (1 - sig)), dact * gate * sig], 1)
    dgu = _values(_quantize(dgu, 1))
    dx = dgu @ wgu
    return {"y": y, "dx": dx.to(x.dtype), "dw_gate_up": (dgu.T @ xv).to(x.dtype), "dw_down": (dy.float().T @ act).to(x.dtype)}


def _plain(state):
    case = state["case"]
    if case["op"] == "checkpoint":
        return _values(_quantize(state["x"], 1)).to(torch.bfloat16)
    if case["op"] == "norm":
        h, y = _plain_norm(state["x"], state["residual"], state["gain"])
        out = {"y": _values(_quantize(y, 1)).to(torch.bfloat16)}
        if state["residual"] is not None:
            out["h"] = h
        return out
    if case["op"] == "linear":
        if case["pass"] == "forward":
            y = _values(state["x"]) @ _values(state["w"]).T
        elif case["pass"] == "input_grad":
            y = _values(state["dy"]) @ _values(state["w"])
        else:
            y = _values(state["dy"]).T @ _values(state["x"])
        return y.to(torch.bfloat16)
    with torch.no_grad():
        return _plain_ffn(state["x"], state["gate_up_q"], state["down_q"], state.get("dy"))


# ---------------------------------------------------------------------------------- the framework's operators


def _own(state):
    from elf_b200.ops import fp8

    case = state["case"]
    if case["op"] == "checkpoint":
        return fp8.dequantize(fp8.quantize(state["x"]), torch.bfloat16)
    if case["op"] == "norm":
        if state["residual"] is None:
            q, _ = fp8.rms_norm(state["x"], state["gain"], 1e-5)
            return {"y": fp8.dequantize(q, torch.bfloat16)}
        q, _, h = fp8.add_rms_norm(state["x"], state["residual"], state["gain"], 1e-5)
        return {"y": fp8.dequantize(q, torch.bfloat16), "h": h}
    if case["op"] == "linear":
        held = {name: fp8.BlockScaled(*state[name]) for name in ("x", "dy", "w") if name in state}
        if case["pass"] == "forward":
            return fp8.linear_forward(held["x"], held["w"])
        if case["pass"] == "input_grad":
            return fp8.linear_input_grad(held["dy"], held["w"])
        return fp8.linear_weight_grad(held["dy"], held["x"])
    weights = {"gate_up_q": fp8.BlockScaled(*state["gate_up_q"]), "down_q": fp8.BlockScaled(*state["down_q"])}
    if not case["train"]:
        with torch.no_grad():
            return {"y": fp8.gated_ffn(state["x"], state["gate_up"], state["down"], **weights)}
    leaves = [state["x"], state["gate_up"], state["down"]]
    y = fp8.gated_ffn(*leaves, **weights)
    dx, dgu, dd = torch.autograd.grad(y, leaves, state["dy"])
    return {"y": y.detach(), "dx": dx, "dw_gate_up": dgu, "dw_down": dd}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "checkpoint":
        n, size = case["rows"] * case["cols"], {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        kept = n + case["rows"] * -(-case["cols"] // BLOCK)
        return {"bytes": n * size + 2 * kept + 2 * n, "flops": 0}  # read, kept in 8 bits (written, read again), restored
    if op == "norm":
        n = case["rows"] * case["dim"]
        kept = n + case["rows"] * -(-case["dim"] // BLOCK)
        return {"bytes": n * (6 if case["residual"] else 2) + 2 * kept + 2 * n + 2 * case["dim"], "flops": 0}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        read = {"forward": m * k + n * k, "input_grad": m * n + n * k, "weight_grad": m * n + m * k}[case["pass"]]
        wrote = {"forward": m * n, "input_grad": m * k, "weight_grad": n * k}[case["pass"]]
        return {"bytes": read + 2 * wrote, "flops": 2 * m * n * k}
    m, d, f = case["m"], case["d"], case["f"]
    flops = 2 * m * d * 3 * f
    if not case["train"]:
        return {"bytes": 2 * m * d + 3 * d * f + 2 * m * d, "flops": flops}
    return {"bytes": 2 * (2 * m * d) + 3 * d * f + 2 * (2 * m * d) + 2 * 3 * d * f, "flops": 3 * flops}


# ---------------------------------------------------------------------------------- the definition, in 64 bits


def _held64(x, block_rows=1):
    """The values a block-scaled tensor stands for, from the definition: for each block the
    smallest power of two s with max|x| <= 448 s, each value rounded to e4m3 (four significant
    bits, steps of 2^-9 below 2^-6, ties to even) in units of s."""
    x = x.double()
    rows, cols = x.shape
    pad_r, pad_c = -rows % block_rows, -cols % BLOCK
    full = torch.zeros(rows + pad_r, cols + pad_c, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    tiles = full.reshape(-1, block_rows, full.shape[1] // BLOCK, BLOCK).transpose(1, 2)
    top = tiles.abs().flatten(2).amax(2)
    power = torch.ceil(torch.log2(torch.where(top > 0, top / 448, 2.0**-126)))
    power = power + (448 * torch.exp2(power) < top) - (448 * torch.exp2(power - 1) >= top).double()  # next to a border the logarithm may be off
    s = torch.exp2(power.clamp(-126, 127))[:, :, None, None]
    u = tiles / s
    grid = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0**-6))) - 3)
    v = torch.round(u / grid) * grid * s
    return v.transpose(1, 2).reshape(full.shape)[:rows, :cols]


def _double(q):
    data, scale, block_rows = q
    rows, cols = data.shape
    r = torch.arange(rows, device=data.device) // block_rows
    c = torch.arange(cols, device=data.device) // BLOCK
    return data.double() * torch.exp2(scale.double() - 127)[r[:, None], c[None, :]]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "checkpoint":
            return _held64(state["x"])
        if op == "norm":
            h = state["x"].double()
            out = {}
            if state["residual"] is not None:
                h = (h + state["residual"].double()).to(torch.bfloat16).double()
                out["h"] = h
            y = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + 1e-5) * state["gain"].double()
            out["y"] = _held64(y)
            return out
        if op == "linear":
            if case["pass"] == "forward":
                return torch.einsum("mk,nk->mn", _double(state["x"]), _double(state["w"]))
            if case["pass"] == "input_grad":
                return torch.einsum("mn,nk->mk", _double(state["dy"]), _double(state["w"]))
            return torch.einsum("mn,mk->nk", _double(state["dy"]), _double(state["x"]))
        x, wgu, wd = _held64(state["x"]), _double(state["gate_up_q"]), _double(state["down_q"])
        f = case["f"]
        gate, up = torch.einsum("mk,nk->mn", x, wgu[:f]), torch.einsum("mk,nk->mn", x, wgu[f:])
        act = _held64(gate * torch.sigmoid(gate) * up)
        out = {"y": torch.einsum("mk,nk->mn", act, wd)}
        if not case["train"]:
            return out
        gate, up, dy = _held64(gate), _held64(up), state["dy"].double()
        dact = torch.einsum("mn,nk->mk", _held64(state["dy"]), wd)
        sig = torch.sigmoid(gate)
        dgate = _held64(dact * up * (sig + gate * sig * (1 - sig)))
        dup = _held64(dact * gate * sig)
        out["dx"] = torch.einsum("mn,nk->mk", dgate, wgu[:f]) + torch.einsum("mn,nk->mk", dup, wgu[f:])
        out["dw_gate_up"] = torch.cat([torch.einsum("mn,mk->nk", dgate, x), torch.einsum("mn,mk->nk", dup, x)])
        out["dw_down"] = torch.einsum("mn,mk->nk", dy, act)
        return out
