"""8-bit operators on the CPU: their plain forms against the definition, gradients, refusals, the split-backward
layer and the Llama option."""

import copy

import pytest
import torch

from elf_b200 import Pipeline
from elf_b200.models.llama import LlamaConfig, LlamaMLPBlock, build_llama_stages, llama_loss_fn
from elf_b200.ops import fp8
from elf_b200.ops.fp8 import BlockScaled
from elf_b200.zb_utils import LinearDW, LinearFP8DW, replace_layer_with_layer_dw, replace_linear_with_linear_fp8

from .dist_utils import _free_port
from .fp8_oracle import held, product_bound, values

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def rand(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 130), (130, 256), (5, 1000)])
def test_plain_quantize_is_exact(rows, cols, dtype):
    x = rand(rows, cols, dtype=dtype, seed=rows) * 30
    x[0, 0] = float("inf")
    if cols > 1:
        x[-1, 1] = float("nan")
        x[:, 2::3] *= 1e-3
    for make, block_rows in ((fp8.quantize, 1), (fp8.quantize_weight, 128)):
        q = make(x)
        want, exps = held(x, block_rows)
        assert torch.equal(q.scale, exps)
        assert torch.equal(values(q).isnan(), want.isnan()) and torch.equal(values(q).nan_to_num(0.0), want.nan_to_num(0.0))
        assert torch.equal(q.dequantize(torch.float32).double().nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (7, 130, 140), (40, 64, 300)])
def test_plain_products(m, n, k):
    x, dy, w = fp8.quantize(rand(m, k)), fp8.quantize(rand(m, n, seed=1)), fp8.quantize_weight(rand(n, k, seed=2))
    for got, a, b in ((fp8.linear_forward(x, w), values(x), values(w).T), (fp8.linear_input_grad(dy, w), values(dy), values(w)),
                      (fp8.linear_weight_grad(dy, x), values(dy).T, values(x))):
        assert got.dtype == torch.bfloat16 and ((got.double() - a @ b).abs() <= product_bound(a, b, torch.bfloat16)).all()


def test_gate_gradient_formula_against_differences():
    """d silu(g) u as the operators form it, against central differences in 64 bits."""
    g, u, d = (rand(64, seed=s).double() * 4 for s in (0, 1, 2))
    f = lambda g, u: (torch.nn.functional.silu(g) * u * d).sum()
    s = torch.sigmoid(g)
    for i in range(64):
        e = torch.zeros(64, dtype=torch.float64)
        e[i] = 1e-5
        # the second differences' error: h^2/6 of a third derivative below 1, plus rounding 2^-52 / h
        assert abs((f(g + e, u) - f(g - e, u)) / 2e-5 - d[i] * u[i] * s[i] * (1 + g[i] * (1 - s[i]))) < 1e-8
        assert abs((f(g, u + e) - f(g, u - e)) / 2e-5 - d[i] * g[i] * s[i]) < 1e-8


def test_linear_gradients_are_those_of_the_rounded_operands():
    x, w, b = rand(2, 9, 200).requires_grad_(), rand(72, 200, seed=1).requires_grad_(), rand(72, seed=2).requires_grad_()
    dy = rand(2, 9, 72, seed=3)
    y = fp8.linear(x, w, b)
    y.backward(dy)
    xq, wq, dyq = (held(t.detach().reshape(-1, t.shape[-1]), r)[0] for t, r in ((x, 1), (w, 128), (dy, 1)))
    for got, a, m in ((x.grad, dyq, wq), (w.grad, dyq.T, xq)):
        assert ((got.reshape(-1, got.shape[-1]).double() - a @ m).abs() <= product_bound(a, m, torch.float32)).all()
    assert ((y.detach().view(18, 72).double() - (xq @ wq.T + b.detach().double())).abs() <= product_bound(xq, wq.T, torch.float32) + 1e-6).all()
    # 18 fp32 additions
    assert ((b.grad.double() - dy.double().sum((0, 1))).abs() <= 18 * 2.0**-24 * dy.double().abs().sum((0, 1))).all()
    # with the copy the program keeps: the same
    x2, w2 = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    y2 = fp8.linear(x2, w2, b.detach(), fp8.quantize_weight(w.detach()))
    y2.backward(dy)
    assert torch.equal(y2, y) and torch.equal(x2.grad, x.grad) and torch.equal(w2.grad, w.grad)


def test_gated_ffn_matches_its_parts_and_saves_8_bits():
    x, wg, wd = rand(12, 144, seed=4).requires_grad_(), (rand(512, 144, seed=5) * 0.1).requires_grad_(), (rand(80, 256, seed=6) * 0.1).requires_grad_()
    dy = rand(12, 80, seed=7)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        y = fp8.gated_ffn(x, wg, wd)
    y.backward(dy)
    weights = {wg.data_ptr(), wd.data_ptr()}
    activations = [t for t in kept if t.data_ptr() not in weights]
    assert all(t.element_size() == 1 for t in activations)
    assert sum(t.numel() for t in activations if t.dtype != torch.uint8) == 12 * (144 + 3 * 256)
    gq, dq = fp8.quantize_weight(wg.detach()), fp8.quantize_weight(wd.detach())
    xq = fp8.quantize(x.detach())
    act, gu = fp8.gated_forward(xq, gq)
    assert torch.equal(y, fp8.linear_forward(act, dq, out_dtype=torch.float32))
    dgu = fp8.gated_backward(fp8.quantize(dy), dq, gu)
    assert torch.equal(x.grad, fp8.linear_input_grad(dgu, gq, torch.float32))
    assert torch.equal(wg.grad, fp8.linear_weight_grad(dgu, xq, out_dtype=torch.float32))
    assert torch.equal(wd.grad, fp8.linear_weight_grad(dy, act, out_dtype=torch.float32))
    with torch.no_grad():
        assert torch.equal(fp8.gated_ffn(x, wg, wd), y)


def test_weight_gradient_operands():
    """Plain operands enter with their own type's bits; a push takes only what is one bf16 matrix."""
    x = rand(40, 30)
    for dtype in DTYPES:
        dy = rand(40, 20, dtype=dtype, seed=1)
        a, b = dy.double().T, x.double()
        assert ((fp8.linear_weight_grad(dy, x, out_dtype=torch.float32).double() - a @ b).abs() <= product_bound(a, b, torch.float32)).all()
    with pytest.raises(TypeError, match="dy must be"):
        fp8.linear_weight_grad(rand(40, 20).double(), x)
    with pytest.raises(ValueError, match="push takes"):
        fp8.linear_weight_grad(rand(40, 20), x.bfloat16(), out=torch.zeros(20, 30, dtype=torch.bfloat16), push={"tag": 1})
    with pytest.raises(ValueError, match="CUDA operands that have elements"):
        fp8.linear_weight_grad(fp8.quantize(rand(40, 20)), fp8.quantize(x), out=torch.zeros(20, 30, dtype=torch.bfloat16), push={"tag": 1})


def test_only_requested_gradients():
    x, w = rand(4, 64), rand(8, 64).requires_grad_()
    fp8.linear(x, w).sum().backward()
    assert w.grad is not None and x.grad is None
    x, wg, wd = rand(4, 64).requires_grad_(), rand(256, 64), rand(8, 128)
    fp8.gated_ffn(x, wg, wd).sum().backward()
    assert x.grad is not None
    wd.requires_grad_()
    fp8.gated_ffn(x.detach(), wg, wd).sum().backward()
    assert wd.grad is not None


def test_refusals():
    data, scale = torch.zeros(4, 200).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8)
    q, w = BlockScaled(data, scale), fp8.quantize_weight(rand(256, 200))
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        BlockScaled(torch.zeros(4, 200), scale)
    with pytest.raises(ValueError, match="block_rows"):
        BlockScaled(data, scale, 64)
    with pytest.raises(ValueError, match="expected exponents"):
        BlockScaled(data, scale[:, :1])
    with pytest.raises(ValueError, match="expected exponents"):
        BlockScaled(data, scale, 128)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        fp8.quantize(torch.zeros(4, 4, dtype=torch.int32))
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        fp8.quantize(torch.zeros(4, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="at least one dimension"):
        fp8.quantize(torch.tensor(1.0))
    with pytest.raises(ValueError, match="matrix"):
        fp8.quantize_weight(torch.zeros(2, 3, 4))
    with pytest.raises(TypeError, match="not torch.float64"):
        fp8.dequantize(q, torch.float64)
    with pytest.raises(ValueError, match="out does not match"):
        fp8.dequantize(q, out=torch.empty(4, 100))
    with pytest.raises(ValueError, match="reduction lengths"):
        fp8.linear_forward(fp8.quantize(rand(4, 199)), w)
    with pytest.raises(ValueError, match="scaled by rows"):
        fp8.linear_forward(w, w)
    with pytest.raises(ValueError, match="bias"):
        fp8.linear_forward(q, w, torch.zeros(3))
    with pytest.raises(TypeError, match="products come in"):
        fp8.linear_forward(q, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="tiles of 128 x 128"):
        fp8.linear_input_grad(fp8.quantize(rand(4, 256)), fp8.quantize(rand(256, 200)))
    with pytest.raises(ValueError, match="numbers of rows"):
        fp8.linear_weight_grad(q, fp8.quantize(rand(5, 8)))
    with pytest.raises(ValueError, match="scaled by rows"):
        fp8.linear_weight_grad(w, fp8.quantize(rand(256, 8)))
    with pytest.raises(ValueError, match="out must be"):
        fp8.linear_weight_grad(q, q, out=torch.zeros(200, 199))
    with pytest.raises(ValueError, match="multiple of 128"):
        fp8.gated_forward(q, fp8.quantize_weight(rand(200, 200)))
    with pytest.raises(ValueError, match="multiple of 128"):
        fp8.gated_ffn(rand(4, 16), rand(200, 16), rand(16, 100))
    with pytest.raises(ValueError, match="do not match"):
        fp8.gated_ffn(rand(4, 16), rand(256, 16), rand(16, 256))
    with pytest.raises(ValueError, match="expected gate_up"):
        fp8.gated_backward(fp8.quantize(rand(4, 16)), fp8.quantize_weight(rand(16, 128)), q)
    with pytest.raises(ValueError, match="does not match a weight"):
        fp8.linear(rand(4, 16), rand(8, 17))
    with pytest.raises(ValueError, match="8-bit copy"):
        fp8.linear(rand(4, 200), rand(8, 200), w_q=w)
    with pytest.raises(ValueError, match="gain"):
        fp8.rms_norm(rand(4, 16), torch.ones(8))
    with pytest.raises(ValueError, match="residual"):
        fp8.add_rms_norm(rand(4, 16), rand(4, 8), torch.ones(16))
    with pytest.raises(ValueError, match="on one device"):
        fp8.linear(rand(4, 16), torch.empty(8, 16, device="meta"))


@pytest.mark.parametrize("m,d,f,out", [(0, 16, 128, 8), (3, 0, 128, 8), (3, 16, 0, 8), (3, 16, 128, 0)])
def test_gated_ffn_without_elements(m, d, f, out):
    x, wg, wd = (torch.randn(*s, requires_grad=True) for s in ((m, d), (2 * f, d), (out, f)))
    y = fp8.gated_ffn(x, wg, wd)
    assert y.shape == (m, out) and (not y.any() or (d and f))
    for g, t in zip(torch.autograd.grad(y.sum(), (x, wg, wd)), (x, wg, wd)):
        assert g.shape == t.shape and not g.isnan().any()


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_is_refused(which):
    """A dual tensor need not require grad: its tangent is refused, not dropped, whichever argument carries it."""
    from torch.autograd import forward_ad

    calls = ((fp8.linear, [rand(4, 64), rand(8, 64, seed=1), rand(8, seed=2)]), (fp8.gated_ffn, [rand(4, 64), rand(256, 64, seed=1), rand(8, 128, seed=2)]))
    for f, args in calls:
        with forward_ad.dual_level():
            dual = list(args)
            dual[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*dual)
            assert torch.equal(f(*args), f(*args))  # without a tangent: as ever
        call = lambda t: f(*args[:which], t, *args[which + 1 :])  # noqa: B023, E731
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (args[which],), (torch.ones_like(args[which]),))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_residual_stream_keeps_its_gradient(dtype):
    """``h`` of ``add_rms_norm`` passes its gradient to both terms; values and statistic are those without a graph."""
    x, r, w = rand(3, 5, 64, dtype=dtype), rand(3, 5, 64, dtype=dtype, seed=1), rand(64, dtype=dtype, seed=2)
    want = fp8.add_rms_norm(x, r, w)
    dh = rand(3, 5, 64, dtype=dtype, seed=3)
    for needs in ((True, True), (True, False), (False, True)):
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, r), needs)]
        q, rstd, h = fp8.add_rms_norm(leaves[0], leaves[1], w.clone().requires_grad_())
        assert torch.equal(h, want[2]) and torch.equal(rstd, want[1]) and not rstd.requires_grad
        assert torch.equal(values(q), values(want[0])) and torch.equal(q.scale, want[0].scale)
        h.backward(dh)
        for t, n in zip(leaves, needs):
            assert torch.equal(t.grad, dh) if n else t.grad is None
    both = x.clone().requires_grad_()  # the same tensor twice
    fp8.add_rms_norm(both, both, w)[2].backward(dh)
    assert torch.equal(both.grad, dh + dh)
    with torch.no_grad():
        assert not fp8.add_rms_norm(x.requires_grad_(), r, w)[2].requires_grad
    x.requires_grad_(False)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: fp8.add_rms_norm(t, r, w)[2], (x,), (dh,))
    assert torch.equal(torch.func.grad(lambda t: (fp8.add_rms_norm(t, r, w)[2] * dh).sum())(x), dh)


@pytest.mark.parametrize("lead", [(7,), (2, 3), ()])
def test_bias_keeps_its_gradient(lead):
    """The product of 8-bit operands is differentiable with respect to its bias, and to nothing else."""
    x, w = fp8.quantize(rand(*lead, 200)), fp8.quantize_weight(rand(24, 200, seed=1))
    bias = rand(24, seed=2)
    plain = fp8.linear_forward(x, w, bias, torch.float32)
    y = fp8.linear_forward(x, w, bias.requires_grad_(), torch.float32)
    assert torch.equal(y, plain) and not plain.requires_grad
    dy = rand(*lead, 24, seed=3)
    y.backward(dy)
    # an fp32 sum of as many terms as there are rows
    rows = dy.reshape(-1, 24).double()
    assert ((bias.grad.double() - rows.sum(0)).abs() <= len(rows) * 2.0**-24 * rows.abs().sum(0)).all()
    with torch.no_grad():
        assert not fp8.linear_forward(x, w, bias).requires_grad
    twice = torch.func.grad(lambda b: (fp8.linear_forward(x, w, b, torch.float32) * dy).sum())(bias.detach())
    assert torch.equal(twice, bias.grad)


# ------------------------------------------------------------------------------ split-backward layer


def test_split_backward_layer():
    lin = torch.nn.Linear(200, 72)
    layer = LinearFP8DW(copy.deepcopy(lin))
    x = rand(2, 9, 200).requires_grad_()
    dy = rand(2, 9, 72, seed=1)
    h = x * 1.0
    y = layer(h)
    y.backward(dy)
    assert layer.weight.grad is None  # B pass leaves parameters alone
    assert isinstance(layer.last_input, BlockScaled) and isinstance(layer.last_grad_output, BlockScaled)
    assert not layer.last_input.is_model_input
    layer.move_last_computed("input", 3)
    layer.move_last_computed("grad_output", 3)
    layer.offload_last(3, "cpu")
    layer.backward(3)
    x2 = x.detach().clone().requires_grad_()
    ref = fp8.linear(x2, lin.weight, lin.bias)
    ref.backward(dy)
    assert torch.equal(y, ref) and torch.equal(x.grad, x2.grad)
    assert torch.equal(layer.weight.grad, lin.weight.grad)
    # the bias gradient sums the 8-bit stash: each value is off by 2^-4 of itself or 2^-10 of its block's scale
    assert ((layer.bias.grad - lin.bias.grad).abs() <= (dy.abs() * 2.0**-4 + dy.abs().amax() * 2.0**-16).sum((0, 1)) + 1e-5).all()
    with pytest.raises(ValueError, match="incomplete"):
        layer.backward(3)
    first = layer.weight.grad.clone()
    layer(x.detach())  # accumulates, and a stage input stays
    assert layer.last_input.is_model_input
    layer.last_grad_output = fp8.quantize(dy)
    layer.move_last_computed("input", 0)
    layer.move_last_computed("grad_output", 0)
    layer.backward(0)
    assert torch.allclose(layer.weight.grad, 2 * first, rtol=1e-5, atol=1e-5)


def test_weight_copy_is_held_for_a_step_only():
    layer = LinearFP8DW(torch.nn.Linear(64, 32, bias=False))
    x = rand(4, 64)
    before = layer(x)
    with torch.no_grad():
        layer.weight.mul_(2)
    assert torch.equal(layer(x), 2 * before)  # outside a step: always the weight as it is
    layer.begin_step()
    q = layer.weight_q()
    assert layer.weight_q() is q
    layer.clear()
    with torch.no_grad():
        layer.weight.mul_(2)
    assert torch.equal(layer(x), 4 * before)


def test_layer_applied_twice_sums_its_output_gradients():
    layer = LinearFP8DW(torch.nn.Linear(64, 64, bias=False))
    x = rand(4, 64).requires_grad_()
    layer(layer(x)).sum().backward()
    assert isinstance(layer.last_grad_output, torch.Tensor) and layer.last_grad_output.dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("times", [2, 3])
def test_layer_applied_to_one_input_several_times(times, dtype):
    """The gradients of all applications arrive at the weight and the bias with the bits of the layer's type."""
    layer = LinearFP8DW(torch.nn.Linear(64, 40).to(dtype))
    x = rand(6, 64, dtype=dtype)
    dys = [rand(6, 40, dtype=dtype, seed=s + 1) for s in range(times)]
    torch.autograd.backward([layer(x) for _ in dys], dys)
    layer.move_last_computed("input", 0)
    layer.move_last_computed("grad_output", 0)
    layer.offload_last(0, "cpu")
    layer.backward(0)
    xq = held(x)[0]
    total, mag = sum(held(dy)[0] for dy in dys), sum(held(dy)[0].abs() for dy in dys)
    # each sum of gradients is rounded to the layer's bits (8 of bf16, 16 in two parts, 24 in three), half a unit of them
    half = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-16, torch.float32: 2.0**-23}[dtype]
    spread = (times - 1) * half * mag
    bound = product_bound(total.T, xq, dtype) + spread.T @ xq.abs() * (1 + torch.finfo(dtype).eps)
    assert ((layer.weight.grad.double() - total.T @ xq).abs() <= bound).all()
    want = total.sum(0)
    assert ((layer.bias.grad.double() - want).abs() <= spread.sum(0) + 6 * 2.0**-24 * mag.sum(0) + torch.finfo(dtype).eps / 2 * (want.abs() + mag.sum(0) * 2.0**-8)).all()


def test_layer_ships_without_its_stash():
    import pickle

    layer = LinearFP8DW(torch.nn.Linear(64, 32))
    layer(rand(4, 64))
    layer.move_last_computed("input", 1)
    layer(rand(4, 64))
    for twin in (pickle.loads(pickle.dumps(layer)), copy.deepcopy(layer)):
        assert twin.last_input is None and twin.is_empty("input") and twin._weight_q is None
        assert torch.equal(twin(rand(4, 64)), layer(rand(4, 64)))
    assert isinstance(layer.ctx["input"][1], BlockScaled)


def test_replacement_selects_layers():
    model = torch.nn.Sequential(torch.nn.Linear(8, 8), torch.nn.ReLU(), torch.nn.Linear(8, 8))
    replace_layer_with_layer_dw(model)
    replace_linear_with_linear_fp8(model, lambda name, m: name == "2")
    assert type(model[0]) is LinearDW and type(model[2]) is LinearFP8DW
    inner = model[2]
    replace_linear_with_linear_fp8(model)
    assert type(model[0]) is LinearFP8DW and model[2] is inner


# ------------------------------------------------------------------------------ Llama

CFG = LlamaConfig(n_layers=2, d_model=128, n_heads=4, n_kv_heads=2, ffn=256, vocab=512, seq_len=32, rope_theta=10000.0)


def test_llama_option_builds_8_bit_layers():
    cfg = LlamaConfig(**{**CFG.__dict__, "ffn_fp8": True})
    (stage,) = build_llama_stages(cfg, 1, dtype=torch.float32)
    kinds = {name.rpartition(".")[2]: type(m) for name, m in stage.named_modules() if isinstance(m, LinearDW)}
    assert kinds == {"wqkv": LinearDW, "wo": LinearDW, "w_gate_up": LinearFP8DW, "w_down": LinearFP8DW, "out": LinearDW}
    assert [n for n, _ in stage.named_parameters()] == [n for n, _ in build_llama_stages(CFG, 1, dtype=torch.float32)[0].named_parameters()]
    with pytest.raises(ValueError, match="split_backward"):
        build_llama_stages(cfg, 1, split_backward=False)


@pytest.mark.parametrize("scheduler", ["zbv", "afab", "full_remat"])
def test_llama_pipeline_steps_in_8_bits(scheduler):
    """Whole steps through the pipeline: the loss and the gradients stay near those of the 16-bit feed-forward
    layers.  Rounding an operand to e4m3 moves it by at most 2^-4 of itself, 2^-4 / sqrt(3) = 3.6 % in the mean
    square; a feed-forward gradient passes five such roundings, 3.6 % sqrt(5) = 8 %, and 16 % allows for their meeting
    in the second layer."""
    tok = torch.randint(0, CFG.vocab, (4, CFG.seq_len + 1), generator=torch.Generator().manual_seed(0))
    grads, losses = [], []
    for ffn_fp8 in (False, True):
        cfg = LlamaConfig(**{**CFG.__dict__, "ffn_fp8": ffn_fp8})
        placement = [0, 0]
        stages = build_llama_stages(cfg, 2, dtype=torch.float32, seed=3)
        pipe = Pipeline(stages, None, partitioner=False, scheduler=scheduler, placement=placement, outputs="none")
        for _ in range(2):
            pipe.zero_grad()
            _, loss = pipe(tok[:, :-1].contiguous(), tok[:, 1:].contiguous(), llama_loss_fn, split_size=1)
        losses.append(float(loss))
        grads.append({n: p.grad.clone() for n, p in pipe.named_parameters()})
        assert all(m._weight_q is None and m.is_empty("input") for b in pipe.blocks for m in b.dw_layers() if isinstance(m, LinearFP8DW))
    assert abs(losses[0] - losses[1]) < 0.02 * losses[0]
    for name, g in grads[0].items():
        assert (grads[1][name] - g).norm() <= 0.16 * g.norm(), name


def test_mlp_block_composes_on_cpu():
    torch.manual_seed(0)
    blk = LlamaMLPBlock(CFG)
    replace_linear_with_linear_fp8(blk)
    x = rand(2, 8, CFG.d_model).requires_grad_()
    blk(x).sum().backward()
    assert x.grad is not None and isinstance(blk.w_down.last_input, BlockScaled)


@pytest.mark.parametrize("partitioner", ["handcrafted", "naive"])
def test_command_runs_in_8_bits(partitioner):
    """``run_transformer.py --ffn-fp8``: hand-made stages, and a traced, cut and shipped model."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1", "--master-port", str(_free_port()),
           os.path.join(root, "benchmarks", "run_transformer.py"), "--architecture", "llama", "--name", "llama-tiny", "--partitioner", partitioner, "--ffn-fp8",
           "--scheduler", "zbh1", "--nmb", "4", "--mb-size", "1", "--niters", "1", "--warmup", "1", "--backend", "gloo"]
    if partitioner != "handcrafted":
        cmd.append("--check")  # one step against the same model in a single process
    out = subprocess.run(cmd, cwd=root, capture_output=True, text=True, timeout=300, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""))
    assert out.returncode == 0, out.stdout[-1500:] + out.stderr[-3000:]
    assert "tokens_per_s" in out.stdout
