"""8-bit operators on the GPU against their definition in 64 bits (``fp8_oracle``)."""

import pytest
import torch

from .fp8_oracle import held, product_bound, values

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def dev():
    from elf_b200.ops import _ext

    assert _ext.available(), "the native extension must be built for GPU tests"
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def no_kernel_error():
    yield
    from elf_b200.ops import gemm

    gemm.check_status()


def activations(rows, cols, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, cols, device=dev, generator=g)
    loud = torch.rand(cols, device=dev, generator=g) < 0.02
    return (x * (1 + 19 * loud)).to(dtype)


def same(got, want):
    """Equal bit for bit, NaN included."""
    got, want = got.double().cpu(), want.double().cpu()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


# ------------------------------------------------------------------------------ quantise / restore


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (33, 200), (130, 256), (5, 1000), (64, 528), (257, 16)])
def test_quantize_is_exact(dev, rows, cols, dtype):
    from elf_b200.ops import fp8

    x = activations(rows, cols, dtype, dev, rows + cols)
    for make, block_rows in ((fp8.quantize, 1), (fp8.quantize_weight, 128)):
        q = make(x)
        want, exps = held(x, block_rows)
        assert torch.equal(q.scale.cpu(), exps)
        assert same(values(q), want)
        for out in DTYPES:
            assert same(fp8.dequantize(q, out), want.to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_special_values(dev, dtype):
    from elf_b200.ops import fp8

    inf, nan = float("inf"), float("nan")
    x = activations(12, 272, dtype, dev, 3)
    x[0] = 0
    x[1, 5], x[1, 6], x[1, 200] = inf, -inf, nan  # the rest of each block keeps its own scale
    x[2, :128] = nan
    x[3, :128] = inf
    x[4] = torch.finfo(dtype).max
    x[5] = torch.finfo(dtype).smallest_normal
    x[6] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # smallest subnormal
    x[7] = x[7] * 0 - 0.0
    x[8, :128] = 448.0  # on the border: the scale stays 1
    x[9, :128] = 448.0
    x[9, 3] = 450.0  # just over it (fp16, fp32; bf16 rounds to 450)
    x[10, :128] = torch.arange(128, device=dev).to(dtype) * 3.5
    for make, block_rows in ((fp8.quantize, 1), (fp8.quantize_weight, 128)):
        q = make(x)
        want, exps = held(x, block_rows)
        assert torch.equal(q.scale.cpu(), exps)
        assert same(values(q), want)


@pytest.mark.parametrize("cols", [256, 250])
def test_quantize_strides_and_leading_dimensions(dev, cols):
    from elf_b200.ops import fp8

    base = activations(24, 2 * 640, torch.bfloat16, dev, 5).view(2, 12, 1280)
    for x in (base[:, :, :cols], base[:, :, 3 : cols + 3], base[:, ::2, 16 : 16 + cols], base.transpose(0, 1)[:, :, :cols], base[0, 0, :cols],
              base[0].t()[:cols, :7], base[:1, :1, :cols].expand(2, 5, cols)):
        q = fp8.quantize(x)
        assert q.shape == x.shape
        want, exps = held(x.reshape(-1, x.shape[-1]))
        assert torch.equal(q.scale.reshape(exps.shape).cpu(), exps)
        assert same(values(q), want)
        assert same(fp8.dequantize(q).reshape(want.shape), want)


def test_quantize_leaves_neighbours_alone(dev):
    """Padding behind a row's last value and rows behind the last one keep what they held."""
    from elf_b200.ops import _ext

    x = activations(5, 140, torch.bfloat16, dev)
    data, scale = (torch.full((7, n), 0x5A, dtype=torch.uint8, device=dev) for n in (160, 8))
    _ext.get().fp8_quantize(x, False, data[:5, :140], scale[:5, :2])
    assert bool((data[5:] == 0x5A).all()) and bool((data[:, 140:] == 0x5A).all())
    assert bool((scale[5:] == 0x5A).all()) and bool((scale[:, 2:] == 0x5A).all())
    out = torch.full((7, 160), 7.0, dtype=torch.bfloat16, device=dev)
    _ext.get().fp8_dequantize(data[:5, :140], scale[:5, :2], 0, torch.bfloat16, out[:5, :140])
    assert bool((out[5:] == 7).all()) and bool((out[:, 140:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 15, 16, 17, 40, 127, 129, 515, 1040])
def test_rows_that_start_anywhere(dev, dtype, cols):
    """Views at every offset to 16 bytes, with rows that touch: neighbours are neither read into a block nor written."""
    from elf_b200.ops import fp8

    rows = 37
    want_x = activations(rows, cols, dtype, dev, cols)
    aligned = torch.zeros(rows, -(-cols // 16) * 16, dtype=dtype, device=dev)[:, :cols]
    aligned.copy_(want_x)
    want, want_w = fp8.quantize(aligned), fp8.quantize_weight(aligned)
    restored = fp8.dequantize(want, dtype, out=torch.zeros_like(aligned))
    for offset in range(0, 32 // dtype.itemsize + 1):
        for pitch in (cols, cols + 1, cols + 3):
            buffer = torch.full((offset + rows * pitch + 40,), 3e4, dtype=dtype, device=dev)
            view = buffer[offset : offset + rows * pitch].view(rows, pitch)[:, :cols]
            view.copy_(want_x)
            for got, ref in ((fp8.quantize(view), want), (fp8.quantize_weight(view), want_w)):
                assert torch.equal(got.scale, ref.scale) and torch.equal(got.data.view(torch.uint8), ref.data.view(torch.uint8))
            buffer.fill_(5)
            fp8.dequantize(want, out=view)
            assert torch.equal(view, restored)
            view.fill_(5)
            assert (buffer == 5).all()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(2304, 2304), (2300, 2200)])  # 81 tiles: 7 are left over on 74 pairs, and split
def test_weight_grad_of_split_tiles(dev, n, k, out):
    """The parts of a split tile are added in fp32, in one order, and rounded once."""
    from elf_b200.ops import fp8

    dy, x = fp8.quantize(activations(4100, n, torch.bfloat16, dev, 1)), fp8.quantize(activations(4100, k, torch.bfloat16, dev, 2))
    a, b = values(dy).T, values(x)
    got = fp8.linear_weight_grad(dy, x, out_dtype=out)
    bound = product_bound(a, b, out)
    assert ((got.double() - a @ b).abs() <= bound).all()
    assert (got.double() - a @ b).norm() / (a @ b).norm() < (2.0**-9 if out == torch.bfloat16 else 1e-5)
    for _ in range(3):
        assert torch.equal(got, fp8.linear_weight_grad(dy, x, out_dtype=out))
    # added to a gradient: one more rounding, of the sum
    results = []
    for _ in range(4):
        grad = torch.full((n, k), 3.0, device=dev, dtype=out)
        results.append(fp8.linear_weight_grad(dy, x, out=grad))
    assert all(torch.equal(results[0], r) for r in results[1:])
    want = a @ b + 3.0
    assert ((results[0].double() - want).abs() <= bound + (want.abs() + 3.0) * torch.finfo(out).eps).all()


@pytest.mark.parametrize("n,k", [(1, 1), (7, 33), (40, 129), (33, 1043), (129, 7)])
def test_weight_grad_of_odd_widths(dev, n, k):
    """Rows of the result start anywhere; operands from 8 bits and as they are."""
    from elf_b200.ops import fp8

    dy, x = activations(300, n, torch.bfloat16, dev, n), activations(300, k, torch.bfloat16, dev, k)
    dyq, xq = fp8.quantize(dy), fp8.quantize(x)
    for a, b, av, bv in ((dyq, xq, values(dyq), values(xq)), (dy, xq, dy.double(), values(xq)), (dy, x, dy.double(), x.double())):
        for out in DTYPES:
            got = fp8.linear_weight_grad(a, b, out_dtype=out)
            assert got.shape == (n, k) and got.is_contiguous()
            # an fp32 sum of 300 products, rounded once (through fp32 to fp16)
            mag = av.abs().T @ bv.abs()
            want = av.T @ bv
            assert ((got.double() - want).abs() <= mag * 300 * 2.0**-23 + want.abs() * torch.finfo(out).eps + 2.0**-24).all()


def parts_bound(a, b, out, pairs):
    """Bound on the error of ``a @ b`` as the sum of ``pairs`` products of bf16 parts of the operands, added in fp32: the parts
    of a value add up to at most 1 + 2^-7 + 2^-15 of its magnitude, which enters once for each operand, and every product after the first
    adds half a unit of the sum."""
    return product_bound(a, b, out) * (1 + 2.0**-6 + 2.0**-12) + pairs * 2.0**-24 * (a.abs() @ b.abs()) * (1 + 2.0**-5)


@pytest.mark.parametrize("tokens,n,k", [(1, 1, 1), (5, 7, 33), (64, 136, 264), (300, 130, 72), (2304, 264, 1040)])
@pytest.mark.parametrize("dtype,parts", [(torch.float16, 2), (torch.float32, 3)])
def test_weight_grad_of_whole_operands(dev, tokens, n, k, dtype, parts):
    """fp16 and fp32 operands enter with all their bits, at any address and pitch."""
    from elf_b200.ops import fp8

    wide = activations(tokens, n + 40, dtype, dev, 1)
    x16 = activations(tokens, k, dtype, dev, 2)
    xq = fp8.quantize(x16)
    for dy in (wide[:, :n], wide[:, 3 : n + 3], wide[:, 8 : n + 8].contiguous()):
        for x, xv, pairs in ((xq, values(xq), parts), (x16, x16.double(), parts * parts), (x16.bfloat16(), x16.bfloat16().double(), parts)):
            a = dy.double().T
            for out in DTYPES:
                got = fp8.linear_weight_grad(dy, x, out_dtype=out)
                assert got.dtype == out and ((got.double() - a @ xv).abs() <= parts_bound(a, xv, out, pairs)).all()
                assert torch.equal(got, fp8.linear_weight_grad(dy, x, out_dtype=out))
            for out in (torch.bfloat16, torch.float32):
                grad = torch.full((n, k), 3.0, device=dev, dtype=out)
                assert fp8.linear_weight_grad(dy, x, out=grad).data_ptr() == grad.data_ptr()
                want = a @ xv + 3.0
                bound = parts_bound(a, xv, torch.float32, pairs) + (pairs + 1) * 2.0**-23 * (3.0 + (a.abs() @ xv.abs()))
                assert ((grad.double() - want).abs() <= bound + torch.finfo(out).eps / 2 * (want.abs() + bound)).all()
        # the other operand in 8 bits
        dyq = fp8.quantize(dy)
        a = values(dyq).T
        assert ((fp8.linear_weight_grad(dyq, x16, out_dtype=torch.float32).double() - a @ x16.double()).abs() <= parts_bound(a, x16.double(), torch.float32, parts)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_weight_grad_of_whole_operands_not_finite(dev, dtype):
    """An infinity stays one, a NaN as well, also one whose payload is in its low bits; columns do not see each other."""
    from elf_b200.ops import fp8

    dy, x = activations(40, 72, dtype, dev, 1), fp8.quantize(torch.ones(40, 136, device=dev))
    clean = fp8.linear_weight_grad(dy, x, out_dtype=torch.float32)
    bits = torch.int16 if dtype == torch.float16 else torch.int32
    dy[3, 5], dy[7, 9], dy[0, 70] = float("inf"), float("-inf"), float("nan")
    dy.view(bits)[2, 33] = 0x7C01 if dtype == torch.float16 else 0x7F800001
    got = fp8.linear_weight_grad(dy, x, out_dtype=torch.float32)
    rows = torch.ones(72, dtype=torch.bool, device=dev)
    rows[[5, 9, 33, 70]] = False
    assert torch.equal(got[rows], clean[rows])
    assert (got[5] == float("inf")).all() and (got[9] == float("-inf")).all() and got[70].isnan().all() and got[33].isnan().all()


def test_weight_grad_of_the_largest_and_smallest_operands(dev):
    """fp32 from its largest values to below bf16's smallest normal one."""
    from elf_b200.ops import fp8

    for scale in (2.0**126, 2.0**-120, 2.0**-128):
        dy = (torch.rand(3, 40, device=dev, dtype=torch.float64) + 1) * scale
        dy = dy.float()
        x = fp8.quantize(torch.ones(3, 16, device=dev) * 2.0**-4)
        a, b = dy.double().T, values(x)
        got = fp8.linear_weight_grad(dy, x, out_dtype=torch.float32)
        # what lies below 2^-133 of a value is not held by bf16, and the tensor core's fp32 sums may drop subnormal ones
        assert ((got.double() - a @ b).abs() <= parts_bound(a, b, torch.float32, 3) + 3 * 2.0**-126).all()


def test_empty_tensors(dev):
    from elf_b200.ops import fp8

    for shape in ((0, 128), (3, 0), (2, 0, 64)):
        q = fp8.quantize(torch.empty(shape, device=dev))
        assert q.shape == torch.Size(shape) and fp8.dequantize(q).shape == torch.Size(shape)
    w = fp8.quantize_weight(torch.randn(40, 64, device=dev))
    assert fp8.linear_forward(fp8.quantize(torch.empty(0, 64, device=dev)), w).shape == (0, 40)
    dw = fp8.linear_weight_grad(fp8.quantize(torch.empty(0, 40, device=dev)), fp8.quantize(torch.empty(0, 64, device=dev)))
    assert dw.shape == (40, 64) and not dw.any()


def test_quantize_beyond_32_bit_offsets(dev):
    """Rows whose byte offset passes 2^32, in input and in the 8-bit copy."""
    from elf_b200.ops import fp8

    rows, cols = (1 << 32) // 4096 + 3, 4096
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=dev)
    tail = activations(3, cols, torch.bfloat16, dev, 9)
    x[-3:] = tail
    x[:2] = tail[:2] * 2
    q = fp8.quantize(x)
    want, exps = held(tail)
    assert torch.equal(q.scale[-3:].cpu(), exps)
    assert same(fp8.dequantize(fp8.BlockScaled(q.data[-3:], q.scale[-3:])), want)
    assert same(fp8.dequantize(fp8.BlockScaled(q.data[:2], q.scale[:2])), held(tail[:2] * 2)[0])
    del x
    y = fp8.dequantize(q)
    assert same(y[-3:], want) and not y[2:-3].any()


# ------------------------------------------------------------------------------ RMSNorm


@pytest.mark.parametrize("rows,dim", [(1, 8), (9, 128), (33, 264), (5, 512), (7, 1000), (130, 1024), (64, 2048), (3, 2056), (17, 4096), (2, 4104), (11, 5120), (5, 8192)])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(dev, rows, dim, residual):
    from elf_b200.ops import fp8

    x, r = activations(rows, dim, torch.bfloat16, dev, 1), activations(rows, dim, torch.bfloat16, dev, 2)
    w = (1 + 0.1 * torch.randn(dim, device=dev)).to(torch.bfloat16)
    if residual:
        q, rstd, h = fp8.add_rms_norm(x, r, w, 1e-5)
        hd = (x.double() + r.double()).to(torch.bfloat16).double()
        assert same(h, hd)
    else:
        q, rstd = fp8.rms_norm(x, w, 1e-5)
        hd = x.double()
    want_rstd = (hd.square().mean(1) + 1e-5).rsqrt()
    # dim additions of fp32 squares, each off by half a unit at most, halved by the root; the root itself 2^-22
    assert ((rstd.double() - want_rstd).abs() <= want_rstd * (dim * 2.0**-25 + 2.0**-22)).all()
    y = hd * want_rstd[:, None] * w.double()
    got = values(q)
    # one rounding to e4m3 in units of the block's scale (half a step: 2^-4 of the value, 2^-10 units below
    # 2^-6), after an fp32 error that is smaller than that by three orders of magnitude
    unit = torch.exp2(q.scale.double() - 127).repeat_interleave(128, 1)[:, :dim]
    fp32 = y.abs() * (dim * 2.0**-25 + 2.0**-21)
    assert ((got - y).abs() <= torch.maximum(y.abs() * 2.0**-4, unit * 2.0**-10) + fp32).all()
    # and the scale is the smallest that holds the block, up to that fp32 error
    top = torch.nn.functional.pad(y.abs(), (0, -dim % 128)).view(rows, -1, 128).amax(2)
    scale = torch.exp2(q.scale.double() - 127)
    slack = 1 + dim * 2.0**-25 + 2.0**-21
    assert (top <= 448 * scale * slack).all() and (top * slack >= 224 * scale).all()


@pytest.mark.parametrize("rows,dim", [(4000, 1024), (4096, 4096)])
def test_rms_norm_rounds_once(dev, rows, dim):
    """The 8-bit values are the roundings of the exact ones: an error of 1e-9 in a row's statistic moves one value in 10^8."""
    from elf_b200.ops import fp8

    for seed in range(24):
        x = activations(rows, dim, torch.bfloat16, dev, seed)
        w = (1 + 0.1 * torch.randn(dim, device=dev)).to(torch.bfloat16)
        xd = x.double()
        y = xd / (xd.square().sum(1, keepdim=True) / dim + 1e-5).sqrt() * w.double()
        q = fp8.rms_norm(x, w, 1e-5)[0]
        unit = torch.exp2(q.scale.double() - 127).repeat_interleave(128, 1)
        step = unit * torch.exp2(torch.floor(torch.log2((y / unit).abs().clamp_min(2.0**-6))) - 3)
        assert torch.equal(values(q), torch.round(y / step) * step)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,dim", [(9, 1032), (700, 1304), (65, 1536), (3, 1544), (5, 1800), (7, 2040), (3000, 1800), (2500, 4096), (1800, 5120), (1300, 8192)])
def test_rms_norm_of_other_widths_and_more_rows(dev, rows, dim, residual):
    """The widest rows that a warp takes and the narrowest that a block does; more rows than blocks, so that each walks to its next one."""
    test_rms_norm(dev, rows, dim, residual)


@pytest.mark.parametrize("rows,dim", [(3000, 1304), (3000, 1800), (2000, 5120)])
def test_rms_norm_of_a_sum_rounds_once(dev, rows, dim):
    from elf_b200.ops import fp8

    for seed in range(6):
        x, r = activations(rows, dim, torch.bfloat16, dev, seed), activations(rows, dim, torch.bfloat16, dev, 100 + seed)
        w = (1 + 0.1 * torch.randn(dim, device=dev)).to(torch.bfloat16)
        hd = (x.double() + r.double()).to(torch.bfloat16).double()
        y = hd / (hd.square().sum(1, keepdim=True) / dim + 1e-5).sqrt() * w.double()
        q, _, h = fp8.add_rms_norm(x, r, w, 1e-5)
        assert same(h, hd)
        unit = torch.exp2(q.scale.double() - 127).repeat_interleave(128, 1)[:, :dim]
        step = unit * torch.exp2(torch.floor(torch.log2((y / unit).abs().clamp_min(2.0**-6))) - 3)
        assert torch.equal(values(q), torch.round(y / step) * step)


def test_rms_norm_rows_without_finite_values(dev):
    from elf_b200.ops import fp8

    x = activations(4, 256, torch.bfloat16, dev)
    x[0], x[1, 7], x[2, 9] = 0, float("nan"), float("inf")
    w = torch.ones(256, device=dev, dtype=torch.bfloat16)
    got = fp8.rms_norm(x, w)[0].dequantize()
    assert not got[0].any()
    assert got[1].isnan().all()
    assert got[2, 9].isnan() and not got[2, :9].any()  # 1/inf = 0 for the others, inf * 0 for it
    alone = fp8.rms_norm(x[3:], w)[0].dequantize()
    assert same(got[3:], alone)  # rows do not see each other


# ------------------------------------------------------------------------------ products

SHAPES = [(1, 1, 1), (1, 16, 32), (128, 256, 128), (130, 260, 140), (7, 129, 513), (256, 128, 640), (300, 520, 1000), (64, 1040, 16), (1000, 72, 392)]


def operands(m, n, k, dev, seed=0):
    from elf_b200.ops import fp8

    x = fp8.quantize(activations(m, k, torch.bfloat16, dev, seed))
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    # weights whose tiles differ in magnitude, so that a scale taken from the wrong tile shows
    w = torch.randn(n, k, device=dev, generator=g)
    w = w * torch.exp2((torch.arange(n, device=dev) // 128 % 5).float())[:, None] * torch.exp2(-(torch.arange(k, device=dev) // 128 % 7).float())[None]
    return x, fp8.quantize_weight(w.to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out", DTYPES)
def test_linear_forward(dev, m, n, k, out):
    from elf_b200.ops import fp8

    x, w = operands(m, n, k, dev)
    a, b = values(x), values(w).T
    y = fp8.linear_forward(x, w, out_dtype=out)
    assert y.dtype == out and ((y.double() - a @ b).abs() <= product_bound(a, b, out)).all()
    bias = torch.randn(n, device=dev).to(out)
    yb = fp8.linear_forward(x, w, bias, out_dtype=out)
    want = a @ b + bias.double()
    assert ((yb.double() - want).abs() <= product_bound(a, b, out) + (bias.double().abs() + want.abs()) * (torch.finfo(out).eps / 2 + 2.0**-24)).all()


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_forward_row_scaled_weight(dev, m, n, k):
    from elf_b200.ops import fp8

    x = fp8.quantize(activations(m, k, torch.bfloat16, dev, 1))
    w = fp8.quantize(activations(n, k, torch.bfloat16, dev, 2) * torch.exp2((torch.arange(n, device=dev) % 11).float())[:, None].bfloat16())
    a, b = values(x), values(w).T
    y = fp8.linear_forward(x, w)
    assert ((y.double() - a @ b).abs() <= product_bound(a, b, torch.bfloat16)).all()


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_linear_input_grad(dev, m, n, k, out):
    from elf_b200.ops import fp8

    _, w = operands(1, n, k, dev)
    dy = fp8.quantize(activations(m, n, torch.bfloat16, dev, 4) * 1e-3)
    a, b = values(dy), values(w)
    dx = fp8.linear_input_grad(dy, w, out)
    assert dx.shape == (m, k) and ((dx.double() - a @ b).abs() <= product_bound(a, b, out)).all()


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_weight_grad(dev, m, n, k):
    from elf_b200.ops import fp8

    dy, x = fp8.quantize(activations(m, n, torch.bfloat16, dev, 4) * 1e-3), fp8.quantize(activations(m, k, torch.bfloat16, dev, 5))
    a, b = values(dy).T, values(x)
    want, bound32 = a @ b, product_bound(a, b, torch.float32)
    dw = fp8.linear_weight_grad(dy, x, out_dtype=torch.float32)
    assert ((dw.double() - want).abs() <= bound32).all()
    # bf16 results of tiles that are split along K are sums of rounded parts
    dw = fp8.linear_weight_grad(dy, x)
    assert ((dw.double() - want).abs() <= product_bound(a, b, torch.bfloat16) + 4 * 2.0**-8 * (a.abs() @ b.abs())).all()
    acc = torch.ones(n, k, device=dev)
    got = fp8.linear_weight_grad(dy, x, out=acc)
    assert got.data_ptr() == acc.data_ptr()
    assert ((acc.double() - 1 - want).abs() <= bound32 + 2.0**-23 * (1 + want.abs())).all()


def test_products_of_many_tiles(dev):
    """Several tiles for every SM, so that accumulators, ring slots and scale slots wrap around."""
    from elf_b200.ops import fp8

    for m, n, k in ((2100, 5000, 300), (4096, 2560, 1100)):
        x, w = operands(m, n, k, dev, 7)
        a, b = values(x), values(w).T
        assert ((fp8.linear_forward(x, w).double() - a @ b).abs() <= product_bound(a, b, torch.bfloat16)).all()
        dy = fp8.quantize(activations(m, n, torch.bfloat16, dev, 4))
        a, b = values(dy), values(w)
        assert ((fp8.linear_input_grad(dy, w).double() - a @ b).abs() <= product_bound(a, b, torch.bfloat16)).all()


# ------------------------------------------------------------------------------ gated feed-forward block


def check_held(q, y, err):
    """``q`` holds the matrix ``y`` known to within ``err`` (elementwise): one rounding to e4m3 on top of it, in units of
    a scale that is right for some matrix within ``err`` of ``y``."""
    rows, cols = y.shape
    unit = torch.exp2(q.scale.double().reshape(rows, -1) - 127)
    wide = unit.repeat_interleave(128, 1)[:, :cols]
    got = values(q)
    assert ((got - y).abs() <= err + torch.maximum((y.abs() + err) * 2.0**-4, wide * 2.0**-10)).all()
    blocks = lambda t: torch.nn.functional.pad(t, (0, -cols % 128)).view(rows, -1, 128).amax(2)  # noqa: E731
    assert (blocks((y.abs() - err).clamp_min(0)) <= 448 * unit).all()
    small = unit <= 2.0**-126
    assert ((blocks(y.abs() + err) >= 224 * unit) | small).all()


def projections(x, w, k):
    a, b = values(x), values(w).T
    gu = a @ b
    return gu, k * 2.0**-23 * (a.abs() @ b.abs())


@pytest.mark.parametrize("m,k,f", [(1, 16, 128), (3, 200, 128), (128, 256, 512), (130, 128, 384), (300, 1000, 640), (2000, 528, 2560)])
@pytest.mark.parametrize("keep", [True, False])
def test_gated_forward(dev, m, k, f, keep):
    from elf_b200.ops import fp8

    x, w = operands(m, 2 * f, k, dev, 11)
    act, gu = fp8.gated_forward(x, w, keep=keep)
    want, err = projections(x, w, k)
    assert act.shape == (m, f) and (gu is None) != keep
    if keep:
        check_held(gu, want, err)
    g, u = want[:, :f], want[:, f:]
    s = torch.sigmoid(g)
    # |d silu| <= 1.1 |dg|; the exponential, the division and two products add a few units: 2^-20 relative, and
    # |g| 2^-22 for the exponent's argument
    err_act = 1.1 * err[:, :f] * u.abs() + (g * s).abs() * err[:, f:] + 1.1 * err[:, :f] * err[:, f:] + (g * s * u).abs() * (2.0**-20 + g.abs() * 2.0**-22)
    check_held(act, g * s * u, err_act + 1e-37)


def test_gated_forward_not_finite(dev):
    """An infinite or NaN projection reaches only its own row, and only as NaN."""
    from elf_b200.ops import fp8

    x = activations(40, 128, torch.bfloat16, dev)
    clean_act, clean_gu = fp8.gated_forward(fp8.quantize(x), w := fp8.quantize_weight(activations(256, 128, torch.bfloat16, dev, 1)))
    x[7, 3], x[30, 100] = float("nan"), float("inf")
    act, gu = fp8.gated_forward(fp8.quantize(x), w)
    rows = torch.ones(40, dtype=torch.bool, device=dev)
    rows[7] = rows[30] = False
    for got, want in ((act, clean_act), (gu, clean_gu)):
        assert values(got)[~rows].isnan().all()
        assert torch.equal(got.scale[rows], want.scale[rows]) and same(values(got)[rows], values(want)[rows])


@pytest.mark.parametrize("m,d,f", [(1, 16, 128), (3, 200, 128), (130, 128, 384), (300, 1000, 640), (1500, 528, 2560)])
def test_gated_backward(dev, m, d, f):
    from elf_b200.ops import fp8

    _, w_down = operands(1, d, f, dev, 3)
    dy = fp8.quantize(activations(m, d, torch.bfloat16, dev, 4) * 1e-3)
    gu = fp8.quantize(activations(m, 2 * f, torch.bfloat16, dev, 5))
    got = fp8.gated_backward(dy, w_down, gu)
    a, b = values(dy), values(w_down)
    da, err = a @ b, d * 2.0**-23 * (a.abs() @ b.abs())
    g, u = values(gu)[:, :f], values(gu)[:, f:]
    s = torch.sigmoid(g)
    fg, fu = u * s * (1 + g * (1 - s)), g * s
    rel = 2.0**-19 + g.abs() * 2.0**-21
    # 1 - s cancels for large gates: an absolute error of 2^-22 there, times |g|
    err_g = err * fg.abs() + (da * fg).abs() * rel + (da.abs() + err) * (u * s).abs() * (g.abs() + 1) * 2.0**-21 * (1 + g.abs())
    err_u = err * fu.abs() + (da * fu).abs() * rel
    check_held(got, torch.cat([da * fg, da * fu], 1), torch.cat([err_g, err_u], 1) + 1e-37)


@pytest.mark.parametrize("m,d,f", [(4000, 528, 5248), (2600, 200, 6272)])  # 16 x 21 and 11 x 25 tiles on 74 pairs
def test_gated_backward_of_many_tiles(dev, m, d, f):
    """Three and more units for every pair of CTAs: both accumulators, each barrier's next phase, a last tile of half the columns."""
    test_gated_backward(dev, m, d, f)


@pytest.mark.parametrize("m,d,f", [(300, 200, 640), (4000, 136, 5248)])
def test_gated_backward_not_finite(dev, m, d, f):
    """What is not finite in the output's gradient reaches its own row, in the checkpoint its own column of its row, and only as NaN."""
    from elf_b200.ops import fp8

    _, w = operands(1, d, f, dev, 3)
    dy, gate_up = activations(m, d, torch.bfloat16, dev, 4), activations(m, 2 * f, torch.bfloat16, dev, 5)
    rows, cols = [5, 130, m - 1], [3, f // 2 + 7, f - 1]
    for r, c in zip(rows, cols):  # no block's largest gradient, with or without them
        gate_up[r, c] = gate_up[r, f + c] = 0
    clean = fp8.gated_backward(fp8.quantize(dy), w, fp8.quantize(gate_up))
    inf, nan = float("inf"), float("nan")
    gate_up[rows[0], cols[0]] = nan  # gate: both gradients
    gate_up[rows[1], f + cols[1]] = inf  # up: that of gate alone
    gate_up[rows[2], cols[2]] = -inf
    dy[7, 3], dy[200, d - 1] = nan, inf
    got = fp8.gated_backward(fp8.quantize(dy), w, fp8.quantize(gate_up))
    want = values(clean)
    want[rows[0], [cols[0], f + cols[0]]] = nan
    want[rows[1], cols[1]] = nan
    want[rows[2], [cols[2], f + cols[2]]] = nan
    whole = torch.zeros(m, dtype=torch.bool, device=dev)
    whole[[7, 200]] = True
    assert values(got)[whole].isnan().all()
    assert same(values(got)[~whole], want[~whole])
    finite_blocks = ~whole
    assert torch.equal(got.scale[finite_blocks], clean.scale[finite_blocks])


@pytest.mark.parametrize("m,n,k", [*SHAPES, (2047, 264, 528), (4100, 2304, 1040)])
def test_weight_grad_rounds_once(dev, m, n, k):
    """bf16 results are fp32 sums rounded once, tiles that are split along the tokens among them."""
    from elf_b200.ops import fp8

    dy, x = fp8.quantize(activations(m, n, torch.bfloat16, dev, 4) * 1e-3), fp8.quantize(activations(m, k, torch.bfloat16, dev, 5))
    a, b = values(dy).T, values(x)
    assert ((fp8.linear_weight_grad(dy, x).double() - a @ b).abs() <= product_bound(a, b, torch.bfloat16)).all()


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (16, 1000, 5504), (100, 136, 9000), (128, 264, 4100), (77, 20000, 640), (2, 128, 30000)])
def test_products_of_few_rows(dev, m, n, k):
    """Up to 128 rows: the reduction is split over the CTAs of a cluster."""
    from elf_b200.ops import fp8

    x, w = operands(m, n, k, dev, 13)
    a, b = values(x), values(w).T
    bias = torch.randn(n, device=dev)
    y = fp8.linear_forward(x, w, bias, out_dtype=torch.float32)
    want = a @ b + bias.double()
    assert ((y.double() - want).abs() <= product_bound(a, b, torch.float32) + (bias.double().abs() + want.abs()) * 2.0**-23).all()
    assert torch.equal(y, fp8.linear_forward(x, w, bias, out_dtype=torch.float32))  # the order of the sums is fixed
    dy = fp8.quantize(activations(m, n, torch.bfloat16, dev, 4) * 1e-3)
    a, b = values(dy), values(w)
    assert ((fp8.linear_input_grad(dy, w).double() - a @ b).abs() <= product_bound(a, b, torch.bfloat16)).all()


def test_split_last_wave(dev):
    """More tiles than CTA pairs and a long reduction: the last wave's tiles are split along K."""
    from elf_b200.ops import fp8

    m, n, k = 2304, 2304, 14336 + 200  # 81 tiles: 7 are left over on 74 pairs
    x, w = operands(m, n, k, dev, 17)
    a, b = values(x), values(w).T
    y = fp8.linear_forward(x, w, out_dtype=torch.float32)
    assert ((y.double() - a @ b).abs() <= product_bound(a, b, torch.float32)).all()
    # the bound above grows with K; a part of a sum that is lost or added twice is far outside this
    assert (y.double() - a @ b).norm() / (a @ b).norm() < 1e-4
    for _ in range(3):
        assert torch.equal(y, fp8.linear_forward(x, w, out_dtype=torch.float32))


def loud_and_quiet(rows, cols, dev, block_rows=1, seed=0):
    """Block-scaled matrix whose neighbouring blocks differ by up to 2^24 in scale, drawn block by block: a block multiplied by
    the scale of another is far off."""
    from elf_b200.ops import fp8

    g = torch.Generator(device=dev).manual_seed(seed)
    q = (fp8.quantize if block_rows == 1 else fp8.quantize_weight)(torch.randn(rows, cols, device=dev, generator=g))
    scale = torch.randint(115, 140, q.scale.shape, device=dev, generator=g).to(torch.uint8)
    q.scale.copy_(scale)
    return q


@pytest.mark.parametrize("m,n,k", [(3000, 4100, 4200), (2304, 2304, 14336)])
def test_scales_belong_to_their_blocks(dev, m, n, k):
    """Scale words that the tensor core reads are those of the blocks it multiplies, in every tile and at every repetition."""
    from elf_b200.ops import fp8

    x, w = loud_and_quiet(m, k, dev, seed=1), loud_and_quiet(n, k, dev, 128, seed=2)
    a, b = values(x), values(w).T
    want, bound = a @ b, product_bound(a, b, torch.float32)
    first = fp8.linear_forward(x, w, out_dtype=torch.float32)
    assert ((first.double() - want).abs() <= bound).all()
    for _ in range(40):
        assert torch.equal(fp8.linear_forward(x, w, out_dtype=torch.float32), first)
    dy = loud_and_quiet(m, n, dev, seed=3)
    a, b = values(dy), values(w)
    want, bound = a @ b, product_bound(a, b, torch.float32)
    first = fp8.linear_input_grad(dy, w, torch.float32)
    assert ((first.double() - want).abs() <= bound).all()
    for _ in range(40):
        assert torch.equal(fp8.linear_input_grad(dy, w, torch.float32), first)


def test_gated_forms_repeat_themselves(dev):
    """Several units for every pair of CTAs, blocks of very different scales: every repetition gives the same bits."""
    from elf_b200.ops import fp8

    m, d, f = 3000, 1160, 3200
    x, wg, wd = loud_and_quiet(m, d, dev, seed=1), loud_and_quiet(2 * f, d, dev, 128, seed=2), loud_and_quiet(d, f, dev, 128, seed=3)
    dy, gate_up = loud_and_quiet(m, d, dev, seed=4), fp8.quantize(activations(m, 2 * f, torch.bfloat16, dev, 5))
    same_bits = lambda p, q: torch.equal(p.data.view(torch.uint8), q.data.view(torch.uint8)) and torch.equal(p.scale, q.scale)  # noqa: E731
    act, gu = fp8.gated_forward(x, wg)
    grad = fp8.gated_backward(dy, wd, gate_up)
    want, err = projections(x, wg, d)
    check_held(gu, want, err)
    for _ in range(40):
        for got, first in zip((*fp8.gated_forward(x, wg), fp8.gated_backward(dy, wd, gate_up)), (act, gu, grad)):
            assert same_bits(got, first)
