"""Linear layers, norms and activation checkpoints in 8 bits (kernels in ``elf_b200/csrc/fp8_ops.cu``,
``fp8_gemm_sm100.cu`` and ``fp8_gemm_sm100_2cta.cu``).

A ``BlockScaled`` tensor holds e4m3 values and one power-of-two scale per block of 128 columns,
for each row (activations, gradients) or for each 128 rows (weights).  A block's scale is the smallest
power of two ``s`` with ``max |x| <= 448 s`` over its finite values; each value is rounded once, to the
nearest e4m3 multiple of ``s`` (relative error at most 2^-4; absolute at most ``2^-10 s`` where the
value is below ``2^-6 s``).  What is not finite becomes NaN.  Powers of two cost no significant bits,
so a restored value is exact in bf16 and the tensor core can apply the scales itself.

=====================  ==============================================  ================================
operator               computes                                        reduction blocks lie along
=====================  ==============================================  ================================
``quantize``           block-scaled copy of an activation
``quantize_weight``    the same with 128 x 128 tiles
``rms_norm``           block-scaled ``rmsnorm(x) * w``
``add_rms_norm``       the same of ``x + residual``
``linear_forward``     ``Y = X W^T``                                   X's and W's columns
``linear_input_grad``  ``dX = dY W``                                   dY's columns, W's rows
``linear_weight_grad`` ``dW = dY^T X`` (operands restored to bf16:     (tokens: no common scale)
                       a token's scale is not common to a block of
                       the reduction)
``gated_forward``      ``silu(X Wg^T) * (X Wu^T)`` block-scaled
``gated_backward``     gradient of gate and up from their checkpoint
=====================  ==============================================  ================================

``linear`` and ``gated_ffn`` are the differentiable forms: what they keep for the backward pass they keep
in 8 bits.  ``elf_b200.zb_utils.LinearFP8DW`` is the split-backward layer on top of them.

CUDA tensors run on this package's kernels; CPU tensors (and ``ELF_B200_DISABLE_KERNELS=1``) take a
plain torch form of the same arithmetic.  All entry points run on the current stream of the tensors'
device, allocate their results, and do not synchronise.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _ext
from . import gemm as _gemm

__all__ = [
    "BLOCK",
    "BlockScaled",
    "quantize",
    "quantize_weight",
    "dequantize",
    "rms_norm",
    "add_rms_norm",
    "linear_forward",
    "linear_input_grad",
    "linear_weight_grad",
    "gated_forward",
    "gated_backward",
    "linear",
    "gated_ffn",
]

BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_E4M3_MAX = 448.0
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _round_up(n: int, m: int) -> int:
    return -(-n // m) * m


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


class BlockScaled:
    """e4m3 values and their power-of-two scales: ``value = data * 2^(scale - 127)``.

    ``data``        float8_e4m3fn ``[..., cols]``
    ``scale``       uint8 biased exponents ``[..., ceil(cols / 128)]``; with ``block_rows = 128`` (matrices
                    only) ``[ceil(rows / 128), ceil(cols / 128)]``
    ``block_rows``  rows that share a scale: 1 or 128

    Rows may be padded in memory (the products want row pitches that are multiples of 16 bytes;
    ``quantize`` allocates them so).  Operands whose rows are not are copied by the products."""

    __slots__ = ("data", "scale", "block_rows", "is_model_input")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, block_rows: int = 1):
        if data.dtype != _E4M3 or scale.dtype != torch.uint8:
            raise TypeError(f"block-scaled data must be float8_e4m3fn with uint8 exponents, got {data.dtype} and {scale.dtype}")
        if block_rows not in (1, BLOCK):
            raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
        if data.dim() < 1 or (block_rows == BLOCK and data.dim() != 2):
            raise ValueError(f"block-scaled data must have a last dimension to scale along (a matrix for tiles), got shape {tuple(data.shape)}")
        lead = (_blocks(data.shape[0]),) if block_rows == BLOCK else tuple(data.shape[:-1])
        expected = (*lead, _blocks(data.shape[-1]))
        if tuple(scale.shape) != expected:
            raise ValueError(f"expected exponents of shape {expected} for data {tuple(data.shape)}, got {tuple(scale.shape)}")
        if data.device != scale.device:
            raise ValueError(f"data is on {data.device}, its scales on {scale.device}")
        self.data, self.scale, self.block_rows = data, scale, block_rows
        self.is_model_input = False

    @classmethod
    def _made(cls, data: torch.Tensor, scale: torch.Tensor, block_rows: int = 1) -> "BlockScaled":
        """Without the checks: for what this module's own kernels return."""
        self = object.__new__(cls)
        self.data, self.scale, self.block_rows, self.is_model_input = data, scale, block_rows, False
        return self

    @property
    def shape(self) -> torch.Size:
        return self.data.shape

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.nbytes + self.scale.nbytes

    def numel(self) -> int:
        return self.data.numel()

    def to(self, device, non_blocking: bool = False) -> "BlockScaled":
        moved = BlockScaled._made(self.data.to(device, non_blocking=non_blocking), self.scale.to(device, non_blocking=non_blocking), self.block_rows)
        moved.is_model_input = self.is_model_input
        return moved

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"BlockScaled(shape={tuple(self.shape)}, block_rows={self.block_rows}, device={self.device})"


def _on_kernels(t: torch.Tensor) -> bool:
    if not (t.is_cuda and _gemm._ENABLED):
        return False
    if _ext._module is None:
        _ext.require_on_gpu()
    return True


def _shift(q: BlockScaled) -> int:
    return 7 if q.block_rows == BLOCK else 0


def _new(shape, block_rows: int, device) -> BlockScaled:
    """Uninitialised block-scaled tensor with the row pitches the products want."""
    *lead, cols = shape
    data = torch.empty((*lead, _round_up(cols, 16)), dtype=torch.uint8, device=device).view(_E4M3)[..., :cols]
    rows = (_blocks(lead[0]),) if block_rows == BLOCK else tuple(lead)
    scale = torch.empty((*rows, _round_up(_blocks(cols), 4)), dtype=torch.uint8, device=device)[..., : _blocks(cols)]
    return BlockScaled(data, scale, block_rows)


def _matrix(t: torch.Tensor) -> torch.Tensor:
    """``[..., cols]`` as a matrix with a contiguous last dimension (a copy only where strides force one)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(t.shape[:-1].numel(), t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _need_float(t: torch.Tensor, name: str) -> None:
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name} must be bf16, fp16 or fp32, got {t.dtype}")


def _no_tangent(what: str, *tensors) -> None:
    # a dual tensor need not require grad: past the autograd function its tangent would be lost without a word
    if getattr(_forward_ad, "_current_level", 0) < 0:  # spares small calls a look at every tensor
        return
    if any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: forward-mode derivatives are not implemented")


def _same_device(name: str, t, other: str, u) -> None:
    if u is not None and u.device != t.device:
        raise ValueError(f"{other} is on {u.device}, {name} on {t.device}")


# ------------------------------------------------------------------------------ plain torch forms


def _factors(q: BlockScaled) -> torch.Tensor:
    rows, cols = _matrix(q.data).shape
    e = _matrix(q.scale).to(torch.int32)
    f = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e - 127)
    f = torch.where(e == 255, float("nan"), f)
    return f.repeat_interleave(q.block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _values(q: BlockScaled) -> torch.Tensor:
    """fp32 matrix of the values."""
    return _matrix(q.data).float() * _factors(q)


def _quantize_ref(x: torch.Tensor, block_rows: int) -> BlockScaled:
    q = _new(x.shape, block_rows, x.device)
    if x.numel() == 0:
        return q
    x2 = _matrix(x).float()
    rows, cols = x2.shape
    finite = torch.isfinite(x2)
    mag = torch.where(finite, x2.abs(), 0.0)
    mag = torch.nn.functional.pad(mag, (0, -cols % BLOCK, 0, -rows % block_rows))
    top = mag.view(mag.shape[0] // block_rows, block_rows, mag.shape[1] // BLOCK, BLOCK).amax((1, 3))
    mantissa, exponent = torch.frexp(top)
    byte = exponent - 9 + (mantissa > 0.875).to(exponent.dtype) + 127
    byte = torch.where(top > 0, byte, 1).clamp(1, 254).to(torch.uint8)
    q.scale.copy_(byte.view(q.scale.shape))
    v = x2 / _factors(q)
    v = torch.where(finite, v.clamp(-_E4M3_MAX, _E4M3_MAX), float("nan"))
    q.data.copy_(v.to(_E4M3).view(q.data.shape))
    return q


def _rms_ref(h: torch.Tensor, w: torch.Tensor, eps: float):
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + eps)
    return _quantize_ref(hf * rstd * w.float(), 1), rstd.squeeze(-1)


# ------------------------------------------------------------------------------ quantise, restore


def _quantize(x: torch.Tensor, block_rows: int) -> BlockScaled:
    _need_float(x, "x")
    if not _on_kernels(x):
        return _quantize_ref(x.detach(), block_rows)
    return BlockScaled._made(*_ext.get().fp8_quantize(x, block_rows == BLOCK), block_rows)


def quantize(x: torch.Tensor) -> BlockScaled:
    """Block-scaled copy of ``x [..., cols]`` (bf16, fp16 or fp32): one scale per row and 128 columns.
    Not differentiable; see ``linear`` and ``gated_ffn``."""
    if x.dim() < 1:
        raise ValueError("quantize needs a tensor with at least one dimension")
    return _quantize(x, 1)


def quantize_weight(w: torch.Tensor) -> BlockScaled:
    """Block-scaled copy of a matrix with one scale per tile of 128 x 128, usable in ``linear_forward`` and,
    transposed, in ``linear_input_grad``."""
    if w.dim() != 2:
        raise ValueError(f"quantize_weight needs a matrix, got shape {tuple(w.shape)}")
    return _quantize(w, BLOCK)


def dequantize(q: BlockScaled, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values ``q`` stands for: exact in fp32 and, from 2^-133 up, in bf16; in fp16 rounded, and infinite above 65504.
    ``out``: tensor to write instead of a new one; its last dimension contiguous, its rows evenly spaced."""
    if out is None:
        if dtype not in _FLOATS:
            raise TypeError(f"dequantize gives bf16, fp16 or fp32, not {dtype}")
    else:
        _need_float(out, "out")
        if not (out.shape == q.shape and out.device == q.device):
            raise ValueError("out does not match the block-scaled tensor")
    if not _on_kernels(q.data):
        y = _values(q).view(q.shape)
        return y.to(dtype) if out is None else out.copy_(y)
    return _ext.get().fp8_dequantize(q.data, q.scale, _shift(q), dtype, out)


# ------------------------------------------------------------------------------ RMSNorm


def _norm(x, residual, w, eps):
    dim = x.shape[-1]
    if not (x.dim() >= 1 and w.dim() == 1 and w.numel() == dim):
        raise ValueError(f"the gain must have {dim} elements, got shape {tuple(w.shape)}")
    if not (residual is None or (residual.shape == x.shape and residual.dtype == x.dtype)):
        raise ValueError("the residual must match x")
    _same_device("x", x, "the gain", w)
    _same_device("x", x, "the residual", residual)
    _need_float(x, "x")
    fits = x.dtype == torch.bfloat16 and w.dtype == torch.bfloat16 and dim % 8 == 0 and 0 < dim <= 8192
    if not (fits and _on_kernels(x)):
        x, w = x.detach(), w.detach()
        h = x if residual is None else x + residual.detach()
        q, rstd = _rms_ref(h, w, eps)
        return q, rstd, h
    data, scale, rstd, h = _ext.get().fp8_rmsnorm(x, w, eps, residual)
    return BlockScaled._made(data, scale), rstd, h


class _AddNorm(torch.autograd.Function):
    """``add_rms_norm`` as a node of the graph: the residual stream passes its gradient on to both terms."""

    @staticmethod
    def forward(x, residual, w, eps):
        q, rstd, h = _norm(x, residual, w, eps)
        return h, q.data, q.scale, rstd

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.mark_non_differentiable(*output[1:])
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, dh, *_):
        return dh, dh, None, None


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-5) -> Tuple[BlockScaled, torch.Tensor]:
    """``(q, rstd)``: ``x * rstd * w`` in 8 bits with ``rstd = (mean(x^2) + eps)^-1/2`` in fp32, the statistic
    that ``elf_b200.ops.fused``'s RMSNorm backward takes; neither is differentiable.  One pass over ``x``; the kernel handles bf16 with a width that
    is a multiple of 8, at most 8192, as ``fused.rms_norm`` does, other inputs take torch operations."""
    q, rstd, _ = _norm(x, None, w, eps)
    return q, rstd


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, w: torch.Tensor, eps: float = 1e-5) -> Tuple[BlockScaled, torch.Tensor, torch.Tensor]:
    """``(q, rstd, h)`` with ``h = x + residual`` (rounded to the inputs' type; the norm is that of the
    rounded sum, which is what later passes read back).  ``h`` is differentiable, ``q`` and ``rstd`` are not."""
    _no_tangent("add_rms_norm", x, residual)
    if residual is None or not (torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad)):
        return _norm(x, residual, w, eps)
    h, data, scale, rstd = _AddNorm.apply(x, residual, w, eps)
    return BlockScaled._made(data, scale), rstd, h


# ------------------------------------------------------------------------------ products


def _check_product(a: BlockScaled, b: BlockScaled, reduce_b: int, what: str) -> None:
    if a.block_rows != 1:
        raise ValueError(f"{what}: the activation or gradient must be scaled by rows")
    if b.data.dim() != 2:
        raise ValueError(f"{what}: the weight must be a matrix")
    if a.shape[-1] != b.shape[reduce_b]:
        raise ValueError(f"{what}: reduction lengths {a.shape[-1]} and {b.shape[reduce_b]} differ")
    _same_device("the activation", a, "the weight", b)


def _product(a: BlockScaled, b: BlockScaled, transposed: bool, bias, out_dtype) -> torch.Tensor:
    if out_dtype not in _FLOATS:
        raise TypeError(f"products come in bf16, fp16 or fp32, not {out_dtype}")
    n = b.shape[1] if transposed else b.shape[0]
    if a.numel() == 0 or n == 0 or not _on_kernels(a.data):
        y = _values(a) @ (_values(b) if transposed else _values(b).T)
        if bias is not None:
            y = y + bias.float()
        return y.to(out_dtype).view(*a.shape[:-1], n)
    bias = None if bias is None else bias.detach().to(out_dtype).contiguous()
    return _ext.get().fp8_gemm(a.data, a.scale, b.data, b.scale, _shift(b), transposed, out_dtype, bias, _gemm.status(a.device))


class _Biased(torch.autograd.Function):
    """``linear_forward`` as a node of the graph: its bias has a gradient, its 8-bit operands have none."""

    @staticmethod
    def forward(bias, x, w, out_dtype):
        return _product(x, w, False, bias, out_dtype)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.dtype = inputs[0].dtype

    @staticmethod
    def backward(ctx, dy):
        return _bias_grad(dy, ctx.dtype), None, None, None


def _bias_grad(dy: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return _matrix(dy).float().sum(0).to(dtype)


def linear_forward(x: BlockScaled, w: BlockScaled, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x W^T (+ bias)`` for ``x [..., K]`` scaled by rows and ``w [N, K]`` scaled by tiles or rows; accumulated in
    fp32 and rounded once.  On the GPU a bias of another type is taken in ``out_dtype``, the type a layer of that type holds
    it in.  The result is differentiable with respect to the bias; ``linear`` is the form for all operands."""
    _check_product(x, w, 1, "linear_forward")
    if not (bias is None or (bias.shape == (w.shape[0],) and bias.device == w.device)):
        raise ValueError("linear_forward: the bias must be a vector with one element per output")
    _no_tangent("linear_forward", bias)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        return _Biased.apply(bias, x, w, out_dtype)
    return _product(x, w, False, bias, out_dtype)


def linear_input_grad(dy: BlockScaled, w: BlockScaled, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dy W`` for ``dy [..., N]`` scaled by rows and ``w [N, K]`` scaled by tiles.  The weight is read as it
    lies: the tensor core takes it transposed, and a tile's scale serves both directions."""
    _check_product(dy, w, 0, "linear_input_grad")
    if w.block_rows != BLOCK:
        raise ValueError("linear_input_grad: the weight must be scaled in tiles of 128 x 128 (quantize_weight)")
    return _product(dy, w, True, None, out_dtype)


def _restored(t: Union[BlockScaled, torch.Tensor]) -> torch.Tensor:
    """bf16 matrix for the 16-bit weight-gradient product, exact for a block-scaled tensor."""
    return _matrix(t.dequantize() if isinstance(t, BlockScaled) else t.detach())


def linear_weight_grad(dy: Union[BlockScaled, torch.Tensor], x: Union[BlockScaled, torch.Tensor], out: Optional[torch.Tensor] = None,
                       out_dtype: torch.dtype = torch.bfloat16, push: Optional[dict] = None) -> torch.Tensor:
    """``dy^T x`` summed over all leading dimensions, from 8-bit checkpoints or 16-bit tensors, on the bf16
    tensor path: the reduction runs over tokens, which have scales of their own.  Accumulated in fp32 and rounded
    once, the same from call to call; fp16 and fp32 operands enter whole, as two and three bf16 parts, each with a
    stretch of the reduction.  Added to ``out`` when it is given (bf16 or fp32); ``push`` as in ``gemm.linear_weight_grad``, from 8-bit or
    bf16 operands."""
    n, k = dy.shape[-1], x.shape[-1]
    if dy.shape[:-1].numel() != x.shape[:-1].numel():
        raise ValueError("linear_weight_grad: dy and x have different numbers of rows")
    if any(isinstance(t, BlockScaled) and t.block_rows != 1 for t in (dy, x)):
        raise ValueError("linear_weight_grad: activations and gradients must be scaled by rows")
    _same_device("dy", dy, "x", x)
    for name, t in (("dy", dy), ("x", x)):
        if not isinstance(t, BlockScaled):
            _need_float(t, name)
            if push and t.dtype != torch.bfloat16:
                raise ValueError(f"linear_weight_grad: a push takes 8-bit or bf16 operands, got {name} in {t.dtype}")
    if not (out is None or (out.shape == (n, k) and out.device == x.device and out.dtype in (torch.bfloat16, torch.float32))):
        raise ValueError(f"linear_weight_grad: out must be a bf16 or fp32 matrix [{n}, {k}]")
    if out_dtype not in _FLOATS:
        raise TypeError(f"products come in bf16, fp16 or fp32, not {out_dtype}")
    data = x.data if isinstance(x, BlockScaled) else x
    if data.numel() == 0 or n == 0 or not _on_kernels(data):
        if push:
            raise ValueError("linear_weight_grad: only the product of CUDA operands that have elements can be pushed")
        plain = lambda t: _values(t) if isinstance(t, BlockScaled) else _matrix(t.detach()).float()  # noqa: E731
        dw = plain(dy).T @ plain(x)
        return dw.to(out_dtype) if out is None else out.add_(dw)
    if not push:
        pair = lambda t: (t.data, t.scale) if isinstance(t, BlockScaled) else (t.detach(), None)  # noqa: E731
        return _ext.get().fp8_weight_grad(*pair(dy), *pair(x), out, out_dtype, _gemm.status(data.device), _gemm._VARIANT, _gemm._SPLIT_TAIL)
    if out is None or k % 8 or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("linear_weight_grad: a push needs a gradient buffer the product can add to in place")
    return _gemm.linear_weight_grad(_restored(dy), _restored(x), out=out, push=push)


# ------------------------------------------------------------------------------ gated feed-forward block


def gated_forward(x: BlockScaled, w_gate_up: BlockScaled, keep: bool = True) -> Tuple[BlockScaled, Optional[BlockScaled]]:
    """``(act, gate_up)`` for ``x [..., K]`` and ``w_gate_up [2F, K]`` (gate rows, then up rows; F a multiple of 128):
    ``act = silu(x Wg^T) * (x Wu^T)`` in 8 bits and, with ``keep``, the two projections in 8 bits for
    ``gated_backward``.  One kernel: the projections stay in fp32 until the activation is formed."""
    _check_product(x, w_gate_up, 1, "gated_forward")
    f2 = w_gate_up.shape[0]
    if f2 % (2 * BLOCK):
        raise ValueError(f"gated_forward: the width of gate and of up must be a multiple of {BLOCK}, got {f2} rows in all")
    f = f2 // 2
    if x.numel() == 0 or f == 0 or not _on_kernels(x.data):
        gu = _values(x) @ _values(w_gate_up).T
        act = torch.nn.functional.silu(gu[:, :f]) * gu[:, f:]
        lead = x.shape[:-1]
        return _quantize_ref(act.view(*lead, f), 1), _quantize_ref(gu.view(*lead, f2), 1) if keep else None
    act, act_scale, gu, gu_scale = _ext.get().fp8_gated(x.data, x.scale, w_gate_up.data, w_gate_up.scale, _shift(w_gate_up), keep, _gemm.status(x.device))
    return BlockScaled._made(act, act_scale), BlockScaled._made(gu, gu_scale) if keep else None


def gated_backward(dy: BlockScaled, w_down: BlockScaled, gate_up: BlockScaled) -> BlockScaled:
    """Gradient of ``gate_up [..., 2F]`` in 8 bits for the gradient ``dy [..., D]`` of the block's output:
    one kernel, ``dact = dy W_down`` in fp32 and ``dgate = dact up s (1 + gate (1 - s))`` and ``dup = dact gate s`` with
    ``s = sigmoid(gate)``, gate and up restored from their checkpoint."""
    _check_product(dy, w_down, 0, "gated_backward")
    f = w_down.shape[1]
    if w_down.block_rows != BLOCK:
        raise ValueError("gated_backward: the weight must be scaled in tiles of 128 x 128 (quantize_weight)")
    if f % BLOCK:
        raise ValueError(f"gated_backward: the width of gate and of up must be a multiple of {BLOCK}, got {f}")
    if not (gate_up.block_rows == 1 and gate_up.shape == (*dy.shape[:-1], 2 * f)):
        raise ValueError(f"gated_backward: expected gate_up of shape {(*dy.shape[:-1], 2 * f)}, got {tuple(gate_up.shape)}")
    _same_device("dy", dy, "gate_up", gate_up)
    if dy.numel() == 0 or f == 0 or not _on_kernels(dy.data):
        dact = _values(dy) @ _values(w_down)
        gu = _values(gate_up)
        gate, up = gu[:, :f], gu[:, f:]
        s = torch.sigmoid(gate)
        dgu = torch.cat([dact * up * s * (1 + gate * (1 - s)), dact * gate * s], 1)
        return _quantize_ref(dgu.view(gate_up.shape), 1)
    return BlockScaled._made(*_ext.get().fp8_gated_bwd(dy.data, dy.scale, w_down.data, w_down.scale, gate_up.data, gate_up.scale, _gemm.status(dy.device)))


# ------------------------------------------------------------------------------ differentiable forms


def _weight_copy(q: Optional[BlockScaled], w: torch.Tensor, name: str) -> BlockScaled:
    if q is None:
        return quantize_weight(w)
    if q.data.shape != w.shape or q.block_rows != BLOCK or q.data.device != w.device:
        raise ValueError(f"{name}: the 8-bit copy does not belong to a weight of shape {tuple(w.shape)} on {w.device}")
    return q


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, q):
        xq = quantize(x)
        # the weight's own tensor is saved when no 8-bit copy was given: the backward makes it
        # again instead of holding one per call in flight
        ctx.given = q is not None
        ctx.w_dtype, ctx.x_dtype, ctx.bias_dtype = w.dtype, x.dtype, None if bias is None else bias.dtype
        ctx.save_for_backward(xq.data, xq.scale, *((q.data, q.scale) if q is not None else (w,)))
        return linear_forward(xq, _weight_copy(q, w, "linear"), bias, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        data, scale, *weight = ctx.saved_tensors
        dx = dw = db = None
        dyq = quantize(dy) if ctx.needs_input_grad[0] or ctx.needs_input_grad[1] else None
        if ctx.needs_input_grad[0]:
            wq = BlockScaled._made(*weight, BLOCK) if ctx.given else quantize_weight(weight[0])
            dx = linear_input_grad(dyq, wq, ctx.x_dtype)
        if ctx.needs_input_grad[1]:
            dw = linear_weight_grad(dyq, BlockScaled._made(data, scale), out_dtype=ctx.w_dtype)
        if ctx.needs_input_grad[2]:
            db = _bias_grad(dy, ctx.bias_dtype)
        return dx, dw, db, None


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, w_q: Optional[BlockScaled] = None) -> torch.Tensor:
    """``x W^T (+ bias)`` with the products in 8 bits and ``x`` kept in 8 bits for the weight gradient.

    ``w_q``: the weight's block-scaled copy (``quantize_weight(w)``), which a training loop makes once per
    optimizer step; without it every call makes its own.  The gradients are those of the product with the
    rounded operands, passed through the rounding unchanged; reverse mode only."""
    _check_differentiable("linear", x, w, bias)
    if not (w.dim() == 2 and x.dim() >= 1 and x.shape[-1] == w.shape[1]):
        raise ValueError(f"linear: x {tuple(x.shape)} does not match a weight of shape {tuple(w.shape)}")
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias))):
        return linear_forward(quantize(x), _weight_copy(w_q, w, "linear"), bias, x.dtype)
    return _Linear.apply(x, w, bias, w_q)


def _ffn_forward(x: torch.Tensor, gate_up_q: BlockScaled, down_q: BlockScaled, keep: bool):
    """``(y, [x, act, gate_up])``: the output and, with ``keep``, values and scales of what the backward needs."""
    if x.numel() and down_q.numel() and _on_kernels(x):
        y, *kept = _ext.get().fp8_ffn(x, gate_up_q.data, gate_up_q.scale, down_q.data, down_q.scale, keep, _gemm.status(x.device))
        return y, kept
    xq = quantize(x)
    act, gu = gated_forward(xq, gate_up_q, keep)
    y = linear_forward(act, down_q, None, x.dtype)
    return y, [t for q in (xq, act, gu) for t in (q.data, q.scale)] if keep else []


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate_up, w_down, gate_up_q, down_q):
        y, kept = _ffn_forward(x, _weight_copy(gate_up_q, w_gate_up, "gated_ffn"), _weight_copy(down_q, w_down, "gated_ffn"), True)
        ctx.given = (gate_up_q is not None, down_q is not None)
        ctx.dtypes = (x.dtype, w_gate_up.dtype, w_down.dtype)
        held = [t for q, w in ((gate_up_q, w_gate_up), (down_q, w_down)) for t in ((q.data, q.scale) if q is not None else (w,))]
        ctx.save_for_backward(*kept, *held)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        tensors = ctx.saved_tensors
        kept, rest = tensors[:6], tensors[6:]
        copies = []
        for given in ctx.given:
            n = 2 if given else 1
            copies.append(BlockScaled._made(*rest[:n], BLOCK) if given else quantize_weight(rest[0]))
            rest = rest[n:]
        gate_up_q, down_q = copies
        need = list(ctx.needs_input_grad[:3])
        if dy.numel() and gate_up_q.numel() and down_q.numel() and _on_kernels(dy):
            grads = _ext.get().fp8_ffn_bwd(dy, list(kept), gate_up_q.data, gate_up_q.scale, down_q.data, down_q.scale, need, list(ctx.dtypes),
                                           _gemm.status(dy.device), _gemm._VARIANT, _gemm._SPLIT_TAIL)
            return (*grads, None, None)
        xq, act, gu = (BlockScaled._made(kept[2 * i], kept[2 * i + 1]) for i in range(3))
        x_dtype, gate_up_dtype, down_dtype = ctx.dtypes
        dx = dw_gate_up = dw_down = None
        if need[2]:
            dw_down = linear_weight_grad(dy, act, out_dtype=down_dtype)
        if need[0] or need[1]:
            dgu = gated_backward(quantize(dy), down_q, gu)
            if need[0]:
                dx = linear_input_grad(dgu, gate_up_q, x_dtype)
            if need[1]:
                dw_gate_up = linear_weight_grad(dgu, xq, out_dtype=gate_up_dtype)
        return dx, dw_gate_up, dw_down, None, None


def gated_ffn(x: torch.Tensor, w_gate_up: torch.Tensor, w_down: torch.Tensor, gate_up_q: Optional[BlockScaled] = None,
              down_q: Optional[BlockScaled] = None) -> torch.Tensor:
    """``(silu(x Wg^T) * (x Wu^T)) W_down^T`` for ``x [..., D]``, ``w_gate_up [2F, D]`` (gate rows, then up rows, F a
    multiple of 128) and ``w_down [D', F]``, with the products in 8 bits.

    The backward pass works from 8-bit copies of ``x``, of the activation and of the two projections:
    ``D + 3F`` bytes a token against ``2 D + 6 F`` in bf16.  ``gate_up_q``, ``down_q``: block-scaled copies of the
    weights, as in ``linear``."""
    _check_differentiable("gated_ffn", x, w_gate_up, w_down)
    if not (w_gate_up.dim() == 2 and w_down.dim() == 2 and x.dim() >= 1 and x.shape[-1] == w_gate_up.shape[1] and w_gate_up.shape[0] == 2 * w_down.shape[1]):
        raise ValueError(f"gated_ffn: shapes x {tuple(x.shape)}, w_gate_up {tuple(w_gate_up.shape)}, w_down {tuple(w_down.shape)} do not match")
    if w_down.shape[1] % BLOCK:
        raise ValueError(f"gated_ffn: the inner width must be a multiple of {BLOCK}, got {w_down.shape[1]}")
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate_up, w_down))):
        return _ffn_forward(x, _weight_copy(gate_up_q, w_gate_up, "gated_ffn"), _weight_copy(down_q, w_down, "gated_ffn"), False)[0]
    return _GatedFFN.apply(x, w_gate_up, w_down, gate_up_q, down_q)


def _check_differentiable(what: str, x: torch.Tensor, *others) -> None:
    _no_tangent(what, x, *others)
    for t in (x, *others):
        if t is not None:
            _need_float(t, what)
            if t.device != x.device:
                raise ValueError(f"{what}: all tensors must be on one device, got {t.device} and {x.device}")
