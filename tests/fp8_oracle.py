"""The definition of block-scaled tensors and of the operators on them, in 64 bits and from the formulas."""

import torch

BLOCK = 128


def held(x, block_rows=1):
    """``(values, exponent bytes)`` a block-scaled copy of the matrix ``x`` must stand for: per block the
    smallest power of two s with max|x| <= 448 s over its finite values (not below 2^-126), each value the
    nearest multiple of s representable in e4m3 (ties to even), not finite -> NaN."""
    x = x.detach().double().cpu()
    rows, cols = x.shape
    fin = torch.isfinite(x)
    out = torch.full_like(x, float("nan"))
    nr, nc = -(-rows // block_rows), -(-cols // BLOCK)
    bytes_ = torch.empty(nr, nc, dtype=torch.uint8)
    mag = torch.where(fin, x.abs(), 0.0)
    for i in range(nr):
        r = slice(i * block_rows, (i + 1) * block_rows)
        for j in range(nc):
            c = slice(j * BLOCK, (j + 1) * BLOCK)
            top = mag[r, c].max().item()
            e = -126
            while 448.0 * 2.0**e < top:
                e += 1
            bytes_[i, j] = e + 127
            u = x[r, c] / 2.0**e
            step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0**-6))) - 3)  # 3 fraction bits, subnormals below 2^-6
            v = torch.round(u / step) * step * 2.0**e
            out[r, c] = torch.where(fin[r, c], v, float("nan"))
    return out, bytes_


def values(q):
    """64-bit values of a ``BlockScaled`` (on its device)."""
    data = q.data.reshape(-1, q.data.shape[-1])
    scale = q.scale.reshape(-1, q.scale.shape[-1])
    r = torch.arange(data.shape[0], device=data.device) // q.block_rows
    c = torch.arange(data.shape[1], device=data.device) // BLOCK
    return data.double() * torch.exp2(scale.double() - 127)[r[:, None], c[None, :]]


def product_bound(a, b, out_dtype):
    """Elementwise bound on the error of ``a @ b`` accumulated in fp32 and rounded once to ``out_dtype``: each of
    the K additions is off by at most one unit (2^-23, truncation allowed) of a running sum that never exceeds
    sum |a||b|; the rounding adds half a step of the result, or half the smallest subnormal."""
    k = a.shape[1]
    mag = a.abs() @ b.abs()
    y = a @ b
    half = torch.finfo(out_dtype).eps / 2
    return k * 2.0**-23 * mag + half * (y.abs() + k * 2.0**-23 * mag) + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
