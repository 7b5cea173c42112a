"""Plain implementations, in 64 bits on the CPU, of the 8-bit activations and of the root-mean-square norm."""
import numpy as np
import torch

BLOCK = 128


def rows_of(shape, row_dims):
    lead = shape[:len(shape) - row_dims]
    return int(np.prod(lead, dtype=np.int64)), int(np.prod(shape[len(shape) - row_dims:], dtype=np.int64)), tuple(lead)


def encode(x, row_dims=2):
    """Codes (int8, the shape of x), scales and the values in 64 bits, of a CPU tensor; one block after another."""
    held = np.float64 if x.dtype == torch.float64 else np.float32
    rows, length, lead = rows_of(x.shape, row_dims)
    v = x.to(torch.float64).numpy().reshape(rows, length)
    blocks = -(-length // BLOCK)
    codes = np.zeros((rows, length), np.int8)
    scales = np.zeros((rows, blocks), held)
    values = np.zeros((rows, length))
    least = 2.0 ** (-900 if held == np.float64 else -100)
    for r in range(rows):
        for b in range(blocks):
            part = v[r, b * BLOCK:(b + 1) * BLOCK]
            finite = np.isfinite(part)
            top = held(np.abs(part[finite]).max()) if finite.any() else held(0)
            scale = inverse = held(0)
            if top >= least:
                inverse = held(126) / top
                scale = top * held(held(1) / held(126))
            number = np.where(finite, part, 0.0)
            code = np.rint(number.astype(np.longdouble) * np.longdouble(inverse)).astype(np.int64)
            code = np.where(finite, code, np.where(np.isnan(part), -128, np.where(part > 0, 127, -127)))
            codes[r, b * BLOCK:(b + 1) * BLOCK] = code
            scales[r, b] = scale
            values[r, b * BLOCK:(b + 1) * BLOCK] = np.where(finite, code * np.float64(scale), part)
    return codes.reshape(x.shape), scales.reshape(*lead, blocks), values.reshape(x.shape)


def decode(codes, scales, dtype):
    """The tensor that codes and scales stand for: products of a code and its scale in the type of the scales, rounded to dtype."""
    lead = scales.dim() - 1
    rows, length, _ = rows_of(codes.shape, codes.dim() - lead)
    q = codes.reshape(rows, length).to(scales.dtype)
    s = scales.reshape(rows, scales.shape[-1]).repeat_interleave(BLOCK, 1)[:, :length]
    v = q * s
    v[q == -128] = float("nan")
    v[q == 127] = float("inf")
    v[q == -127] = float("-inf")
    return v.reshape(codes.shape).to(dtype)


def along(weight, x, dim):
    return weight.double().reshape([-1] + [1] * (-1 - dim if dim < 0 else x.dim() - 1 - dim))


def rms_norm(s, weight, eps, dim):
    """y, unrounded, of a sum s of any type."""
    v = s.double()
    y = v / torch.sqrt((v * v).mean(dim, keepdim=True) + eps)
    return y if weight is None else y * along(weight, s, dim)


def rms_norm_backward(s, weight, gy, gsum, eps, dim):
    """Gradients of the sum and of the weight at s, and sums of magnitudes that bound their rounding errors."""
    v, g = s.double(), gy.double()
    u = g if weight is None else g * along(weight, s, dim)
    r = 1 / torch.sqrt((v * v).mean(dim, keepdim=True) + eps)
    pull = r * r * (u * v).mean(dim, keepdim=True)
    grad = r * (u - v * pull)
    # The products u s are rounded before they are added up, and may cancel: the error of their mean goes by their magnitudes.
    size = r * (u.abs() + v.abs() * r * r * (u * v).abs().mean(dim, keepdim=True))
    if gsum is not None:
        grad = grad + gsum.double()
        size = size + gsum.double().abs()
    each = g * v * r
    others = [d for d in range(s.dim()) if d != dim % s.dim()]
    if not others:
        return grad, each, size, each.abs()
    return grad, each.sum(others), size, each.abs().sum(others)
