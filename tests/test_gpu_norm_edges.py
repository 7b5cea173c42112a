"""The root-mean-square norm where its variants meet: many groups of blocks a warp, the shared memory that long norms ask for, factors
out of float's range, weights of another type, calls from several threads."""
import ctypes

import pytest
import torch

import morphocore_b200.functional as F
from test_activation8 import Norm
from test_gpu_rms_norm import EPS, TYPES, cuda, row_dims_of, tensors

pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.float64: 1, torch.float16: 2, torch.bfloat16: 3}


def norm_desc(x, dim, eps=EPS, flags=0):
    inner = x[0].numel() // x.shape[1] if dim == -3 else 1
    return Norm(x.numel() // x.shape[dim] // inner, x.shape[dim], inner, eps, CODE[x.dtype], flags)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,dim", [((3, 64, 40, 36), -3), ((2, 250, 13, 11), -3), ((2, 512, 17, 16), -3), ((300, 4096), -1), ((40, 16384), -1)], ids=str)
def test_scales_of_warps_with_many_blocks(shape, dim, dtype):
    """A warp that encodes several groups of blocks writes each scale once: those of encode_8bit, every time."""
    from _cabi import check, lib, ptr, stream
    x, r, w, _ = cuda(*tensors(shape, dim, dtype))
    y, total = F.rms_norm(x, w, r, EPS, dim)
    wants = [F.encode_8bit(t, row_dims_of(x, dim)) for t in (y, total)]
    d = norm_desc(x, dim)
    for _ in range(20):
        codes = [torch.full_like(p.codes, 99) for p in wants]
        scales = [torch.full_like(p.scales, -1.0) for p in wants]
        check(lib.mc_rms_norm_forward(ctypes.byref(d), ptr(x), ptr(r), ptr(w), ptr(total), None, ptr(codes[0]), ptr(scales[0]), ptr(codes[1]), ptr(scales[1]), stream()))
        for c, s, p in zip(codes, scales, wants):
            assert bool((c == p.codes).all()) and bool((s == p.scales).all())
