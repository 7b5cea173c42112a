"""The root-mean-square norm where its variants meet: many groups of blocks a warp, the shared memory that long norms ask for, factors
out of float's range, weights of another type, calls from several threads."""
import ctypes

import pytest
import torch

import _plain8 as P
import morphocore_b200.functional as F
import morphocore_b200.nn as Mnn
from test_activation8 import Norm
from test_gpu_rms_norm import EPS, TYPES, cuda, grad_bound, make, row_dims_of, tensors, value_bound, weight_bound, within

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


def check_gradients(shape, dim, dtype, keep8, residual, weight, lane_terms):
    """Gradients against 64 bits. Beside the roundings that grad_bound and weight_bound count, `lane_terms` of each: a lane adds that many squares
    and products one after the other in float (what comes of the lanes is added in double). Either sum is then off by at most
    lane_terms half steps of its terms' magnitudes, r by half as much, r^2 mean(u s) by twice: with r's own 2.5 lane_terms half steps of `size`."""
    x, r, w, s = tensors(shape, dim, dtype, residual, weight)
    gy, gs = make(shape, dtype, 4), make(shape, dtype, 5) if residual else None
    leaves = [None if t is None else t.requires_grad_(True) for t in cuda(x, w, r)]
    out = F.checkpoint_8bit(F.rms_norm, *leaves, EPS, dim) if keep8 else F.rms_norm(*leaves, EPS, dim)
    at = s
    if keep8:
        kept = F.encode_8bit(s.cuda(), row_dims_of(x, dim))
        at = P.decode(kept.codes.cpu(), kept.scales.cpu(), dtype)
    want, want_w, size, size_w = P.rms_norm_backward(at, w, gy, gs, EPS, dim)
    got = torch.autograd.grad(out, [t for t in leaves if t is not None], [gy.cuda(), gs.cuda()] if residual else gy.cuda())
    more = 0 if dtype == torch.float64 else 2.5 * lane_terms * 2.0 ** -24
    within(got[0], want, grad_bound(size, want, dtype, shape[dim]) + more * size, "x")
    if weight:
        within(got[1], want_w, weight_bound(size_w, want_w, dtype, channels=shape[dim]) + more * size_w, "weight")


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_maps_of_many_channels(dtype, keep8):
    """Backward passes whose sums of gweight take more and more shared memory, the smallest first: no call relies on the opt-in of one
    with more channels before it. 1792 and 3840 channels are where double leaves 48 KiB with and without what the kernel declares."""
    for channels in (513, 1792, 1793, 2048, 3840, 3841, 8200, 16384):
        for inner in ((2, 2), (1, 3)):
            for residual, weight in ((True, True), (False, True), (False, False)):
                check_gradients((2, channels, *inner), -3, dtype, keep8, residual, weight, -(-channels // 16))


def in_threads(*calls, times):
    """Each call in a thread of its own, `times` times over; ctypes gives up the interpreter's lock meanwhile."""
    import threading
    failed, start = [], threading.Barrier(len(calls))

    def work(call):
        start.wait()
        for _ in range(times):
            rc = call()
            if rc != 0:
                failed.append(rc)

    threads = [threading.Thread(target=work, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return failed


def test_threads_whose_launches_need_different_amounts_of_shared_memory():
    """Two threads launch the same kernel with different amounts of shared memory, each above what needs no opt-in: none is refused, and
    the results are those of calls one after the other."""
    from _cabi import check, lib, make_desc, ptr, stream
    at = stream()
    calls, results, wants = [], [], []
    for width in (4096, 2800):   # 72 and 52 KiB of the per-channel forward pass with codes, 5 x 5
        x, w = torch.randn(1, 1, 8, width, device="cuda"), torch.randn(1, 1, 5, 5, device="cuda")
        y, p = torch.empty_like(x), F.encode_8bit(x)
        codes, scales = torch.empty_like(p.codes), torch.empty_like(p.scales)
        d = make_desc("dilation", x, w, "identity")
        calls.append(lambda d=d, t=(x, w, y, codes, scales): lib.mc_morpho_forward8(ctypes.byref(d), *map(ptr, t), at))
        results.append((y, codes, scales))
        wants.append((F.dilation(x, w, "identity"), p.codes, p.scales))
    for channels in (16000, 2000):   # 160 and 50 KiB of the norm's backward pass
        x, gy, w = (torch.randn(s, dtype=torch.float64, device="cuda") for s in ((1, channels, 2, 2), (1, channels, 2, 2), (channels,)))
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        gx, gw = torch.empty_like(x), torch.empty_like(w)
        d = norm_desc(x, -3)
        need = lib.mc_rms_norm_backward_workspace_bytes(ctypes.byref(d), 1)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        calls.append(lambda d=d, t=(x, w, gy, gx, gw, ws), need=need: lib.mc_rms_norm_backward(
            ctypes.byref(d), ptr(t[0]), None, None, ptr(t[1]), ptr(t[2]), None, ptr(t[3]), ptr(t[4]), ptr(t[5]), ctypes.c_size_t(need), at))
        results.append((gx, gw))
        wants.append(lambda leaves=leaves, gy=gy: torch.autograd.grad(F.rms_norm(*leaves), leaves, gy))
    torch.cuda.synchronize()
    assert in_threads(*calls, times=3000) == []
    for got, want in zip(results, wants):
        for a, b in zip(got, want() if callable(want) else want):
            assert bool((a == b).all())


EVERY_BACKWARD_KERNEL = [((2, 20, 9, 15), -3), ((3, 20, 4, 8), -3), ((2, 50, 9, 15), -3), ((2, 100, 11, 12), -3), ((1, 200, 9, 15), -3), ((1, 500, 5, 8), -3), ((1, 600, 5, 9), -3),
                         ((35, 40), -1), ((33, 127), -1), ((19, 250), -1), ((21, 700), -1), ((3, 5000), -1), ((2, 9000), -1)]


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("eps", [1e-60, 1e-90, 1e-200])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,dim", EVERY_BACKWARD_KERNEL, ids=str)
def test_an_eps_that_leaves_pixels_of_zeros_a_factor_beyond_float(shape, dim, dtype, eps, keep8):
    """A pixel of zeros, masked or padded, has r = eps^-1/2: it gives nothing to gweight, its own gradient is r u, zero where u is, infinite
    where the type does not hold it. Tiles that hang over the image, and rows that do not fill a warp, have such places as well."""
    _, _, w, s = tensors(shape, dim, dtype, False)
    gy = make(shape, dtype, 4)
    pixels, upstream = (t.transpose(dim, -1).reshape(-1, shape[dim]).clone() for t in (s, gy))
    pixels[::3] = 0
    upstream[::6] = 0
    pixels[1::5] *= 2.0 ** -12 if dtype == torch.float16 else 2.0 ** -70
    wide = list(shape)
    wide[dim], wide[-1] = wide[-1], wide[dim]
    s, gy = (t.reshape(wide).transpose(dim, -1).contiguous() for t in (pixels, upstream))
    leaves = [t.requires_grad_(True) for t in cuda(s, w)]
    y = F.checkpoint_8bit(F.rms_norm, *leaves, None, eps, dim) if keep8 else F.rms_norm(*leaves, None, eps, dim)
    got = torch.autograd.grad(y, leaves, gy.cuda())
    at = s
    if keep8:
        kept = F.encode_8bit(s.cuda(), row_dims_of(s, dim))
        at = P.decode(kept.codes.cpu(), kept.scales.cpu(), dtype)
    want, want_w, size, size_w = P.rms_norm_backward(at, w, gy, None, eps, dim)
    assert bool(want_w.isfinite().all())
    more = 0 if dtype == torch.float64 else 2.5 * -(-shape[dim] // 16) * 2.0 ** -24   # as in check_gradients
    bound = grad_bound(size, want, dtype, shape[dim]) + more * size
    beyond = want.abs() > torch.finfo(dtype).max   # rounds to the largest value or to infinity
    gx = got[0].cpu().double()
    assert not bool(gx.isnan().any())
    assert bool(((gx - want).abs() <= bound)[~beyond].all()) and bool((gx[beyond].abs() >= torch.finfo(dtype).max).all())
    assert bool((gx[beyond].sign() == want[beyond].sign()).all())
    within(got[1], want_w, weight_bound(size_w, want_w, dtype, channels=shape[dim]) + more * size_w, "weight")


def test_the_smallest_eps_in_double():
    """r^2 leaves double's range for an eps below 2^-1024; the gradient r u of a pixel of zeros does not."""
    for shape, dim in (((2, 5, 3, 7), -3), ((7, 40), -1), ((1, 200, 3, 3), -3)):
        x = torch.zeros(shape, dtype=torch.float64, device="cuda", requires_grad=True)
        w, g = torch.ones(shape[dim], dtype=torch.float64, device="cuda", requires_grad=True), make(shape, torch.float64, 4).cuda()
        gx, gw = torch.autograd.grad(F.rms_norm(x, w, eps=1e-312, dim=dim), (x, w), g)
        want = g.cpu() / 1e-312 ** 0.5
        assert bool((gw == 0).all()) and bool(((gx.cpu() - want).abs() <= 8 * 2.0 ** -53 * want.abs()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape,dim", [*EVERY_BACKWARD_KERNEL, ((40, 128), -1), ((9, 256), -1), ((4, 512), -1), ((2, 4096), -1), ((2, 16384), -1), ((2, 128, 6, 6), -3)], ids=str)
def test_float_weights_beside_half_precision(shape, dim, dtype):
    """The weight enters unrounded, and its gradient is float32, forward and backward, from the sum and from its codes; also for a weight that
    does not start on the boundary of a wide load."""
    x, r, _, s = tensors(shape, dim, dtype, True, False)
    w = make((shape[dim],), torch.float32, 3, 0.2, 1.0)
    gy, gs = make(shape, dtype, 4), make(shape, dtype, 5)
    more = 2.5 * -(-shape[dim] // 16) * 2.0 ** -24   # as in check_gradients
    for offset in (0, 1):
        for keep8 in (False, True):
            leaves = [t.cuda().requires_grad_(True) for t in (x, torch.cat([torch.zeros(offset), w]), r)]
            args = (leaves[0], leaves[1][offset:], leaves[2], EPS, dim)
            with torch.no_grad():
                coded, _ = F.rms_norm(*args, output="8bit")
            y, total = F.checkpoint_8bit(F.rms_norm, *args) if keep8 else F.rms_norm(*args)
            assert y.dtype == dtype and bool((total.cpu() == s).all())
            want = P.rms_norm(s, w, EPS, dim)
            within(y, want, value_bound(want, dtype, shape[dim]))
            packed = F.encode_8bit(y.detach(), row_dims_of(x, dim))
            assert bool((packed.codes == coded.codes).all()) and bool((packed.scales == coded.scales).all())
            at = s
            if keep8:
                kept = F.encode_8bit(s.cuda(), row_dims_of(x, dim))
                at = P.decode(kept.codes.cpu(), kept.scales.cpu(), dtype)
            want, want_w, size, size_w = P.rms_norm_backward(at, w, gy, gs, EPS, dim)
            gx, gw, _ = torch.autograd.grad((y, total), leaves, (gy.cuda(), gs.cuda()))
            assert gx.dtype == dtype and gw.dtype == torch.float32
            within(gx, want, grad_bound(size, want, dtype) + more * size, "x")
            within(gw[offset:], want_w, weight_bound(size_w, want_w, torch.float32) + more * size_w, "weight")
            # A weight that half precision holds gives what it gives in half precision.
            short = w.to(dtype).cuda()
            assert bool((F.rms_norm(x.cuda(), short.float(), r.cuda(), EPS, dim)[0] == F.rms_norm(x.cuda(), short, r.cuda(), EPS, dim)[0]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_the_module_s_float_weight_beside_half_precision(dtype):
    """nn.RMSNorm as it is made, with maps in half precision and a small eps, without pixels, and what is still refused."""
    norm = Mnn.RMSNorm(6).cuda()
    torch.nn.init.normal_(norm.weight, mean=1.0, std=0.2)
    x, g = make((2, 6, 5, 8), dtype, 1).cuda(), make((2, 6, 5, 8), dtype, 2)
    F.checkpoint_8bit(norm, x).backward(g.cuda())
    assert norm.weight.grad.dtype == torch.float32 and bool(norm.weight.grad.isfinite().all())
    empty = torch.zeros(0, 6, 5, 8, dtype=dtype, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(norm(empty).sum(), (empty, norm.weight))
    assert gx.shape == empty.shape and gw.dtype == torch.float32 and bool((gw == 0).all())
    zeros = torch.zeros(2, 6, 5, 8, dtype=dtype, device="cuda", requires_grad=True)
    gw, = torch.autograd.grad(F.rms_norm(zeros, norm.weight, eps=1e-90), norm.weight, g.cuda())
    assert bool((gw == 0).all())
    for bad, weight in ((x, norm.weight.double()), (x.float(), norm.weight.to(dtype)), (x.double(), norm.weight),
                        (x, norm.weight.to(torch.float16 if dtype == torch.bfloat16 else torch.bfloat16))):
        with pytest.raises(RuntimeError, match="weight must have the type of x"):
            F.rms_norm(bad, weight)
