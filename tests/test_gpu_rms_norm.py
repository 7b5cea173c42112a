"""The root-mean-square norm on the GPU, its gradients and its 8-bit forms, against the plain implementation in 64 bits."""
import pytest
import torch

import _plain8 as P
import morphocore_b200.functional as F
import morphocore_b200.nn as Mnn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]
# Feature maps: channels below, at and above what a thread block holds in each of its variants; planes of one pixel, of a ragged
# block, of odd sizes. Rows: a channel, a ragged block, one warp, several warps, the longest.
MAPS = [((1, 1, 1, 2), -3), ((2, 3, 5, 7), -3), ((3, 20, 9, 12), -3), ((2, 33, 12, 12), -3), ((2, 64, 7, 7), -3), ((1, 65, 16, 16), -3), ((2, 100, 11, 11), -3),
        ((1, 128, 16, 8), -3), ((1, 130, 4, 33), -3), ((1, 300, 6, 6), -3), ((1, 1030, 3, 4), -3), ((4, 16, 3, 40), -2), ((300, 5, 2), -2), ((7, 9, 130), 0)]
ROWS = [((1, 1), -1), ((3, 7), -1), ((5, 64), -1), ((2, 3, 128), -1), ((9, 130), -1), ((4, 512), -1), ((3, 1000), -1), ((2, 2049), -1), ((3, 4096), -1),
        ((2, 5000), -1), ((1, 16384), -1), ((33, 2, 3, 48), -1), ((5, 12, 1, 1), -3), ((9,), 0)]
EPS = 1e-6


def make(shape, dtype, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale + shift).to(dtype)


def row_dims_of(x, dim):
    after = 1
    for n in x.shape[dim % x.dim() + 1:]:
        after *= n
    return x.dim() - dim % x.dim() if after == 1 else x.dim() - 1 - dim % x.dim()


def value_bound(want, dtype, channels):
    """Half a step of the type around a value that 46 bits or more stand behind; in double the sums' own roundings, a half step for
    each square and each addition, half of it after the root, and those of the products."""
    if dtype == torch.float64:
        return want.abs() * (channels + 8) * 2.0 ** -53
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps   # a step of the numbers without a leading one
    return want.abs() * (torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -12) + tiny / 2


def rounding(want, dtype):
    """Half a step of the type, below its smallest normal number half the one step that there is, eps times that number."""
    info = torch.finfo(dtype)
    return (want.abs() * (1 + 2.0 ** -10)).clamp(min=info.smallest_normal) * (info.eps / 2)


def grad_bound(size, want, dtype, channels=0):
    """Gradients of the input: eight roundings in the type that the kernel computes in, each half a step of the terms, and one to
    the tensor's type; in double also those of the sums over the channels."""
    u = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps / 2
    return (8 + 2 * channels * (dtype == torch.float64)) * u * size + rounding(want, dtype)


def weight_bound(size, want, dtype, adds=32, channels=0):
    """Gradients of the weight: `adds` additions one after the other in the computing type (pixels of a thread, lanes, groups of a
    thread block), the rest in double, then a rounding to the tensor's type; in double also those of the sum behind r."""
    u = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps / 2
    return (adds + 4 + channels * (dtype == torch.float64)) * u * size + rounding(want, dtype)


def within(a, want, bound, what=""):
    off = (a.cpu().double() - want).abs()
    assert a.shape == want.shape, (what, a.shape, want.shape)
    assert bool((off <= bound).all()), (what, float(off.max()), float((off - bound).max()))


def tensors(shape, dim, dtype, residual=True, weight=True):
    x = make(shape, dtype, 1)
    r = make(shape, dtype, 2) if residual else None
    w = make((shape[dim],), dtype, 3, 0.2, 1.0) if weight else None
    s = x if r is None else ((x + r) if dtype == torch.float64 else (x.float() + r.float()).to(dtype))
    return x, r, w, s


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,dim", MAPS + ROWS, ids=str)
def test_forward_and_codes(shape, dim, dtype):
    for residual, weight in ((True, True), (False, True), (True, False)):
        x, r, w, s = tensors(shape, dim, dtype, residual, weight)
        want = P.rms_norm(s, w, EPS, dim)
        out = F.rms_norm(*cuda(x, w, r), eps=EPS, dim=dim, output="both")
        y, packed = out[:2]
        assert len(out) == (3 if residual else 2) and y.dtype == dtype
        within(y, want, value_bound(want, dtype, shape[dim]))
        if residual:
            assert bool((out[2].cpu() == s).all())
        # The codes are those of encode_8bit, to the bit, whatever is asked for beside them.
        again = F.encode_8bit(y, row_dims_of(x, dim))
        assert bool((packed.codes == again.codes).all()) and packed.scales.shape == again.scales.shape and bool((packed.scales == again.scales).all())
        alone = F.rms_norm(*cuda(x, w, r), eps=EPS, dim=dim, output="8bit")
        alone = alone[0] if residual else alone
        assert bool((alone.codes == packed.codes).all()) and bool((alone.scales == packed.scales).all())
        plain = F.rms_norm(*cuda(x, w, r), eps=EPS, dim=dim)
        assert bool(((plain[0] if residual else plain) == y).all())


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,dim", MAPS + ROWS, ids=str)
def test_gradients(shape, dim, dtype, keep8):
    for residual, weight in ((True, True), (False, True), (True, False)):
        x, r, w, s = tensors(shape, dim, dtype, residual, weight)
        gy, gs = make(shape, dtype, 4), make(shape, dtype, 5) if residual else None
        leaves = [None if t is None else t.requires_grad_(True) for t in cuda(x, w, r)]
        out = F.checkpoint_8bit(F.rms_norm, *leaves, EPS, dim) if keep8 else F.rms_norm(*leaves, EPS, dim)
        at = s
        if keep8:
            kept = F.encode_8bit(s.cuda(), row_dims_of(x, dim))
            at = P.decode(kept.codes.cpu(), kept.scales.cpu(), dtype)
        want, want_w, size, size_w = P.rms_norm_backward(at, w, gy, gs, EPS, dim)
        given = [t for t in leaves if t is not None]
        got = torch.autograd.grad(out, given, [gy.cuda(), gs.cuda()] if residual else gy.cuda())
        within(got[0], want, grad_bound(size, want, dtype, shape[dim]), "x")
        if residual:
            assert bool((got[-1] == got[0]).all())
        if weight:
            within(got[1], want_w, weight_bound(size_w, want_w, dtype, channels=shape[dim]), "weight")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,channels", [(1, 3), (2, 64), (34, 20), (67, 127), (3, 128), (1, 129), (18, 200), (33, 256), (3, 257), (9, 600), (5, 1500), (3, 4095), (2, 8192),
                                           (2, 9001)], ids=str)
def test_rows_that_share_warps_and_warps_that_share_rows(rows, channels, dtype):
    test_forward_and_codes((rows, channels), -1, dtype)
    for keep8 in (False, True):
        test_gradients((rows, channels), -1, dtype, keep8)


@pytest.mark.parametrize("dtype", TYPES[:3], ids=str)
@pytest.mark.parametrize("shape,dim", [((3, 20, 31, 33), -3), ((2, 64, 40, 40), -3), ((2, 61, 25, 41), -3), ((2, 128, 28, 28), -3), ((1, 300, 24, 24), -3), ((700, 64), -1), ((300, 250), -1),
                                       ((64, 1024), -1), ((9, 5001), -1), ((3, 16384), -1)], ids=str)
def test_results_are_rounded_once(shape, dim, dtype):
    """A result is within half a step of its own binade of the value in 64 bits: what it is rounded from is off by less than 2^-40 of
    it (46 bits of r and of the products, a sum in double), which is 2^-15 of half a step in float and less in the other types. Half
    precision is rounded from the float that is nearest, off by at most 2^-24 of the value, which is less than 2^-23 of its binade, more."""
    x, r, w, s = tensors(shape, dim, dtype)
    want = P.rms_norm(s, w, EPS, dim)
    got = F.rms_norm(*cuda(x, w, r), eps=EPS, dim=dim)[0].cpu().double()
    through_float = 0.0 if dtype == torch.float32 else 2.0 ** -23
    binade = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=torch.finfo(dtype).smallest_normal))))
    assert bool(((got - want).abs() <= binade * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -14) + through_float)).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,dim", [((35, 40), -1), ((35, 128), -1), ((19, 250), -1), ((5, 700), -1), ((21, 700), -1), ((2, 9, 13, 12), -3), ((2, 70, 13, 11), -3), ((1, 600, 6, 6), -3)], ids=str)
def test_nothing_of_a_neighbour(shape, dim, dtype):
    """Rows, and pixels, that leave the range of float, hold infinities or NaN, change not one bit of the others."""
    info = torch.finfo(dtype)
    results = []
    for special in (False, True):
        s = make(shape, dtype, 6)
        pixels = s.transpose(dim, -1).reshape(-1, s.shape[dim]).clone()
        others = torch.ones(len(pixels), dtype=torch.bool)
        for i, value in enumerate((info.max, float("inf"), info.smallest_normal, float("nan"), 0.0)):
            others[2 * i % len(pixels)::10] = False
            if special:
                pixels[2 * i % len(pixels)::10] = value
        wide = list(s.shape)
        wide[dim], wide[-1] = wide[-1], wide[dim]
        x = pixels.reshape(wide).transpose(dim, -1).contiguous().cuda().requires_grad_(True)
        w = make((shape[dim],), dtype, 3, 0.2, 1.0).cuda()
        y = F.rms_norm(x, w, eps=1e-30, dim=dim)
        gx, = torch.autograd.grad(y, x, make(shape, dtype, 4).cuda())
        results.append([t.detach().cpu().transpose(dim, -1).reshape(-1, s.shape[dim])[others] for t in (y, gx)])
    for usual, beside in zip(*results):
        assert bool((usual == beside).all())


@pytest.mark.parametrize("shape,dim", [((40, 24, 60, 60), -3), ((24, 65, 64, 64), -3), ((6, 200, 72, 72), -3), ((60000, 48), -1), ((9000, 520), -1), ((700, 4100), -1)], ids=str)
@pytest.mark.parametrize("keep8", [False, True])
def test_more_tiles_than_thread_blocks(shape, dim, keep8):
    """Thread blocks of the backward pass that walk over several tiles; the same twice to the bit."""
    x, r, w, s = tensors(shape, dim, torch.float32)
    gy, gs = make(shape, torch.float32, 4), make(shape, torch.float32, 5)
    leaves = [t.requires_grad_(True) for t in cuda(x, w, r)]
    grads = []
    for _ in range(2):
        out = F.checkpoint_8bit(F.rms_norm, *leaves, EPS, dim) if keep8 else F.rms_norm(*leaves, EPS, dim)
        grads.append(torch.autograd.grad(out, leaves, [gy.cuda(), gs.cuda()]))
    assert all(bool((a == b).all()) for a, b in zip(*grads))
    at = s
    if keep8:
        kept = F.encode_8bit(s.cuda(), row_dims_of(x, dim))
        at = P.decode(kept.codes.cpu(), kept.scales.cpu(), torch.float32)
    want, want_w, size, size_w = P.rms_norm_backward(at, w, gy, gs, EPS, dim)
    within(out[0], P.rms_norm(s, w, EPS, dim), value_bound(P.rms_norm(s, w, EPS, dim), torch.float32, shape[dim]))
    within(grads[0][0], want, grad_bound(size, want, torch.float32))
    # At most a few hundred elements of a channel go through one lane.
    within(grads[0][1], want_w, weight_bound(size_w, want_w, torch.float32, adds=400))


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("shape,dim", [((2, 3, 4, 5), -3), ((3, 6), -1)], ids=str)
def test_gradients_against_differences(shape, dim, keep8):
    x, r, w, _ = tensors(shape, dim, torch.float64)
    if keep8:
        x = x.cuda()
        for _ in range(2):
            x = F.decode_8bit(F.encode_8bit(x, row_dims_of(x, dim)))
        leaves = [t.requires_grad_(True) for t in (x, w.cuda())]
        assert torch.autograd.gradcheck(lambda a, b: F.checkpoint_8bit(F.rms_norm, a, b, None, EPS, dim), leaves)
    else:
        leaves = [t.requires_grad_(True) for t in cuda(x, w, r)]
        assert torch.autograd.gradcheck(lambda a, b, c: F.rms_norm(a, b, c, EPS, dim), leaves)
        assert torch.autograd.gradcheck(lambda a: F.rms_norm(a, dim=dim), leaves[:1])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,dim", [((2, 24, 5, 28), -3), ((2, 24, 5, 7), -3), ((12, 260), -1)], ids=str)
def test_extremes(shape, dim, dtype):
    """Zeros, the type's smallest and largest values, infinities and NaN: what 64-bit arithmetic gives, and nothing of it in other
    pixels."""
    s = make(shape, dtype, 6)
    pixels = s.transpose(dim, -1).reshape(-1, s.shape[dim]).clone()
    info = torch.finfo(dtype)
    pixels[0] = 0
    pixels[1] = info.smallest_normal
    pixels[2] = info.max
    pixels[3, ::2], pixels[3, 1::2] = info.max, info.min
    pixels[4, 3] = float("inf")
    pixels[5, 4] = float("nan")
    pixels[6, 0], pixels[6, 1] = float("inf"), -float("inf")
    pixels[7] *= 2.0 ** 15 if dtype == torch.float16 else 2.0 ** 100
    pixels[8] *= 2.0 ** -14 if dtype == torch.float16 else 2.0 ** -100
    s = pixels.reshape(s.transpose(dim, -1).shape).transpose(dim, -1).contiguous()
    w = make((shape[dim],), dtype, 3, 0.2, 1.0)
    for eps in (1e-6, 1e-30):
        want = P.rms_norm(s, w, eps, dim)
        y = F.rms_norm(s.cuda(), w.cuda(), eps=eps, dim=dim).cpu().double()
        if dtype == torch.float64:   # squares of its largest and smallest values leave its range, here and there
            keep = torch.isfinite(s * s) & ((s * s >= info.smallest_normal) | (s == 0))
            keep = keep.all(dim, keepdim=True).expand_as(s)
            y, want = y[keep], want[keep]
        assert bool((y.isnan() == want.isnan()).all())
        ok = want.isfinite()
        bound = value_bound(want, dtype, shape[dim])
        beyond = want.abs() > info.max   # rounds to the largest value or to infinity
        assert bool(((y - want).abs()[ok & ~beyond] <= bound[ok & ~beyond]).all()) and bool((y[beyond].abs() >= info.max).all())
    big = make((shape[dim],), dtype, 3)
    big[0], big[1], big[2] = info.max, float("inf"), float("nan")
    x = make(shape, dtype, 7)
    y = F.rms_norm(x.cuda(), big.cuda(), dim=dim).cpu()
    want = P.rms_norm(x, big, EPS, dim).to(dtype)
    assert bool((y.isnan() == want.isnan()).all()) and bool((y.isinf() == want.isinf()).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts_and_alignment(dtype):
    n = 2 * 6 * 4 * 8
    flat = [make((n + 8,), dtype, seed).cuda() for seed in (1, 2, 3)]
    base = None
    for offset in (0, 1, 3, 4):
        for who in range(3):   # one tensor off the boundary, the others on it
            x, r, gy = (t[:n].clone() if k != who else torch.cat([t.new_zeros(offset), t[:n]])[offset:] for k, t in enumerate(flat))
            x, r, gy = (t.view(2, 6, 4, 8) for t in (x, r, gy))
            y, total = F.rms_norm(x.requires_grad_(True), None, r)
            got = (y, total, torch.autograd.grad(y, x, gy)[0])
            base = got if base is None else base
            assert all(bool((a == b).all()) for a, b in zip(got, base))
    x, r, w, s = tensors((3, 8, 6, 10), 1, dtype)
    want = F.rms_norm(*cuda(x, w, r))
    for view in (lambda t: t.to(memory_format=torch.channels_last), lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
                 lambda t: torch.cat([t, t], 1)[:, :8], lambda t: torch.stack([t, t], -1)[..., 0]):
        got = F.rms_norm(view(x.cuda()), w.cuda(), view(r.cuda()))
        assert all(bool((a == b).all()) for a, b in zip(got, want))
    leaf = x.cuda().requires_grad_(True)
    a = torch.autograd.grad(F.rms_norm(leaf, w.cuda())[:, ::2].sum(), leaf)[0]   # a strided and broadcast gradient
    mask = torch.zeros_like(leaf)
    mask[:, ::2] = 1
    assert bool((a == torch.autograd.grad(F.rms_norm(leaf, w.cuda()), leaf, mask)[0]).all())
    wide = torch.stack([w, w], 1).cuda()[:, 0]
    assert bool((F.rms_norm(x.cuda(), wide) == F.rms_norm(x.cuda(), w.cuda())).all())


def test_parts_of_the_graph():
    """Outputs that are not used, inputs that need no gradient, a residual that is the input."""
    x, r, w, s = tensors((2, 5, 6, 7), 1, torch.float32)
    x, r, w = (t.requires_grad_(True) for t in cuda(x, r, w))
    g = torch.randn(2, 5, 6, 7, device="cuda")
    y, total = F.rms_norm(x, w, r)
    assert bool((torch.autograd.grad(total, (x, r), g, retain_graph=True)[0] == g).all())
    gx, gw = torch.autograd.grad(total, (x, w), g, retain_graph=True, allow_unused=True)
    assert bool((gx == g).all()) and (gw is None or bool((gw == 0).all()))
    both = torch.autograd.grad((y, total), x, (g, g), retain_graph=True)[0]
    alone = torch.autograd.grad(y, x, g)[0]
    assert bool((both - alone - g).abs().max() <= 1e-5)
    y, packed, total = F.rms_norm(x, w, r, output="both")
    assert not packed.codes.requires_grad and not packed.scales.requires_grad and total.requires_grad
    only = torch.autograd.grad(F.rms_norm(x.detach(), w), w, g)[0]
    assert bool((only == torch.autograd.grad(F.rms_norm(x, w), w, g)[0]).all())
    twice, _ = F.rms_norm(x, w, x)
    single = F.rms_norm(x + x, w)
    assert bool((torch.autograd.grad(twice, x, g)[0] - torch.autograd.grad(single, x, g)[0]).abs().max() <= 1e-6)
    x.grad = r.grad = w.grad = None
    y, total = F.rms_norm(x, w, r)
    (y.sum() + total.sum()).backward()
    first = x.grad.clone()
    r.grad.zero_()   # gradients of the two inputs are not one tensor
    assert bool((x.grad == first).all())


def test_empty_and_refusals():
    for shape, dim in (((0, 5, 3, 3), -3), ((2, 5, 0, 3), -3), ((0, 8), -1)):
        x, w = torch.zeros(shape, device="cuda", requires_grad=True), torch.ones(shape[dim], device="cuda", requires_grad=True)
        y, packed = F.rms_norm(x, w, dim=dim, output="both")
        assert y.shape == shape and packed.codes.shape == shape
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert gx.shape == shape and bool((gw == 0).all())
        assert F.decode_8bit(packed).shape == shape
    x = torch.randn(2, 5, 4, 4, device="cuda")
    for bad in (dict(weight=torch.ones(4, device="cuda")), dict(weight=torch.ones(5, 1, device="cuda")), dict(weight=torch.ones(5)),
                dict(weight=torch.ones(5, device="cuda").half()), dict(residual=x[:1]), dict(residual=x.double()), dict(residual=x.cpu()), dict(dim=4),
                dict(dim=-5), dict(eps=0.0), dict(eps=-1e-6), dict(eps=float("nan"))):
        with pytest.raises(RuntimeError):
            F.rms_norm(x, **bad)
    for bad in (x.int(), x.cpu(), torch.zeros(2, 0, 4, 4, device="cuda"), torch.zeros(16385, 2, 2, device="cuda"), x[0, 0]):
        with pytest.raises(RuntimeError):
            F.rms_norm(bad)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="has no gradient"):
        F.rms_norm(leaf, output="8bit")
    with torch.no_grad():
        F.rms_norm(leaf, output="8bit")
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(F.rms_norm(leaf).sum(), leaf, create_graph=True)
    kept = leaf * 1
    y = F.rms_norm(kept)
    kept.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_tangents_are_refused():
    """Forward-mode tangents and functorch transforms have no rule here: they raise instead of being dropped on the way."""
    import torch.autograd.forward_ad as fwad
    x, w = torch.randn(2, 4, 5, 6, device="cuda"), torch.ones(4, device="cuda")
    for call in (lambda t: F.rms_norm(t, w), lambda t: F.rms_norm(x, w, t)[0], lambda t: F.checkpoint_8bit(F.rms_norm, t, w),
                 lambda t: F.checkpoint_8bit(F.dilation, t, w.expand(3, 4)[:, :, None, None])):
        with pytest.raises(RuntimeError), fwad.dual_level():
            call(fwad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).sum())(x)


def test_streams_and_graphs():
    """Two replayed graphs and a side stream, forward and backward: each has workspaces of its own."""
    x, r, w, s = cuda(*tensors((4, 70, 20, 21), 1, torch.float32))
    gy = torch.randn_like(x)

    def step(x, r, w):
        a, b, c = (t.detach().requires_grad_(True) for t in (x, r, w))
        y, packed, total = F.checkpoint_8bit(F.rms_norm, a, c, b, output="both")
        return (y, packed.codes, packed.scales, total, *torch.autograd.grad((y, total), (a, c), (gy, gy)))

    want = [t.clone() for t in step(x, r, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, r, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(bool((a == b).all()) for a, b in zip(got, want))
    fixed = [torch.zeros_like(x) for _ in range(2)]
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, f in zip(graphs, fixed):
        with torch.cuda.graph(graph):
            held.append(step(f, r, w))
    fixed[0].copy_(x)
    fixed[1].copy_(-x)
    graphs[0].replay()
    graphs[1].replay()
    assert all(bool((a == b).all()) for a, b in zip(held[0], want))
    assert all(bool((a == b).all()) for a, b in zip(held[1], step(-x, r, w)))


def test_many_small_images_and_long_tensors():
    """More tiles than 2^16, and offsets beyond 2^31 elements: the last image is that of a tensor of its own."""
    x = make((70001, 3, 2, 2), torch.float32, 1).cuda()
    y = F.rms_norm(x)
    assert bool((y[-3:] == F.rms_norm(x[-3:])).all())
    C, H, W = 66, 255, 257
    N = 2 ** 31 // (C * H * W) + 2
    x = torch.ones(N, C, H, W, dtype=torch.bfloat16, device="cuda")
    x[-1] = make((C, H, W), torch.bfloat16, 2).cuda()
    w = make((C,), torch.bfloat16, 3, 0.2, 1.0).cuda()
    y, packed = F.rms_norm(x, w, output="both")
    last, last_packed = F.rms_norm(x[-1:], w, output="both")
    assert bool((y[-1:] == last).all()) and bool((packed.codes[-1:] == last_packed.codes).all()) and bool((packed.scales[-1:] == last_packed.scales).all())
    del y, packed
    leaf = x.requires_grad_(True)
    gy = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(x.shape)
    gx, = torch.autograd.grad(F.checkpoint_8bit(F.rms_norm, leaf, w), leaf, gy)
    tail = leaf[-1:].detach().requires_grad_(True)
    assert bool((gx[-1:] == torch.autograd.grad(F.checkpoint_8bit(F.rms_norm, tail, w), tail, gy[-1:])[0]).all())


def test_residual_block():
    """Norm, smooth layer and the next norm as a residual block, everything that is kept in 8 bits: the module's way and the explicit
    one with the norm's own codes give the same gradients, and those of the plain layers at the kept values."""
    torch.manual_seed(0)
    norm, layer = Mnn.RMSNorm(6).cuda(), Mnn.SMorph(6, 6, 3, "mean", init_alpha=1.0).cuda()
    torch.nn.init.normal_(layer.weight, std=0.1)
    torch.nn.init.normal_(norm.weight, mean=1.0, std=0.2)
    parameters = [*norm.parameters(), *layer.parameters()]
    x, r = (make((2, 6, 15, 18), torch.float32, seed).cuda().requires_grad_(True) for seed in (1, 2))
    g, gs = (torch.randn(2, 6, 15, 18, device="cuda") for _ in range(2))

    def one():
        y, total = F.checkpoint_8bit(norm, x, r)
        z = F.checkpoint_8bit(layer, y)
        return z, total

    def two():
        y, packed, total = F.checkpoint_8bit(F.rms_norm, x, norm.weight, r, output="both")
        return F.checkpoint_8bit(layer, y, packed=packed), total

    def at_the_codes():
        with torch.no_grad():
            y, total = norm(x, r)
        kept_total, kept_y = (F.decode_8bit(F.encode_8bit(t)) for t in (total, y))
        a, b = kept_total.requires_grad_(True), kept_y.requires_grad_(True)
        gy, *rest = torch.autograd.grad(layer(b), (b, *layer.parameters()), g)
        gx, gw = torch.autograd.grad(norm(a), (a, norm.weight), gy)
        return (gx + gs, gx + gs, gw, *rest)

    grads = [torch.autograd.grad(f(), (x, r, *parameters), (g, gs)) for f in (one, two)] + [at_the_codes()]
    outs = [f() for f in (one, two)]
    assert bool((outs[0][0] == outs[1][0]).all()) and bool((outs[0][1] == outs[1][1]).all())
    for a, b, c in zip(*grads):
        # Smorph's sums of gradients are atomic: the order of a few hundred additions in float.
        bound = 1e-4 * max(1.0, float(c.abs().max()))
        assert bool(((a - b).abs() <= bound).all()) and bool(((a - c).abs() <= bound).all())
