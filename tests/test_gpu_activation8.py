"""8-bit activations on the GPU, and the layers that keep their input in them, against plain implementations in 64 bits."""
import numpy as np
import pytest
import torch

import _plain8 as P
import morphocore_b200.functional as F
import morphocore_b200.nn as Mnn
from oracle import oracle as O

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]
SHAPES = [((1,), 1), ((3, 2), 1), ((2, 3, 1, 1), 2), ((5, 127), 1), ((2, 128), 1), ((3, 129), 1), ((1, 260), 1), ((7, 8192), 1), ((2, 3, 7, 7), 2),
          ((3, 5, 12, 20), 2), ((2, 2, 75, 101), 2), ((2, 3, 4, 5), 4), ((700, 3), 1), ((0, 4), 1), ((2, 0, 4, 4), 2), ((2, 3, 0, 4), 2)]


def make(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * 3).to(dtype)


def same(a, b):
    """Equal, NaN included."""
    return a.shape == b.shape and bool(((a == b) | ((a != a) & (b != b))).all())


def check(x, row_dims, device_x=None):
    """Codes and scales bit for bit, and the decoded values: a code is a whole number, so there is nothing to tolerate but in
    double, where the plain product is rounded to 64 bits of mantissa before it is rounded to a whole number."""
    packed = F.encode_8bit(x.cuda() if device_x is None else device_x, row_dims)
    codes, scales, _ = P.encode(x, row_dims)
    assert packed.dtype == x.dtype and packed.codes.dtype == torch.int8
    assert packed.scales.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    assert np.array_equal(packed.scales.cpu().numpy(), scales)
    assert np.array_equal(packed.codes.cpu().numpy(), codes)
    values = F.decode_8bit(packed)
    assert values.dtype == x.dtype
    assert same(values.cpu(), P.decode(torch.from_numpy(codes), torch.from_numpy(scales), x.dtype))
    return packed, values


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,row_dims", SHAPES, ids=str)
def test_codes(shape, row_dims, dtype):
    x = make(shape, dtype)
    packed, values = check(x, row_dims)
    if not x.numel():
        return
    # Half a scale, its own rounding and that of the product (three half steps of values up to 126 scales), and the type's.
    rows, length, _ = P.rows_of(shape, row_dims)
    u = torch.finfo(packed.scales.dtype).eps / 2
    scale = packed.scales.cpu().double().reshape(rows, -1).repeat_interleave(P.BLOCK, 1)[:, :length].reshape(shape)
    bound = scale * (0.5 + 3 * 126 * u) + values.cpu().double().abs() * torch.finfo(dtype).eps / 2
    assert bool(((values.cpu().double() - x.double()).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("length", [128, 131, 300])
def test_values_without_a_number(dtype, length):
    """Infinities and NaN come back as they are and leave the rest of their block alone; blocks of nothing else, of zeros, of the type's
    lowest value, of its largest, and of magnitudes too small for a scale."""
    x = make((12, length), dtype, 1)
    inf, nan, info = float("inf"), float("nan"), torch.finfo(dtype)
    x[0, 3], x[0, 64], x[0, 100] = inf, -inf, nan
    x[1, ::2] = -inf
    x[2] = nan
    x[3] = -inf
    x[4] = 0
    x[5] = info.min
    x[6, 5], x[6, 6] = info.max, info.min
    x[7] *= 2.0 ** -100 if dtype != torch.float64 else 2.0 ** -900
    x[8] = info.tiny
    x[9] = info.smallest_normal * 0.25
    x[10, :127] = 0
    x[11] = -0.0
    packed, values = check(x, 1)
    plain = x.double()
    assert bool((values.isnan().cpu() == x.isnan()).all()) and bool((values.isinf().cpu() == x.isinf()).all())
    assert bool((values[4] == 0).all()) and bool((values[11] == 0).all())
    if dtype in (torch.float32, torch.float64):
        assert not packed.scales[8].any() and not packed.scales[9].any()
    # The finite ones beside the infinities: half a scale, top / 252, with the roundings of 126 / m, of the scale and of its product
    # with a code (three half steps of top at most), and half a step of the tensor's type, of top or less.
    top = float(plain[1, 1::2].abs().max())
    u = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps / 2
    off = (values[1, 1::2].cpu().double() - plain[1, 1::2]).abs().max()
    assert bool((values[1, ::2] == -inf).all()) and float(off) <= top * (1 / 252 + 3 * u + info.eps / 2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts_and_alignment(dtype):
    """Views that start off the boundary of a wide load, strided, broadcast and permuted tensors, and a sliced 8-bit form."""
    flat = make((4 * 6 * 128 + 7,), dtype, 2)
    for offset in (0, 1, 2, 3, 4):
        x = flat[offset:offset + 4 * 6 * 128].view(4, 6, 128)
        check(x, 1, flat.cuda()[offset:offset + 4 * 6 * 128].view(4, 6, 128))
    x = make((3, 4, 6, 10), dtype, 3)
    for view in (lambda t: t.permute(0, 2, 3, 1), lambda t: t[:, ::2, 1:, ::3], lambda t: t[:1].expand(5, 4, 6, 10), lambda t: t.transpose(0, 3),
                 lambda t: t.to(memory_format=torch.channels_last)):
        check(view(x).contiguous(), 2, view(x.cuda()))
    packed, values = check(x, 2)
    assert same(F.decode_8bit(F.Activation8(packed.codes[1:], packed.scales[1:], dtype)), values[1:])
    assert same(F.decode_8bit(F.Activation8(packed.codes[:, ::2], packed.scales[:, ::2], dtype)), values[:, ::2])


def test_long_tensors():
    """More than 2^31 elements: the last rows are those of a tensor of their own."""
    length, rows = 128 * 1024 + 64, 16500
    assert length * rows > 2 ** 31
    x = torch.empty(rows, length, dtype=torch.bfloat16, device="cuda")
    x[:-2] = 1.0
    x[-2:] = make((2, length), torch.bfloat16, 4).cuda()
    packed = F.encode_8bit(x, 1)
    tail = F.encode_8bit(x[-2:], 1)
    assert bool((packed.codes[-2:] == tail.codes).all()) and bool((packed.scales[-2:] == tail.scales).all())
    assert bool((packed.codes[:-2:611] == 126).all())
    values = F.decode_8bit(packed)
    assert bool((values[-2:] == F.decode_8bit(tail)).all()) and bool((values[::997][:-1] == 1).all())


def test_streams_and_graphs():
    x = make((6, 10, 33, 35), torch.float32, 5).cuda()
    want = F.encode_8bit(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.encode_8bit(x)
        values = F.decode_8bit(got)
    torch.cuda.current_stream().wait_stream(side)
    assert bool((got.codes == want.codes).all()) and bool((got.scales == want.scales).all()) and bool((values == F.decode_8bit(want)).all())
    graph = torch.cuda.CUDAGraph()
    fixed = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        held = F.encode_8bit(fixed)
        values = F.decode_8bit(held)
    for seed in (6, 7):
        fixed.copy_(make(x.shape, x.dtype, seed))
        graph.replay()
        assert bool((held.codes == F.encode_8bit(fixed).codes).all()) and bool((values == F.decode_8bit(F.encode_8bit(fixed))).all())


def test_refusals():
    x = make((2, 3, 4, 5), torch.float32).cuda()
    packed = F.encode_8bit(x)
    for bad in (lambda: F.encode_8bit(x, 0), lambda: F.encode_8bit(x, -1), lambda: F.encode_8bit(x.int()), lambda: F.encode_8bit(x[0, 0, 0, 0]),
                lambda: F.decode_8bit(F.Activation8(packed.codes, packed.scales, torch.float64)),
                lambda: F.decode_8bit(F.Activation8(packed.codes.int(), packed.scales, x.dtype)),
                lambda: F.decode_8bit(F.Activation8(packed.codes, packed.scales.half(), x.dtype)),
                lambda: F.decode_8bit(F.Activation8(packed.codes, packed.scales[:1], x.dtype)),
                lambda: F.decode_8bit(F.Activation8(packed.codes, packed.scales[..., None], x.dtype)),
                lambda: F.decode_8bit(F.Activation8(packed.codes, packed.scales.cpu(), x.dtype)),
                lambda: F.decode_8bit(F.Activation8(packed.codes, packed.scales[0, 0, 0], x.dtype))):
        with pytest.raises(RuntimeError):
            bad()
    assert F.encode_8bit(x[0, 0, 0]).scales.shape == (1,)   # fewer dimensions than a row would have


# ---- layers that keep their input in 8 bits -------------------------------------------------------------------------------

LAYERS = [(op, merge) for op in ("dilation", "erosion", "smorph") for merge in ("sum", "mean", "max", "min", "identity")] + [("smorph_scm", "sum")]


def layer_tensors(op, merge, dtype, shape=(2, 3, 13, 18), Co=4, k=3, seed=0):
    C = shape[1]
    Co, Ci = (C, 1) if merge == "identity" else (Co, C)
    x, w = make(shape, dtype, seed), (make((Co, Ci, k, k), torch.float64, seed + 1) * 0.1).to(dtype)
    more = []
    if op.startswith("smorph"):
        more.append((1 + 0.1 * make((Co, Ci), torch.float64, seed + 2)).to(dtype))
    if op == "smorph_scm":
        more.append((0.5 + 0.1 * make((Co,), torch.float64, seed + 3)).to(dtype))
    return x, w, *more, make((shape[0], Co, *shape[2:]), dtype, seed + 4)


def call(op, merge, x, w, *more, save_indices=False):
    if op == "smorph":
        return F.smorph, (x, w, *more), dict(channel_merge_mode=merge)
    if op == "smorph_scm":
        return F.smorph, (x, w, *more), {}
    return getattr(F, op), (x, w, merge), dict(save_indices=save_indices)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("op,merge", LAYERS)
def test_layer_gradients_are_those_at_the_codes(op, merge, dtype):
    """Output: bit for bit the plain call's. Gradients: those of the plain layer, in double, at the values that the codes stand
    for. Dilation and erosion add a handful of gradients a pixel, and some hundred a weight, in float: 1e-4 of the largest is the
    bound that the layers' own tests use; smorph's likewise. Half precision widens to float and rounds the results once."""
    *tensors, gz = layer_tensors(op, merge, dtype)
    leaves = [t.cuda().requires_grad_(True) for t in tensors]
    function, args, kwargs = call(op, merge, *leaves)
    with torch.no_grad():
        plain = function(*args, **kwargs)
    z = F.checkpoint_8bit(function, *args, **kwargs)
    assert z.dtype == dtype and bool((z == plain).all())
    got = torch.autograd.grad(z, leaves, gz.cuda())

    # The layer computes in float for half precision, and so does it decode.
    kept = F.encode_8bit(leaves[0].detach())
    work = torch.float64 if dtype == torch.float64 else torch.float32
    values = P.decode(kept.codes.cpu(), kept.scales.cpu(), work)
    if op in ("dilation", "erosion"):
        # The winners are those among values as the kernels' type holds them: the oracle in that type, sums of gradients in it.
        wk = tensors[1].to(work).numpy()
        wk = wk if op == "dilation" else np.ascontiguousarray(wk[..., ::-1, ::-1])
        gx, gw = O.morpho_backward(op, values.numpy(), wk, gz.to(work).numpy(), merge)
        want = [torch.from_numpy(gx), torch.from_numpy(np.ascontiguousarray(gw[..., ::-1, ::-1]) if op == "erosion" else gw)]
    else:
        at = [values.double().cuda().requires_grad_(True)] + [t.double().cuda().requires_grad_(True) for t in tensors[1:]]
        function, args, kwargs = call(op, merge, *at)
        want = torch.autograd.grad(function(*args, **kwargs), at, gz.double().cuda())
    tol = 1e-11 if dtype == torch.float64 else 1e-4
    step = 0.0 if dtype in (torch.float32, torch.float64) else torch.finfo(dtype).eps / 2
    for a, b in zip(got, want):
        b = b.cpu().double()
        assert a.dtype == dtype and a.shape == b.shape
        bound = tol * max(1.0, float(b.abs().max())) + step * b.abs()
        assert bool(((a.cpu().double() - b).abs() <= bound).all()), float((a.cpu().double() - b).abs().max())


@pytest.mark.parametrize("op", ["dilation", "erosion"])
@pytest.mark.parametrize("merge", ["max", "min"])
def test_saved_winners_keep_exact_gradients(op, merge):
    *tensors, gz = layer_tensors(op, merge, torch.float64)
    leaves = [t.cuda().requires_grad_(True) for t in tensors]
    function, args, kwargs = call(op, merge, *leaves, save_indices=True)
    want = torch.autograd.grad(function(*args, **kwargs), leaves, gz.cuda())
    z = F.checkpoint_8bit(function, *args, **kwargs)
    kept = [t for t in z.grad_fn.saved_tensors] if hasattr(z.grad_fn, "saved_tensors") else []
    assert all(t is None or t.dtype != torch.int8 for t in kept)
    for a, b in zip(torch.autograd.grad(z, leaves, gz.cuda()), want):
        assert bool(((a - b).abs() <= 1e-12 * (1 + b.abs())).all())   # atomic sums of a few terms, in double


@pytest.mark.parametrize("op,merge", [("dilation", "sum"), ("erosion", "identity"), ("dilation", "max"), ("smorph", "mean"), ("smorph", "identity"),
                                      ("smorph_scm", "sum"), ("sigma_layer", "sum")])
def test_gradients_against_differences(op, merge):
    """At an input that its codes give back, the gradients are those of the layer itself, so that differences show them."""
    *tensors, gz = layer_tensors("smorph" if op == "sigma_layer" else op, merge, torch.float64, (1, 2, 5, 6), 3)
    x = tensors[0].cuda()
    for _ in range(2):
        x = F.decode_8bit(F.encode_8bit(x))
    # Distinct sums x + w: a tie has no gradient to compare with.
    leaves = [x.requires_grad_(True)] + [t.cuda().requires_grad_(True) for t in tensors[1:]]

    def layer(*t):
        if op == "sigma_layer":
            return F.checkpoint_8bit(F.sigma_layer, *t, merge, padding_mode="geodesic", save_indices=False)
        function, args, kwargs = call(op, merge, *t)
        if op in ("dilation", "erosion"):   # a border pixel that wins by way of the padding gets no gradient: none here
            kwargs["padding_mode"] = "geodesic"
        return F.checkpoint_8bit(function, *args, **kwargs)

    assert torch.autograd.gradcheck(layer, leaves, eps=1e-6, atol=1e-5, nondet_tol=1e-10)


@pytest.mark.parametrize("shape,k", [((1, 1, 1, 1), 3), ((3, 2, 1, 1), 3), ((2, 3, 1, 7), 5), ((1, 2, 40, 33), 11), ((5, 6, 7, 7), 3), ((2, 2, 9, 9), 2)])
def test_layer_sizes(shape, k):
    """Planes of one pixel (one scale an image), of odd sizes, smaller than the structuring element."""
    for op, merge in (("dilation", "sum"), ("smorph", "mean"), ("erosion", "identity")):
        *tensors, gz = layer_tensors(op, merge, torch.float64, shape, 3, k)
        leaves = [t.cuda().requires_grad_(True) for t in tensors]
        kept = F.decode_8bit(F.encode_8bit(leaves[0].detach(), 3 if shape[2:] == (1, 1) else 2))
        function, args, kwargs = call(op, merge, *leaves)
        got = torch.autograd.grad(F.checkpoint_8bit(function, *args, **kwargs), leaves, gz.cuda())
        at = [kept.requires_grad_(True)] + leaves[1:]
        function, args, kwargs = call(op, merge, *at)
        for a, b in zip(got, torch.autograd.grad(function(*args, **kwargs), at, gz.cuda())):
            assert bool(((a - b).abs() <= 1e-11 * max(1.0, float(b.abs().max()))).all())


def test_fewer_dimensions_and_empty_batches():
    w = make((3, 2, 3, 3), torch.float32, 1).cuda().requires_grad_(True)
    x = make((2, 6, 7), torch.float32).cuda().requires_grad_(True)
    gx, gw = torch.autograd.grad(F.checkpoint_8bit(F.dilation, x, w).sum(), (x, w))
    assert gx.shape == x.shape and gw.shape == w.shape
    kept = F.decode_8bit(F.encode_8bit(x.detach())).requires_grad_(True)
    assert bool((gx - torch.autograd.grad(F.dilation(kept, w).sum(), kept)[0]).abs().max() <= 1e-5)
    plane, square = make((6, 7), torch.float32).cuda().requires_grad_(True), make((3, 3), torch.float32).cuda().requires_grad_(True)
    gx, gw = torch.autograd.grad(F.checkpoint_8bit(F.erosion, plane, square, "identity").sum(), (plane, square))
    assert gx.shape == (6, 7) and gw.shape == (3, 3)
    empty = torch.zeros(0, 2, 6, 7, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(F.checkpoint_8bit(F.dilation, empty, w).sum(), (empty, w))
    assert gx.shape == empty.shape and bool((gw == 0).all())


@pytest.mark.parametrize("padding", ["zero", "geodesic", "constant", "replicate"])
def test_masked_inputs_and_padding(padding):
    """-inf in the input (what a geodesic border or a dropped weight leaves behind) stays out of the winners and out of its
    block's scale."""
    x = make((2, 3, 10, 17), torch.float32, 8)
    x[torch.rand(x.shape, generator=torch.Generator().manual_seed(9)) < 0.2] = -float("inf")
    w, gz = make((4, 3, 3, 3), torch.float32, 10) * 0.1, make((2, 4, 10, 17), torch.float32, 11)
    leaves = [x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)]
    z = F.checkpoint_8bit(F.dilation, *leaves, "sum", padding, padding_value=0.25)
    got = torch.autograd.grad(z, leaves, gz.cuda())
    kept = F.encode_8bit(x.cuda())
    values = P.decode(kept.codes.cpu(), kept.scales.cpu(), torch.float32)
    assert bool((values.isinf() == x.isinf()).all())
    gx, gw = O.morpho_backward("dilation", values.numpy(), w.numpy(), gz.numpy(), "sum", padding, 0.25)
    np.testing.assert_allclose(got[0].cpu().numpy(), gx, rtol=1e-4, atol=1e-4)
    np.testing.assert_allclose(got[1].cpu().numpy(), gw, rtol=1e-4, atol=1e-3)


def test_what_is_kept():
    """The graph holds codes and no float tensor of the input's size, the input may change before the backward pass, no_grad
    encodes nothing, and a module or a model is called like a function."""
    x = make((4, 8, 64, 64), torch.float32).cuda().requires_grad_(True)
    layer = Mnn.Dilation(8, 8, 3, "identity").cuda()
    torch.nn.init.normal_(layer.weight, std=0.1)

    def allocated_by(f):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        kept = f()
        return torch.cuda.memory_allocated() - before, kept

    hidden = (x * 1.0)
    size = hidden.nbytes
    plain, a = allocated_by(lambda: layer(x * 1.0))
    packed, b = allocated_by(lambda: F.checkpoint_8bit(layer, x * 1.0))
    assert plain >= 2 * size and packed <= size + size * 0.27
    g = torch.randn_like(a)
    want = torch.autograd.grad(layer(F.decode_8bit(F.encode_8bit(x.detach())).requires_grad_(True)), layer.weight, g)[0]
    hidden = x.detach().clone()
    z = F.checkpoint_8bit(layer, hidden)
    hidden.zero_()
    assert bool((torch.autograd.grad(z, layer.weight, g)[0] - want).abs().max() <= 1e-3)
    from morphocore_b200 import _native
    with torch.no_grad():
        layer(x)
        before = _native.launch_count()
        layer(x)
        one = _native.launch_count() - before
        F.checkpoint_8bit(layer, x)
        assert _native.launch_count() - before == 2 * one
    model = torch.nn.Sequential(Mnn.Opening(8, 8, 3), Mnn.SigmaLayer(8, 8, 3), Mnn.RMSNorm(8), Mnn.SMorph(8, 4, 3, init_alpha=1.0)).cuda()
    out = F.checkpoint_8bit(model, x)
    assert bool((out == model(x)).all())
    out.square().mean().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in model.parameters())


def test_packed_input_of_a_layer():
    x = make((2, 4, 9, 14), torch.float32, 3).cuda().requires_grad_(True)
    w = (make((4, 4, 3, 3), torch.float32, 4) * 0.1).cuda().requires_grad_(True)
    alpha = torch.full((4, 4), 1.5, device="cuda")
    other = F.encode_8bit(x.detach() * 2)   # not that of x: what is used shows
    g = torch.randn(2, 4, 9, 14, device="cuda")
    at = F.decode_8bit(other).requires_grad_(True)
    for function, more in ((F.dilation, ("sum",)), (F.smorph, (alpha,)), (F.sigma_layer, (alpha, "max")), (F.sigma_layer, (alpha, "sum", "replicate", False))):
        with torch.no_grad():
            plain = function(x, w, *more)
        z = F.checkpoint_8bit(function, x, w, *more, packed=other)
        assert bool((z == plain).all())
        got = torch.autograd.grad(z, (x, w), g)
        want = torch.autograd.grad(function(at if more[-1] != "max" else x, w, *more), (at if more[-1] != "max" else x, w), g)
        for a, b in zip(got, want):
            assert bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())
    # Codes of a token's layout decode by their own rows.
    rows = F.encode_8bit(x.detach(), 3)
    assert rows.scales.shape == (2, 4)
    torch.autograd.grad(F.checkpoint_8bit(F.dilation, x, w, packed=rows), (x, w), g)
    half = F.encode_8bit(x.detach().half())
    for bad in (F.encode_8bit(x.detach()[:1]), F.encode_8bit(x.detach().double()), F.Activation8(other.codes, other.scales[:, :2], x.dtype),
                F.Activation8(other.codes.cpu(), other.scales, x.dtype)):
        with pytest.raises(RuntimeError):
            F.checkpoint_8bit(F.dilation, x, w, packed=bad)
    xh, wh = x.detach().half().requires_grad_(True), w.detach().half().requires_grad_(True)
    assert torch.autograd.grad(F.checkpoint_8bit(F.dilation, xh, wh, packed=half), xh, g.half())[0].dtype == torch.float16


def test_noise_and_dropout_in_8_bits():
    """What is drawn in the call is drawn as in the plain call, and the gradients are those of that draw at the codes."""
    x = make((3, 4, 9, 11), torch.float32, 3).cuda().requires_grad_(True)
    w = (make((4, 4, 3, 3), torch.float32, 4) * 0.1).cuda().requires_grad_(True)
    g = make((3, 4, 9, 11), torch.float32, 5).cuda()
    for function in (F.dilation, F.erosion):
        for kwargs in (dict(noise_scale=0.2), dict(weight_dropout=0.3)):
            def drawn(call, x):
                torch.manual_seed(11)
                return call(x, w, training=True, **kwargs)

            z = drawn(lambda *t, **k: F.checkpoint_8bit(function, *t, **k), x)
            assert bool((z == drawn(function, x)).all())
            kept = F.decode_8bit(F.encode_8bit(x.detach())).requires_grad_(True)
            # The same kernels on the same numbers, atomic sums in float.
            for a, b in zip(torch.autograd.grad(z, (x, w), g), torch.autograd.grad(drawn(function, kept), (kept, w), g)):
                assert bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())


def test_training_step_in_a_graph():
    """Forward and backward under checkpoint_8bit, captured and replayed on new data."""
    w = (make((4, 4, 3, 3), torch.float32, 4) * 0.1).cuda().requires_grad_(True)
    alpha = torch.full((4, 4), 1.5, device="cuda", requires_grad=True)
    fixed, g = torch.zeros(2, 4, 16, 20, device="cuda", requires_grad=True), torch.randn(2, 4, 16, 20, device="cuda")

    def step(x, w, alpha):
        return torch.autograd.grad(F.checkpoint_8bit(F.smorph, x, w, alpha), (x, w, alpha), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fixed, w, alpha)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(fixed, w, alpha)
    for seed in (1, 2):
        x = make(fixed.shape, torch.float32, seed).cuda()
        with torch.no_grad():
            fixed.copy_(x)
        graph.replay()
        got = [t.clone() for t in held]
        for a, b in zip(got, step(x.requires_grad_(True), w.detach().requires_grad_(True), alpha.detach().requires_grad_(True))):
            assert bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())


# ---- per-channel layers: the kernels that write and read the codes themselves ---------------------------------------------

PLANES = [(1, 1, 1, 4), (2, 3, 5, 8), (3, 2, 9, 28), (1, 2, 40, 32), (2, 2, 31, 36), (1, 3, 70, 64), (2, 1, 33, 100), (1, 2, 130, 112), (1, 2, 66, 128), (2, 1, 20, 132),
          (1, 2, 75, 244), (1, 1, 9, 1000), (70, 40, 12, 16), (1, 1, 300, 240)]


@pytest.mark.parametrize("k", [3, 5])
@pytest.mark.parametrize("shape", PLANES, ids=str)
@pytest.mark.parametrize("op", ["dilation", "erosion"])
def test_per_channel_layers(op, shape, k):
    """Strips, runs and column tiles of every kind: the output bit for bit, the input's gradient within the rounding of its sums, of at most
    k * k terms, the weight's of one sum a lane and row and then of a few in a fixed order."""
    C = shape[1]
    x, w, gz = make(shape, torch.float32, 1), make((C, 1, k, k), torch.float32, 2) * 0.1, make(shape, torch.float32, 3)
    for padding in ("replicate", "geodesic", "constant"):
        leaves = [x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)]
        args = dict(channel_merge_mode="identity", padding_mode=padding, padding_value=0.125)
        with torch.no_grad():
            plain = getattr(F, op)(*leaves, **args)
        z = F.checkpoint_8bit(getattr(F, op), *leaves, **args)
        assert bool((z == plain).all())
        got = torch.autograd.grad(z, leaves, gz.cuda())
        codes, scales, _ = P.encode(x, 2)
        kept = P.decode(torch.from_numpy(codes), torch.from_numpy(scales), torch.float32)
        wk = w.numpy() if op == "dilation" else np.ascontiguousarray(w.numpy()[..., ::-1, ::-1])
        gx32, gw32 = O.morpho_backward(op, kept.numpy(), wk, gz.numpy(), "identity", padding, 0.125)
        gw32 = gw32 if op == "dilation" else gw32[..., ::-1, ::-1]
        size, size_w = (np.abs(t) for t in O.morpho_backward(op, kept.numpy(), wk, np.abs(gz.numpy()), "identity", padding, 0.125))
        size_w = size_w if op == "dilation" else size_w[..., ::-1, ::-1]
        u = 2.0 ** -24
        assert np.all(np.abs(got[0].cpu().numpy() - gx32) <= 2 * k * k * u * size + 1e-30)
        # A lane adds up its four columns of up to 64 rows one after the other, then 32 lanes; the oracle, all pixels in float.
        pixels = shape[0] * shape[2] * shape[3]
        assert np.all(np.abs(got[1].cpu().numpy() - gw32) <= (256 + 6 + min(pixels, 20000)) * u * size_w + 1e-30)
        again = torch.autograd.grad(F.checkpoint_8bit(getattr(F, op), *leaves, **args), leaves, gz.cuda())
        assert all(bool((a == b).all()) for a, b in zip(got, again))


@pytest.mark.parametrize("op", ["dilation", "erosion"])
def test_per_channel_ties_and_masks(op):
    """Zero structuring elements (every quantised neighbourhood has ties), planes of one value, and pixels without a number."""
    for seed, shape in enumerate([(2, 3, 17, 40), (1, 2, 12, 260)]):
        x = make(shape, torch.float32, seed)
        inf = float("inf")
        r = torch.rand(shape, generator=torch.Generator().manual_seed(seed))
        x[:, 0] = torch.round(x[:, 0])
        x[:, 1][r[:, 1] < 0.3] = -inf
        x[:, 1][r[:, 1] > 0.8] = inf
        x[:, -1][r[:, -1] < 0.05] = float("nan")
        x[0, 0, 3:9] = 2.0
        x[0, 1, 2:8, 4:30] = -inf if op == "dilation" else inf
        w = torch.zeros(shape[1], 1, 3, 3)
        w[-1] = make((1, 3, 3), torch.float32, 5) * 0.1
        gz = make(shape, torch.float32, 7)
        leaves = [x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)]
        for padding in ("replicate", "geodesic", "zero"):
            with torch.no_grad():
                plain = getattr(F, op)(*leaves, "identity", padding)
            z = F.checkpoint_8bit(getattr(F, op), *leaves, "identity", padding)
            assert same(z, plain)
            got = torch.autograd.grad(z, leaves, gz.cuda())
            kept = F.decode_8bit(F.encode_8bit(x.cuda()))
            assert bool((kept.isinf() == leaves[0].isinf()).all()) and bool((kept.isnan() == leaves[0].isnan()).all())
            at = [kept.requires_grad_(True), leaves[1]]
            want = torch.autograd.grad(getattr(F, op)(*at, "identity", padding), at, gz.cuda())
            for a, b in zip(got, want):   # the plain layers' kernels, whose atomic sums of a few hundred terms are in float
                assert bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())


def test_per_channel_noise_uses_each_image_s_weights():
    x, w = make((3, 2, 11, 20), torch.float32, 1).cuda().requires_grad_(True), (make((2, 1, 5, 5), torch.float32, 2) * 0.1).cuda().requires_grad_(True)
    g = make((3, 2, 11, 20), torch.float32, 3).cuda()
    for function in (F.dilation, F.erosion):
        torch.manual_seed(5)
        z = F.checkpoint_8bit(function, x, w, "identity", noise_scale=0.5, training=True)
        torch.manual_seed(5)
        kept = F.decode_8bit(F.encode_8bit(x.detach())).requires_grad_(True)
        y = function(kept, w, "identity", noise_scale=0.5, training=True)
        for a, b in zip(torch.autograd.grad(z, (x, w), g), torch.autograd.grad(y, (kept, w), g)):
            assert bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())


def test_per_channel_layers_through_the_c_abi():
    """What the entry points refuse with nothing launched, and an empty batch."""
    import ctypes

    from _cabi import lib, make_desc, ptr, stream
    from morphocore_b200 import _native
    x, w = make((2, 3, 8, 12), torch.float32).cuda(), make((3, 1, 3, 3), torch.float32).cuda()
    y, codes, scales = torch.empty_like(x), torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(2, 3, 1, device="cuda")
    gw = torch.ones(3, 1, 3, 3, device="cuda")
    before = _native.launch_count()

    def forward(d, x=x, codes=codes):
        return lib.mc_morpho_forward8(ctypes.byref(d), ptr(x), ptr(w), ptr(y), ptr(codes), ptr(scales), stream())

    def backward(d, need=None):
        size = lib.mc_morpho_backward8_workspace_bytes(ctypes.byref(d)) if need is None else need
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        return lib.mc_morpho_backward8(ctypes.byref(d), ptr(codes), ptr(scales), ptr(w), ptr(y), ptr(x), ptr(gw), ptr(ws), ctypes.c_size_t(size), stream())

    good = make_desc("dilation", x, w, "identity")
    for field, value in (("merge", 2), ("dtype", 1), ("W", 13), ("W", 4100), ("kH", 5), ("kW", 7), ("flags", 2)):
        d = make_desc("dilation", x, w, "identity")
        setattr(d, field, value)
        assert forward(d) == -2 and backward(d) == -2, field
        assert lib.mc_morpho_backward8_workspace_bytes(ctypes.byref(d)) == 0
    odd = torch.empty(x.numel() + 1, device="cuda")[1:].view_as(x)
    assert forward(good, x=odd) == -2 and forward(good, codes=None) == -1 and backward(good, need=0) == -3
    bad = make_desc("dilation", x, w, "identity")
    bad.flags = 8
    assert forward(bad) == -1
    empty = make_desc("dilation", x, w, "identity")
    empty.B = 0
    assert forward(empty) == 0
    assert _native.launch_count() == before
    assert backward(empty) == 0 and not gw.any()
    assert forward(good) == 0 and backward(good) == 0 and _native.launch_count() == before + 3


def test_packed_is_not_the_form_of_a_later_layer_s_input():
    """A module derived from a layer that runs two of them, and a hook that runs one: every layer but the one on the caller's tensor encodes
    its own input, and the gradients are those of the calls one by one."""
    class Twice(Mnn.Dilation):
        def forward(self, x):
            return super().forward(super().forward(x))

    layer, plain = Twice(3, 3, 3).cuda(), Mnn.Dilation(3, 3, 3).cuda()
    torch.nn.init.normal_(layer.weight, std=0.1)
    plain.load_state_dict(layer.state_dict())
    x = make((2, 3, 12, 18), torch.float32, 3).cuda().requires_grad_(True)
    packed, g = F.encode_8bit(x.detach()), make((2, 3, 12, 18), torch.float32, 4).cuda()

    def one_by_one():
        return F.checkpoint_8bit(plain, F.checkpoint_8bit(plain, x, packed=packed))

    hooked = Mnn.Dilation(3, 3, 3).cuda()
    hooked.load_state_dict(layer.state_dict())
    hooked.register_forward_hook(lambda module, inputs, y: F.dilation(y, module.weight))
    want = torch.autograd.grad(one_by_one(), (x, plain.weight), g)
    for module in (layer, hooked):
        z = F.checkpoint_8bit(module, x, packed=packed)
        assert bool((z == one_by_one()).all())
        for a, b in zip(torch.autograd.grad(z, (x, module.weight), g), want):
            assert bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())   # atomic sums in float, as elsewhere here
    # One 8-bit form, two layers on the same tensor.
    w = torch.nn.Parameter(make((3, 3, 3, 3), torch.float32, 5).cuda() * 0.1)
    alpha = torch.full((3, 3), 1.5, device="cuda")
    both = F.checkpoint_8bit(F.erosion, x, w, packed=packed) + F.checkpoint_8bit(F.smorph, x, w, alpha, packed=packed)
    at = F.decode_8bit(packed).requires_grad_(True)
    for a, b in zip(torch.autograd.grad(both, (x, w), g), torch.autograd.grad(F.erosion(at, w) + F.smorph(at, w, alpha), (at, w), g)):
        assert bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())


@pytest.mark.parametrize("k", [3, 5])
@pytest.mark.parametrize("shape", PLANES, ids=str)
@pytest.mark.parametrize("op", ["dilation", "erosion"])
def test_per_channel_gradients_count_every_output_once(op, shape, k):
    """Gradients that are whole numbers of at most 8 have sums that float holds exactly (72000 of them a channel, 2^20 at most), in any order:
    an output that a strip or a column tile left out, or took twice, shows in either gradient as a difference."""
    C = shape[1]
    x, w = make(shape, torch.float32, 1), make((C, 1, k, k), torch.float32, 2) * 0.1
    gz = torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(3)).float()
    codes, scales, _ = P.encode(x, 2)
    kept = P.decode(torch.from_numpy(codes), torch.from_numpy(scales), torch.float32)
    wk = w.numpy() if op == "dilation" else np.ascontiguousarray(w.numpy()[..., ::-1, ::-1])
    for padding in ("replicate", "geodesic", "constant"):
        leaves = [x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)]
        z = F.checkpoint_8bit(getattr(F, op), *leaves, channel_merge_mode="identity", padding_mode=padding, padding_value=0.125)
        got = torch.autograd.grad(z, leaves, gz.cuda())
        gx, gw = O.morpho_backward(op, kept.numpy(), wk, gz.numpy(), "identity", padding, 0.125)
        assert np.array_equal(got[0].cpu().numpy(), gx)
        assert np.array_equal(got[1].cpu().numpy(), gw if op == "dilation" else gw[..., ::-1, ::-1])


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation(reentrant):
    """Inside torch.utils.checkpoint the recomputed call keeps its input in 8 bits like the first one."""
    from torch.utils.checkpoint import checkpoint
    norm, layer = Mnn.RMSNorm(4).cuda(), Mnn.Dilation(4, 4, 3).cuda()
    torch.nn.init.normal_(layer.weight, std=0.1)
    x, g = make((2, 4, 12, 18), torch.float32, 3).cuda().requires_grad_(True), make((2, 4, 12, 18), torch.float32, 4).cuda()

    def block(x):
        return F.checkpoint_8bit(torch.nn.Sequential(norm, layer), x)

    inputs = (x, norm.weight, layer.weight)
    want = torch.autograd.grad(block(x), inputs, g)
    y = checkpoint(block, x, use_reentrant=reentrant)
    for t in inputs:
        t.grad = None
    y.backward(g)   # torch.autograd.grad does not go through the reentrant form
    for t, b in zip(inputs, want):
        assert bool(((t.grad - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())   # atomic sums in float, as elsewhere here


def test_threads():
    """Threads on streams of their own, with and without the mode, forward and backward: each gets what it gets alone."""
    import threading
    norm, layer = Mnn.RMSNorm(8).cuda(), Mnn.Dilation(8, 8, 3, "identity").cuda()
    torch.nn.init.normal_(layer.weight, std=0.1)

    def step(i):
        x = make((2, 8, 20, 24 + 4 * i), torch.float32, i).cuda().requires_grad_(True)
        y = norm(x)
        y = F.checkpoint_8bit(layer, y) if i % 2 else layer(y)
        packed = F.encode_8bit(y.detach())
        return (y.detach(), packed.codes, packed.scales, *torch.autograd.grad(y, (x, norm.weight), torch.ones_like(y)))

    wants, results, errors = [step(i) for i in range(4)], [None] * 4, []
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    results[i] = step(i)
        except Exception as e:   # what a thread raises is lost otherwise
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for got, want in zip(results, wants):
        for n, (a, b) in enumerate(zip(got, want)):
            assert bool((a == b).all()) if n < 3 else bool(((a - b).abs() <= 1e-4 * max(1.0, float(b.abs().max()))).all())


def test_recomputation_outside_of_the_mode_is_refused():
    """torch.utils.checkpoint inside the call recomputes after it, without the mode: what was kept does not match, and torch says so."""
    from torch.utils.checkpoint import CheckpointError, checkpoint
    x = make((2, 4, 12, 18), torch.float32, 3).cuda().requires_grad_(True)
    alpha = torch.full((4, 4), 1.5, device="cuda", requires_grad=True)
    w = (make((4, 4, 3, 3), torch.float32, 4) * 0.1).cuda().requires_grad_(True)
    for call in (lambda x: F.dilation(x, w), lambda x: F.dilation(x, w, "max"), lambda x: F.erosion(x, w[:, :1], "identity"), lambda x: F.smorph(x, w, alpha),
                 lambda x: F.sigma_layer(x, w, alpha), lambda x: F.rms_norm(x)):
        y = F.checkpoint_8bit(lambda x: checkpoint(call, x, use_reentrant=False), x)
        with pytest.raises(CheckpointError):
            y.sum().backward()
