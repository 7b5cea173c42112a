"""Performance cases of the 8-bit activations and of the root-mean-square norm: what a user's program calls, over the range
of sizes it calls it with.

A case is a dict of plain values; `kind` says which path it takes:

  norm    functional.rms_norm of a sum with a residual, the output in 8 bits, read back (a cache of normalised features)
  train   functional.rms_norm with residual, forward and backward; `keep8`: what the backward pass needs is kept in 8 bits
  store   functional.encode_8bit and decode_8bit: activations put away in 8 bits and fetched again
  layer   a morphological layer whose input is kept in 8 bits for the backward pass, forward and backward
  block   norm, then a layer whose 8-bit input the norm has already written; forward and backward of both

An 8-bit activation is seen as rows (a plane of H x W pixels, or a token's channels), cut into blocks of 128 elements, the
last of a row shorter. With m the largest finite magnitude of a block, scale = m / 126 and code = round(x * (126 / m)), ties
to even; magnitudes below 2^-100 (2^-900 in double) throughout a block are stored as zeros; infinities and NaN keep codes of
their own. The gradients of a layer that keeps its input in 8 bits are those at the values which the codes stand for.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 128
EPS = 1e-6


def _norm(name, kind, dtype, N, C, H, W, tokens=False, residual=True, keep8=False):
    """tokens: the tensor is (N, C), normalised along its last dimension; otherwise (N, C, H, W), normalised over C."""
    c = dict(kind=kind, dtype=dtype, N=N, C=C, H=H, W=W, tokens=tokens, residual=residual, keep8=keep8)
    return dict(c, name=name) if name else c


def _store(name, dtype, N, C, H, W, masked):
    c = dict(kind="store", dtype=dtype, N=N, C=C, H=H, W=W, masked=masked)
    return dict(c, name=name) if name else c


def _layer(name, kind, op, merge, N, C, Co, H, W, k, alpha=0.0):
    c = dict(kind=kind, op=op, merge=merge, dtype="float32", N=N, C=C, Co=Co, H=H, W=W, k=k, alpha_mean=alpha)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One sample's last feature maps, normalised and cached in 8 bits: the smallest call, all latency.
        _norm("norm_one_sample", "norm", "float32", 1, 64, 7, 7),
        # Features of a batch of crops in half precision, cached in 8 bits.
        _norm("norm_half_batch", "norm", "float16", 16, 64, 56, 56),
        # Feature maps of full-size images (the hidden layers of benchmark configuration 5), cached in 8 bits.
        _norm("norm_images", "norm", "float32", 32, 64, 224, 224),
        # Training of a norm on odd image sizes (rows that are not 16-byte aligned), its input kept in 8 bits.
        _norm("train_ragged_keep8", "train", "float32", 5, 20, 75, 101, keep8=True),
        # Mixed-precision training of a norm in the middle of a network, its input kept as it is.
        _norm("train_bf16", "train", "bfloat16", 16, 128, 112, 112),
        # Pooled features, one row of channels a sample.
        _norm("train_rows_keep8", "train", "float32", 8192, 512, 1, 1, tokens=True, keep8=True),
        # Activations of odd sizes, one pixel in a hundred masked with -inf as a geodesic border does.
        _store("store_ragged_masked", "float32", 5, 12, 75, 101, True),
        # Activations of full-size images in mixed precision.
        _store("store_bf16_images", "bfloat16", 32, 64, 224, 224, False),
        # Per-channel dilation of middle-sized feature maps: as many bytes as arithmetic.
        _layer("dilation_identity", "layer", "dilation", "identity", 16, 64, 64, 112, 112, 3),
        # Training of an erosion layer that mixes channels.
        _layer("erosion_sum", "layer", "erosion", "sum", 8, 16, 32, 64, 64, 5),
        # Smooth layer of a classifier on small feature maps.
        _layer("smorph_28", "layer", "smorph", "sum", 8, 8, 16, 28, 28, 3, alpha=1.0),
        # One residual block of the smooth network: norm, then the smooth layer, nothing kept in more than 8 bits.
        _layer("block_smorph_56", "block", "smorph", "mean", 8, 32, 32, 56, 56, 3, alpha=2.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _side(rng, lo, hi):
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.5 else max(lo, n // 8 * 8)  # half of the images have sides that are multiples of 8


def _draw_one(rng):
    kind = rng.choices(("norm", "train", "store", "layer", "block"), (3, 4, 2, 3, 2))[0]
    dtype = rng.choices(("float32", "bfloat16", "float16", "float64"), (6, 3, 1.5, 1))[0]
    N, C, H = _log(rng, 1, 32), _log(rng, 4, 512), _side(rng, 2, 512)
    W = H if rng.random() < 0.4 else _side(rng, max(2, int(H * 0.6)), max(3, int(H * 1.7)))
    if kind in ("norm", "train"):
        tokens = rng.random() < 0.3
        if tokens:
            N, C, H, W = _log(rng, 1, 65536), _side(rng, 8, 8192), 1, 1
        return _norm(None, kind, dtype, N, C, H, W, tokens, rng.random() < 0.7, kind == "train" and rng.random() < 0.6)
    if kind == "store":
        return _store(None, dtype, N, C, H, W, rng.random() < 0.3)
    op = "smorph" if kind == "block" else rng.choice(("dilation", "erosion", "smorph"))
    merge = rng.choice(("sum", "mean", "identity"))
    C, Co, H, W = _log(rng, 1, 64), _log(rng, 1, 64), max(H, 5), max(W, 5)
    if merge == "identity":
        Co = C
    return _layer(None, kind, op, merge, min(N, 16), C, Co, H, W, rng.choices((3, 5, 7), (5, 3, 1))[0], rng.choice((-2.0, 0.5, 1.0, 2.0)) if op == "smorph" else 0.0)


def draw(rng):
    """One more case: 1 to 32 images of 4 to 512 channels and sides of 2 to 512, or 1 to 65536 rows of 8 to 8192 channels, every
    type, with and without residual; layers of 1 to 64 channels and structuring elements of 3 x 3 to 7 x 7. At most 100 M elements a
    tensor (a quarter of that in double), 220 M taps a layer."""
    while True:
        c = _draw_one(rng)
        elements = c["N"] * c["C"] * c["H"] * c["W"] * (4 if c["dtype"] == "float64" else 1)
        if elements <= 100e6 and ("k" not in c or (_taps(c) <= 220e6 and elements <= 14e6)):
            return c


def _taps(c):
    return c["N"] * c["Co"] * (1 if c["merge"] == "identity" else c["C"]) * c["H"] * c["W"] * c["k"] ** 2


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        work = torch.float64 if dtype == torch.float64 else torch.float32
        return (torch.randn(shape, generator=g, device="cuda", dtype=work) * scale + shift).to(dtype)

    s = dict(case)
    N, C, H, W = (case[k] for k in "NCHW")
    shape = (N, C) if case.get("tokens") else (N, C, H, W)
    if case["kind"] == "store":
        x = normal(*shape)
        if case["masked"]:
            x.masked_fill_(torch.rand(shape, generator=g, device="cuda") < 0.01, -math.inf)
        return dict(s, x=x)
    s["x"] = normal(*shape)
    if case["kind"] in ("norm", "train", "block"):
        s["weight"] = normal(C, scale=0.2, shift=1.0)
        s["residual"] = normal(*shape) if case.get("residual", True) else None
    if case["kind"] in ("train", "block"):
        s["gsum"] = normal(*shape) if s["residual"] is not None else None
    if case["kind"] == "train":
        s["gy"] = normal(*shape)
    if case["kind"] in ("layer", "block"):
        identity, k = case["merge"] == "identity", case["k"]
        s["w"] = normal(case["Co"], 1 if identity else C, k, k, scale=0.1)
        if case["op"] == "smorph":
            s["alpha"] = normal(case["Co"], 1 if identity else C, scale=0.25, shift=case["alpha_mean"])
        s["gz"] = normal(N, case["Co"], H, W)
    if case["kind"] != "norm":
        for name in ("x", "residual", "weight", "w", "alpha"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def _own(s):
    import morphocore_b200.functional as F

    kind = s["kind"]
    if kind == "store":
        packed = F.encode_8bit(s["x"])
        return F.decode_8bit(packed), packed.scales
    dim = -1 if s.get("tokens") else -3
    if kind == "norm":
        with torch.no_grad():
            out = F.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS, dim=dim, output="8bit")
            packed, total = out if s["residual"] is not None else (out, None)
            return F.decode_8bit(packed), packed.scales, total
    if kind == "train":
        args = (F.rms_norm, s["x"], s["weight"], s["residual"], EPS, dim)
        out = F.checkpoint_8bit(*args) if s["keep8"] else args[0](*args[1:])
        if s["residual"] is None:
            return (out, *torch.autograd.grad(out, (s["x"], s["weight"]), s["gy"]))
        gx, _, gweight = torch.autograd.grad(out, (s["x"], s["residual"], s["weight"]), (s["gy"], s["gsum"]))
        return (*out, gx, gweight)
    if kind == "layer":
        leaves = [s["x"], s["w"]] + ([s["alpha"]] if "alpha" in s else [])
        if s["op"] == "smorph":
            z = F.checkpoint_8bit(F.smorph, *leaves, channel_merge_mode=s["merge"])
        else:
            z = F.checkpoint_8bit(F.dilation if s["op"] == "dilation" else F.erosion, *leaves, s["merge"])
        return (z, *torch.autograd.grad(z, leaves, s["gz"]))
    y, packed, total = F.checkpoint_8bit(F.rms_norm, s["x"], s["weight"], s["residual"], EPS, dim, "both")
    z = F.checkpoint_8bit(F.smorph, y, s["w"], s["alpha"], channel_merge_mode=s["merge"], packed=packed)
    gx, _, *more = torch.autograd.grad((z, total), (s["x"], s["residual"], s["weight"], s["w"], s["alpha"]), (s["gz"], s["gsum"]))
    return (z, total, gx, *more)


# ---- the plain form -------------------------------------------------------------------------------------------------------


def _wide(t):
    return t.double() if t.dtype == torch.float64 else t.float()


def _coded(x, row_dims):
    """The values that the 8-bit form of x stands for, in x's type, and the scales. Products with 126 / m are taken in 64 bits,
    where they are exact: a rounding before the one to a whole number would move values that lie next to a border."""
    v = _wide(x)
    lead = x.shape[:-row_dims]
    rows = v.reshape(math.prod(lead), -1)
    length = rows.shape[1]
    blocks = -(-length // BLOCK)
    v = torch.zeros(rows.shape[0], blocks * BLOCK, dtype=v.dtype, device=v.device)
    v[:, :length] = rows
    v = v.view(-1, blocks, BLOCK)
    finite = torch.isfinite(v)
    top = torch.where(finite, v.abs(), torch.zeros_like(v)).amax(-1, keepdim=True)
    none = top < (2.0 ** -900 if v.dtype == torch.float64 else 2.0 ** -100)
    zero = torch.zeros_like(top)
    scale = torch.where(none, zero, top * torch.full_like(top, 1 / 126))
    inverse = torch.where(none, zero, torch.full_like(top, 126.0) / top)
    code = torch.round(torch.where(finite, v, torch.zeros_like(v)).double() * inverse.double()).to(v.dtype)
    values = torch.where(finite, code * scale, v).view(rows.shape[0], -1)[:, :length]
    return values.reshape(x.shape).to(x.dtype), scale.view(*lead, blocks)


def _normed(x, weight, residual, dim):
    """Sum and norm. In 64 bits: what the codes of the result are depends on which side of a border it lies."""
    total = x if residual is None else (_wide(x) + _wide(residual)).to(x.dtype)
    v = total.double()
    factor = (v.square().mean(dim, keepdim=True) + EPS).rsqrt()
    return (v * factor * _along(weight.double(), dim)).to(x.dtype), total


def _along(weight, dim):
    return weight if dim == -1 else weight.view(-1, 1, 1)


def _normed_backward(v, weight, gy, gsum, dim):
    """Gradients of the norm at the sum v (in 32 bits or more): of the sum, and of the weight."""
    g = _wide(gy)
    factor = (v.square().mean(dim, keepdim=True) + EPS).rsqrt()
    scaled = g * _along(_wide(weight), dim)
    grad = factor * (scaled - v * factor.square() * (scaled * v).mean(dim, keepdim=True))
    if gsum is not None:
        grad = grad + _wide(gsum)
    others = [d for d in range(v.dim()) if d != v.dim() + dim]
    return grad.to(gy.dtype), (g * v * factor).sum(others, dtype=torch.float64).to(gy.dtype)


def _positions(H, W, k, device):
    """Input row and column of tap (kh, kw) of output pixel (h, w), and whether it lies inside the image."""
    at = torch.arange(k, device=device)
    rows = torch.arange(H, device=device)[None, :] + k // 2 - at[:, None]
    cols = torch.arange(W, device=device)[None, :] + k // 2 - at[:, None]
    inside = ((rows >= 0) & (rows < H))[:, None, :, None] & ((cols >= 0) & (cols < W))[None, :, None, :]
    place = rows.clamp(0, H - 1)[:, None, :, None] * W + cols.clamp(0, W - 1)[None, :, None, :]
    return place.reshape(k * k, H * W), inside.reshape(k * k, H * W)


def _tap_values(x, w, op, place, identity):
    """x + w (or x - flipped w) of every tap: [N, Co, Ci, taps, pixels], Ci = 1 for the identity merge."""
    N, C = x.shape[:2]
    taps = x.reshape(N, C, -1)[:, :, place]
    taps = taps.unsqueeze(2) if identity else taps.unsqueeze(1)
    w = w.reshape(w.shape[0], w.shape[1], -1, 1)
    return taps - w.flip(2) if op == "erosion" else taps + w


def _scattered(pieces, place, x, identity):
    """Adds [N, Co, Ci, taps, pixels] (or the sum over Co of it) at the input pixels that the taps read, in 64 bits."""
    N, C, H, W = x.shape
    pieces = pieces.squeeze(2) if identity else pieces.sum(1)
    out = torch.zeros(N, C, H * W, dtype=torch.float64, device=x.device)
    return out.scatter_add_(2, place.reshape(1, 1, -1).expand(N, C, -1), pieces.reshape(N, C, -1).double()).view(N, C, H, W)


def _merged(per_pair, merge, x):
    N, Co, Ci = per_pair.shape[:3]
    return (per_pair.sum(2) if merge != "mean" else per_pair.sum(2) / Ci).view(N, Co, *x.shape[2:])


def _spread(gz, merge, Ci):
    g = gz.reshape(gz.shape[0], gz.shape[1], 1, 1, -1)
    return g / Ci if merge == "mean" else g


def _winners(v, op):
    """Lowest tap whose value is the extremum: [N, Co, Ci, taps, pixels], true at one tap of each pixel."""
    best = v.amin(3, keepdim=True) if op == "erosion" else v.amax(3, keepdim=True)
    tap = torch.arange(v.shape[3], device=v.device, dtype=torch.int32).view(1, 1, 1, -1, 1)
    return tap == torch.where(v == best, tap, v.shape[3]).amin(3, keepdim=True)


def _morph(x, w, op, merge):
    place, _ = _positions(*x.shape[2:], w.shape[-1], x.device)
    v = _tap_values(x, w, op, place, merge == "identity")
    return _merged(v.amin(3) if op == "erosion" else v.amax(3), merge, x)


def _morph_backward(x, w, op, merge, gz):
    identity = merge == "identity"
    place, inside = _positions(*x.shape[2:], w.shape[-1], x.device)
    won = _winners(_tap_values(x, w, op, place, identity), op)
    share = won * _spread(gz, merge, x.shape[1])
    gw = share.sum((0, 4), dtype=torch.float64)
    gw = -gw.flip(2) if op == "erosion" else gw
    # A winning tap outside the image, which read the nearest edge pixel, counts for the weight alone.
    return _scattered(share * inside, place, x, identity), gw.view(w.shape)


def _tilde(w, alpha):
    t = torch.tanh(alpha).view(alpha.shape[0], -1, 1, 1)
    return t, t * ((1 - t) / 2 * w.flip(2, 3) + (1 + t) / 2 * w)


def _soft(x, w, alpha, merge):
    place, inside = _positions(*x.shape[2:], w.shape[-1], x.device)
    v = _tap_values(x, _tilde(w, alpha)[1], "smorph", place, merge == "identity")
    a = alpha.view(1, *alpha.shape, 1, 1)
    z = torch.where(inside, v * a, torch.full_like(v[:1, :1, :1, :1, :1], -math.inf))
    p = torch.exp(z - z.amax(3, keepdim=True))
    p = p / p.sum(3, keepdim=True)
    return place, a, v, p, (p * v).sum(3, keepdim=True)


def _smorph(x, w, alpha, merge):
    return _merged(_soft(x, w, alpha, merge)[4].squeeze(3), merge, x)


def _smorph_backward(x, w, alpha, merge, gz):
    place, a, v, p, out = _soft(x, w, alpha, merge)
    g, off = _spread(gz, merge, x.shape[1]), v - out
    share = g * p * (1 + a * off)
    t, _ = _tilde(w, alpha)
    gt = share.sum((0, 4), dtype=torch.float64).view(w.shape)
    galpha = (g * (p * off * off).sum(3, keepdim=True)).sum((0, 3, 4), dtype=torch.float64)
    t, w = t.double(), w.double()
    straight, mirrored, flipped = (1 + t) / 2, (1 - t) / 2, w.flip(2, 3)
    through = mirrored * flipped + straight * w + t * (w - flipped) / 2
    galpha = galpha + (1 - t * t).view(alpha.shape) * (gt * through).sum((2, 3))
    return _scattered(share, place, x, merge == "identity"), t * (straight * gt + mirrored * gt.flip(2, 3)), galpha


def _plain(s):
    kind = s["kind"]
    if kind == "store":
        return _coded(s["x"], 2)
    dim = -1 if s.get("tokens") else -3
    row_dims = 1 if s.get("tokens") else 2
    if kind == "layer":
        kept = _coded(s["x"], 2)[0]
        if s["op"] == "smorph":
            z = _smorph(s["x"], s["w"], s["alpha"], s["merge"])
            grads = _smorph_backward(kept, s["w"], s["alpha"], s["merge"], s["gz"])
        else:
            z = _morph(s["x"], s["w"], s["op"], s["merge"])
            grads = _morph_backward(kept, s["w"], s["op"], s["merge"], s["gz"])
        return (z, *(g.float() for g in grads))
    y, total = _normed(s["x"], s["weight"], s["residual"], dim)
    if kind == "norm":
        return (*_coded(y, row_dims), total if s["residual"] is not None else None)
    if kind == "train":
        kept = _wide(_coded(total, row_dims)[0] if s["keep8"] else total)
        grads = _normed_backward(kept, s["weight"], s["gy"], s["gsum"], dim)
        return (y, total, *grads) if s["residual"] is not None else (y, *grads)
    z = _smorph(y, s["w"], s["alpha"], s["merge"])
    gy, gw, galpha = _smorph_backward(_coded(y, 2)[0], s["w"], s["alpha"], s["merge"], s["gz"])
    gx, gweight = _normed_backward(_coded(total, 2)[0], s["weight"], gy.float(), s["gsum"], dim)
    return z, total, gx, gweight, gw.float(), galpha.float()


# ---- what the path cannot do without --------------------------------------------------------------------------------------


def work(case):
    """Bytes: every input and output once, and the 8-bit form once written and once read where the path has one. Operations:
    a few an element for the norms and codes; for the layers' taps two forward and four backward (dilation, erosion), five
    and eleven (smorph)."""
    size = {"float64": 8, "float32": 4}.get(case["dtype"], 2)
    n = case["N"] * case["C"] * case["H"] * case["W"]
    kind, packed = case["kind"], n + 4 * -(-n // BLOCK)
    if kind == "store":
        return {"bytes": 2 * n * size + 2 * packed, "flops": 4 * n}
    if kind == "norm":
        return {"bytes": n * size * (4 if case["residual"] else 2) + 2 * packed, "flops": 8 * n}
    if kind == "train":
        forward = n * size * (4 if case["residual"] else 2) + (packed if case["keep8"] else 0)
        backward = n * size * (3 if case["residual"] else 2) + (packed if case["keep8"] else n * size)
        return {"bytes": forward + backward, "flops": 20 * n}
    out = case["N"] * case["Co"] * case["H"] * case["W"]
    flops = _taps(case) * (16 if case["op"] == "smorph" else 6)
    if kind == "layer":
        return {"bytes": 2 * (n + out) * size + 2 * packed, "flops": flops}
    # Block: x, residual, sum, output, both packed forms written; gradients of output and sum, both packed forms, gradient of x.
    return {"bytes": (5 * n + 2 * out) * size + 4 * packed, "flops": flops + 20 * n}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        return _exact(prepare(case, seed))


def _exact_codes(x, row_dims):
    """Decoded values in 64 bits, from float64 x whose codes are those of an x held in the type `like`."""
    like = x.dtype
    v = x.double().reshape(math.prod(x.shape[:-row_dims]), -1)
    rows, length = v.shape
    index = torch.arange(length, device=v.device) // BLOCK
    magnitude = torch.where(torch.isfinite(v), v.abs(), 0.0)
    top = torch.zeros(rows, -(-length // BLOCK), dtype=torch.float64, device=v.device)
    top.scatter_reduce_(1, index.expand(rows, -1), magnitude, "amax")
    held = torch.float64 if like == torch.float64 else torch.float32  # the type that the scales and 126 / m are held in
    few = top < (2.0 ** -900 if like == torch.float64 else 2.0 ** -100)
    inverse = torch.where(few, 0.0, 126.0 / top).to(held).double()
    scale = torch.where(few, 0.0, top / 126.0)
    code = torch.round(v * inverse[:, index])
    values = torch.where(torch.isfinite(v), code * scale[:, index], v)
    return values.reshape(x.shape), scale.view(*x.shape[:-row_dims], -1)


def _exact_norm_gradients(v, weight, gy, gsum, dim):
    C = v.shape[dim]
    weight = weight.double().view([-1] + [1] * (-1 - dim))
    r = 1 / torch.sqrt((v * v).sum(dim, keepdim=True) / C + EPS)
    unit = v * r
    through = gy.double() * weight
    grad = r * (through - unit * (through * unit).sum(dim, keepdim=True) / C)
    gweight = (gy.double() * unit).transpose(0, dim).reshape(C, -1).sum(1)
    return grad if gsum is None else grad + gsum.double(), gweight


def _unfolded(x, k, replicate):
    """[N, C, taps, H, W]: tap (kh, kw) of pixel (h, w) is x[h + k // 2 - kh, w + k // 2 - kw], from a padded copy."""
    N, C, H, W = x.shape
    before, after = k - 1 - k // 2, k // 2
    if replicate:
        rows = torch.arange(-before, H + after, device=x.device).clamp(0, H - 1)
        cols = torch.arange(-before, W + after, device=x.device).clamp(0, W - 1)
        padded = x[:, :, rows][:, :, :, cols]
    else:
        padded = torch.full((N, C, H + k - 1, W + k - 1), math.nan, dtype=x.dtype, device=x.device)
        padded[:, :, before:before + H, before:before + W] = x
    windows = padded.unfold(2, k, 1).unfold(3, k, 1)          # [N, C, H, W, k, k], offsets ascending
    return windows.flip(4, 5).permute(0, 1, 4, 5, 2, 3).reshape(N, C, k * k, H, W)


def _folded(taps, H, W, k):
    """Adds [N, C, taps, H, W] at the pixels of [N, C, H, W] that the taps read; those outside the image are lost."""
    N, C = taps.shape[:2]
    before = k - 1 - k // 2
    padded = torch.zeros(N, C, H + k - 1, W + k - 1, dtype=taps.dtype, device=taps.device)
    for tap in range(k * k):
        kh, kw = k - 1 - tap // k, k - 1 - tap % k
        padded[:, :, kh:kh + H, kw:kw + W] += taps[:, :, tap]
    return padded[:, :, before:before + H, before:before + W]


def _exact_layer(s, x, kept):
    """Output of the layer at x, gradients at `kept`: float64, but dilation and erosion choose the winning tap among values as the
    tensor's type holds them, which is what decides between values that are the same in it."""
    merge, k, op = s["merge"], s["k"], s["op"]
    N, C, H, W = x.shape
    identity = merge == "identity"
    count = C if merge == "mean" else 1
    side = 2 if identity else 1                                # where taps get their missing channel dimension
    gz = s["gz"].double()[:, :, None, None] / count            # [N, Co, 1, 1, H, W]
    w = s["w"].double()
    if op == "smorph":
        alpha = s["alpha"].double()
        t = torch.tanh(alpha)[..., None, None]
        turned = torch.flip(w, (2, 3))
        used = (t * (((1 - t) * turned + (1 + t) * w) / 2)).reshape(*w.shape[:2], -1, 1, 1)
        a = alpha[:, :, None, None, None]

        def soft(image):
            v = _unfolded(image, k, False).unsqueeze(side) + used
            p = torch.softmax(torch.where(torch.isnan(v), -math.inf, a * v), 3)
            v = torch.nan_to_num(v)
            return v, p, (p * v).sum(3)

        z = soft(x.double())[2].sum(2) / count
        v, p, out = soft(kept.double())
        spread = v - out.unsqueeze(3)
        share = gz * p * (1 + a * spread)
        galpha = (gz * p * spread * spread).sum((0, 3, 4, 5))
        gt = share.sum((0, 4, 5)).view(w.shape)
        half = t / 2
        galpha = galpha + ((1 - t * t) * gt * (((1 - t) * turned + (1 + t) * w) / 2 + half * (w - turned))).sum((2, 3))
        gw = half * ((1 + t) * gt + (1 - t) * torch.flip(gt, (2, 3)))
        more = (gw, galpha)
    else:
        sign = -1.0 if op == "erosion" else 1.0
        used = (torch.flip(w, (2, 3)) if op == "erosion" else w).reshape(*w.shape[:2], -1, 1, 1)
        # The extremum of sign * (value): a maximum in both cases.
        z = sign * (sign * _unfolded(x.double(), k, True).unsqueeze(side) + used).amax(3).sum(2) / count
        v = sign * _unfolded(kept, k, True).unsqueeze(side) + used.to(kept.dtype)
        order = torch.arange(k * k, 0, -1, device=v.device, dtype=torch.int32).view(1, 1, 1, -1, 1, 1)
        first = k * k - torch.where(v == v.amax(3, keepdim=True), order, 0).amax(3, keepdim=True)
        share = torch.where(k * k - order == first, gz, 0.0)
        gw = sign * share.sum((0, 4, 5)).view(w.shape)
        more = (torch.flip(gw, (2, 3)) if op == "erosion" else gw,)
    gx = _folded(share.sum(2) if identity else share.sum(1), H, W, k)
    return z, gx, more


def _exact(s):
    kind = s["kind"]
    if kind == "store":
        return _exact_codes(s["x"], 2)
    dim, row_dims = (-1, 1) if s.get("tokens") else (-3, 2)
    if kind == "layer":
        kept = _exact_codes(s["x"], 2)[0].float()
        z, gx, more = _exact_layer(s, s["x"], kept)
        return (z, gx, *more)
    x, weight, residual = s["x"], s["weight"], s["residual"]
    total = x if residual is None else (x + residual if x.dtype == torch.float64 else (x.float() + residual.float()).to(x.dtype))
    v = total.double()
    y = v / torch.sqrt((v * v).sum(dim, keepdim=True) / v.shape[dim] + EPS) * weight.double().view([-1] + [1] * (-1 - dim))
    if kind == "norm":
        values, scale = _exact_codes(y.to(x.dtype), row_dims)
        return values, scale, None if residual is None else x.double() + residual.double()
    kept = _exact_codes(total, row_dims)[0].to(total.dtype).double() if s.get("keep8", True) else v
    if kind == "train":
        grads = _exact_norm_gradients(kept, weight, s["gy"], s["gsum"], dim)
        return (y, x.double() + residual.double(), *grads) if residual is not None else (y, *grads)
    y = y.float()
    z, gy, more = _exact_layer(s, y, _exact_codes(y, 2)[0].float())
    gx, gweight = _exact_norm_gradients(kept, weight, gy.float(), s["gsum"], dim)
    return (z, v, gx, gweight, *more)
