"""8-bit activations and the root-mean-square norm, what needs no GPU: the plain implementation itself, the checks of arguments
of the C-ABI and of the Python surface, modules."""
import ctypes
import inspect
import os

import numpy as np
import pytest
import torch

import _plain8 as P
import morphocore_b200.functional as F
import morphocore_b200.nn as Mnn
from conftest import ROOT


class Rows(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("length", ctypes.c_int64), ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class Norm(ctypes.Structure):
    _fields_ = [("outer", ctypes.c_int64), ("channels", ctypes.c_int64), ("inner", ctypes.c_int64), ("eps", ctypes.c_double),
                ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def norm(**kw):
    return Norm(**{**dict(outer=2, channels=8, inner=16, eps=1e-6, dtype=0, reserved=0), **kw})


@pytest.fixture(scope="module")
def lib():
    handle = ctypes.CDLL(os.path.join(ROOT, "morphocore_b200", "libmorphocore_b200.so"))
    handle.mc_last_error.restype = ctypes.c_char_p
    handle.mc_rms_norm_backward_workspace_bytes.restype = ctypes.c_size_t
    return handle


def test_plain_encoding_by_hand():
    x = torch.tensor([[126.0, -63.5, 0.5, 1.5, 2.5, float("inf"), float("nan"), -float("inf")]])
    codes, scales, values = P.encode(x, 1)
    assert codes.tolist() == [[126, -64, 0, 2, 2, 127, -128, -127]]
    assert abs(float(scales[0, 0]) - 1) < 2 ** -23
    assert np.isnan(values[0, 6]) and values[0, 5] == np.inf and values[0, 7] == -np.inf and abs(values[0, 1] + 64) < 1e-4
    codes, scales, values = P.encode(torch.full((1, 130), 2.0 ** -101), 1)
    assert not codes.any() and not scales.any() and scales.shape == (1, 2)


def test_rows_are_refused_before_any_launch(lib):
    one = ctypes.c_void_p(16)   # never dereferenced
    for call, args in ((lib.mc_encode8, (one, one, one, None)), (lib.mc_decode8, (one, one, one, None))):
        assert call(None, *args) == -1
        for bad in (dict(rows=-1, length=4), dict(rows=4, length=-1), dict(rows=2 ** 30, length=2 ** 30), dict(rows=2 ** 62, length=4),
                    dict(rows=4, length=4, dtype=4), dict(rows=4, length=4, dtype=-1), dict(rows=4, length=4, reserved=1)):
            assert call(ctypes.byref(Rows(**bad)), *args) == -1, bad
        for missing in range(3):
            given = [None if n == missing else one for n in range(3)]
            assert call(ctypes.byref(Rows(4, 4, 0, 0)), *given, None) == -1
            assert b"NULL" in lib.mc_last_error()
        assert call(ctypes.byref(Rows(0, 4, 0, 0)), None, None, None, None) == 0
        assert call(ctypes.byref(Rows(4, 0, 3, 0)), None, None, None, None) == 0
    assert lib.mc_launch_count() == 0


def test_norm_is_refused_before_any_launch(lib):
    one, no = ctypes.c_void_p(16), ctypes.c_size_t(0)
    forward, backward = lib.mc_rms_norm_forward, lib.mc_rms_norm_backward
    for bad, code in ((dict(outer=-1), -1), (dict(channels=0), -1), (dict(inner=-1), -1), (dict(outer=2 ** 40), -1), (dict(outer=2 ** 62, inner=8), -1),
                      (dict(dtype=4), -1), (dict(reserved=3), -1), (dict(eps=0.0), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1),
                      (dict(eps=float("inf")), -1), (dict(channels=16385), -2)):
        assert forward(ctypes.byref(norm(**bad)), one, None, None, None, one, None, None, None, None, None) == code, bad
        assert backward(ctypes.byref(norm(**bad)), one, None, None, None, one, None, one, None, None, no, None) == code, bad
        assert lib.mc_rms_norm_backward_workspace_bytes(ctypes.byref(norm(**bad)), 1) == 0
    d = ctypes.byref(norm())
    #                    x    residual weight sum  y    codes scales codes scales
    for args in ((None, None, None, None, one, None, None, None, None), (one, one, None, None, one, None, None, None, None),
                 (one, None, None, one, one, None, None, None, None), (one, None, None, None, one, one, None, None, None),
                 (one, None, None, None, one, None, None, None, one), (one, None, None, None, None, None, None, None, None)):
        assert forward(d, *args, None) == -1, args
    #             sum   codes scales weight gy  gsum  gx   gweight
    for args in ((None, None, None, None, one, None, one, None), (one, one, one, None, one, None, one, None), (None, one, None, None, one, None, one, None),
                 (one, None, None, one, one, None, one, None), (one, None, None, None, None, None, one, None), (one, None, None, None, one, None, None, None)):
        assert backward(d, *args, None, no, None) == -1, args
    need = lib.mc_rms_norm_backward_workspace_bytes(d, 1)
    assert need > 0 and need % (8 * 4) == 0 and lib.mc_rms_norm_backward_workspace_bytes(d, 0) == 0
    assert backward(d, one, None, None, one, one, None, one, one, None, no, None) == -3
    assert backward(d, one, None, None, one, one, None, one, one, one, ctypes.c_size_t(need - 1), None) == -3
    empty = ctypes.byref(norm(outer=0))
    assert forward(empty, None, None, None, None, None, None, None, None, None, None) == 0
    assert backward(empty, None, None, None, None, None, None, None, None, None, no, None) == 0
    assert lib.mc_launch_count() == 0


def test_pointers_that_are_not_read_may_be_null(lib):
    """x of a dilation whose winners are given, y of a smorph without a MAX / MIN merge: the checks go on to the next argument."""
    from test_abi import desc
    one, no = ctypes.c_void_p(16), ctypes.c_size_t(0)
    for merge in (0, 1):
        assert lib.mc_morpho_backward(ctypes.byref(desc(merge=merge)), None, None, one, one, one, one, None, no, None) == -1
        assert lib.mc_last_error().startswith(b"w is NULL")
        assert lib.mc_morpho_backward(ctypes.byref(desc(merge=merge)), None, one, None, one, one, one, None, no, None) == -1
        assert lib.mc_last_error().startswith(b"x is NULL")
        assert lib.mc_smorph_backward(ctypes.byref(desc(merge=merge)), one, one, one, None, one, one, one, one, None, no, None) == -1
        assert lib.mc_last_error().startswith(b"y is NULL")
    assert lib.mc_morpho_backward(ctypes.byref(desc(merge=2)), None, one, one, one, one, one, None, no, None) == -1
    assert lib.mc_last_error().startswith(b"x is NULL")


def test_functions_refuse():
    x = torch.zeros(2, 3, 4, 5)
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.encode_8bit(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.decode_8bit(F.Activation8(torch.zeros(2, 3, 4, 5, dtype=torch.int8), torch.zeros(2, 3, 1), torch.float32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.rms_norm(x)
    with pytest.raises(ValueError, match="Unknown output"):
        F.rms_norm(x, output="16bit")
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.checkpoint_8bit(F.dilation, x, torch.zeros(2, 3, 3, 3))
    packed = F.Activation8(torch.zeros(2, 3, 4, 5, dtype=torch.int8), torch.zeros(2, 3, 1), torch.float32)
    for function in (F.opening, F.rms_norm, lambda x: x, Mnn.RMSNorm(3)):
        with pytest.raises(ValueError, match="packed"):
            F.checkpoint_8bit(function, x, packed=packed)


def test_the_mode_ends_with_the_call():
    from morphocore_b200.functional.activation8 import keeping_8bit, kept_codes
    packed = F.Activation8(torch.zeros(2, dtype=torch.int8), torch.zeros(1), torch.float32)

    def look(inner=False):
        if inner:
            assert F.checkpoint_8bit(look) == (True, (None, None))
        return keeping_8bit(), kept_codes()

    look.takes_packed = True
    assert look() == (False, (None, None))
    active, kept = F.checkpoint_8bit(look, packed=packed, inner=True)
    assert active and kept[0] is packed.codes and kept[1] is packed.scales
    assert look() == (False, (None, None))
    with pytest.raises(ZeroDivisionError):
        F.checkpoint_8bit(lambda: 1 / 0)
    assert look() == (False, (None, None))


def test_signatures_and_module():
    assert list(inspect.signature(F.rms_norm).parameters) == ["x", "weight", "residual", "eps", "dim", "output"]
    m = Mnn.RMSNorm(5, eps=1e-5, dtype=torch.float64)
    assert m.weight.shape == (5,) and m.weight.dtype == torch.float64 and bool((m.weight == 1).all()) and set(m.state_dict()) == {"weight"}
    packed = F.Activation8(torch.zeros(2, 3, dtype=torch.int8), torch.zeros(2, 1), torch.float32)
    assert packed.shape == (2, 3) and packed.nbytes == 14


def test_packed_belongs_to_one_tensor():
    """The codes that a caller hands over go to layers on that very tensor, in that very state."""
    from morphocore_b200.functional.activation8 import kept_codes
    x, other = torch.zeros(2, 3), torch.zeros(2, 3)
    packed = F.Activation8(torch.zeros(2, 3, dtype=torch.int8), torch.zeros(2, 1), torch.float32)

    def look(x):
        seen = [kept_codes(x), kept_codes(other), kept_codes(x.view(2, 3)), F.checkpoint_8bit(lambda x: kept_codes(x), x), kept_codes(x)]
        x.add_(1)
        return seen + [kept_codes(x)]

    look.takes_packed = True
    codes, no = (packed.codes, packed.scales), (None, None)
    for call in (lambda: F.checkpoint_8bit(look, x, packed=packed), lambda: F.checkpoint_8bit(look, x=x, packed=packed)):
        for got, want in zip(call(), (codes, no, no, no, codes, no)):
            assert got[0] is want[0] and got[1] is want[1]
    with torch.inference_mode():
        inside = torch.zeros(2, 3)
        assert F.checkpoint_8bit(look, inside, packed=packed)[0][0] is packed.codes


def test_norm_flags_are_refused_before_any_launch(lib):
    """float weights go with tensors in half precision alone, and no other bit means anything."""
    one, no = ctypes.c_void_p(16), ctypes.c_size_t(0)
    for bad in (dict(dtype=0, reserved=1), dict(dtype=1, reserved=1), dict(dtype=2, reserved=2), dict(dtype=3, reserved=3), dict(dtype=2, reserved=-1)):
        d = ctypes.byref(norm(**bad))
        assert lib.mc_rms_norm_forward(d, one, None, one, None, one, None, None, None, None, None) == -1, bad
        assert lib.mc_rms_norm_backward(d, one, None, None, one, one, None, one, one, None, no, None) == -1, bad
        assert lib.mc_rms_norm_backward_workspace_bytes(d, 1) == 0
    for dtype in (2, 3):
        d = ctypes.byref(norm(dtype=dtype, reserved=1))
        assert lib.mc_rms_norm_forward(d, None, None, one, None, one, None, None, None, None, None) == -1
        assert lib.mc_last_error() == b"x is NULL"
        assert lib.mc_rms_norm_backward_workspace_bytes(d, 1) == lib.mc_rms_norm_backward_workspace_bytes(ctypes.byref(norm(dtype=dtype)), 1)
        assert lib.mc_rms_norm_backward(d, one, None, None, one, one, None, one, one, None, no, None) == -3
    assert lib.mc_launch_count() == 0


def test_norm_gradient_thread_blocks_have_tiles(lib):
    """A row of partial sums for every thread block of the backward pass, and a tile, or a row of channels, for each of them at least:
    tiles are 32 to 128 pixels of an image."""
    for dtype, size in ((0, 4), (1, 8), (2, 4), (3, 4)):
        for channels in (1, 32, 33, 64, 65, 128, 129, 256, 257, 512, 513, 16384):
            for outer, inner in ((1, 2), (1, 32), (3, 32), (1, 33), (2, 128), (1, 129), (100000, 3), (1, 10 ** 6)):
                rows, rest = divmod(lib.mc_rms_norm_backward_workspace_bytes(ctypes.byref(norm(outer=outer, channels=channels, inner=inner, dtype=dtype)), 1), size * channels)
                assert rest == 0 and outer * -(-inner // 128) >= 592 or outer * -(-inner // 128) <= rows <= outer * -(-inner // 32), (dtype, channels, outer, inner, rows)
                assert 1 <= rows <= 592
            for outer in (1, 5, 100000):
                rows, rest = divmod(lib.mc_rms_norm_backward_workspace_bytes(ctypes.byref(norm(outer=outer, channels=channels, inner=1, dtype=dtype)), 1), size * channels)
                assert rest == 0 and 1 <= rows <= min(outer, 296)


def test_the_mode_is_that_of_one_thread():
    import threading

    from morphocore_b200.functional.activation8 import keeping_8bit
    seen = []

    def look():
        other = threading.Thread(target=lambda: seen.append(keeping_8bit()))
        other.start()
        other.join()
        return keeping_8bit()

    assert F.checkpoint_8bit(look) and seen == [False] and not keeping_8bit()
