"""Refusals of the dense-layer entry points that need no GPU, and the 64-bit references' own checks."""
import ctypes
import math

import numpy as np
import pytest
import torch

import dense_util as U
from kaldi_amd import _lib, dense


def convert(x, rows, cols, out):
    return _lib.lib().amlike_convert_dev(x, rows, cols, out, None)


def matrix(ptr=4096, type_="bf16", ld=64, scales=0, ld_scales=0):
    return dense.Matrix(ptr, type_, ld, scales, ld_scales).ref


@pytest.mark.parametrize("x,rows,cols,out,text", [
    (dict(), -1, 64, dict(ptr=1 << 20), "rows"),
    (dict(), 4, 0, dict(ptr=1 << 20), "columns"),
    (dict(), 4, (1 << 30) + 1, dict(ptr=1 << 20), "columns"),
    (dict(ptr=0), 4, 64, dict(ptr=1 << 20), "no data"),
    (dict(ptr=4097), 4, 64, dict(ptr=1 << 20), "aligned"),
    (dict(ld=63), 4, 64, dict(ptr=1 << 20), "stride"),
    (dict(ld=-64), 4, 64, dict(ptr=1 << 20), "stride"),
    (dict(ld=1 << 60), 4, 64, dict(ptr=1 << 20), "stride"),
    (dict(), 4, 64, dict(ptr=1 << 20, ld=63), "stride"),
    (dict(), 4, 64, dict(ptr=1 << 20, type_="mx8"), "scales"),
    (dict(), 4, 64, dict(ptr=1 << 20, type_="mx8", scales=1 << 21, ld_scales=1), "stride"),
    (dict(type_="mx8", scales=1 << 21, ld_scales=2), 4, 64, dict(ptr=1 << 20), "8 bits"),
    (dict(), 4, 64, dict(ptr=4096), "overlap"),
    (dict(), 4, 64, dict(ptr=4096 + 4 * 64 * 2 - 2), "overlap"),
    (dict(), 4, 64, dict(ptr=1 << 20, type_="mx8", scales=4100, ld_scales=2), "overlap"),
])
def test_convert_refuses(x, rows, cols, out, text):
    assert convert(matrix(**x), rows, cols, matrix(**out)) == _lib.EINVAL
    assert text in _lib.lib().amlike_last_error().decode()


def test_convert_refuses_unknown_types_and_null():
    bad = _lib.Matrix(4096, 0, 64, 0, 4)
    assert convert(ctypes.byref(bad), 4, 64, matrix(ptr=1 << 20)) == _lib.EINVAL
    bad.type = -1
    assert convert(matrix(), 4, 64, ctypes.byref(bad)) == _lib.EINVAL
    assert convert(None, 4, 64, matrix()) == _lib.EINVAL
    assert convert(matrix(), 4, 64, None) == _lib.EINVAL
    assert convert(matrix(ptr=0), 0, 64, matrix(ptr=0)) == _lib.OK  # no rows: nothing to look at


def test_create_refuses():
    L, h = _lib.lib(), ctypes.c_void_p()
    fp = ctypes.POINTER(ctypes.c_float)
    w = np.ones((4, 8), np.float32)
    p = w.ctypes.data_as(fp)
    for args in ((None, 8, None, 8, 4, 1), (p, 7, None, 8, 4, 1), (p, 8, None, 0, 4, 1), (p, 8, None, 8, 0, 1), (p, 8, None, 8, 4, 0),
                 (p, 8, None, 8, 4, 4), (p, (1 << 20) + 1, None, (1 << 20) + 1, 4, 1), (p, 8, None, 8, (1 << 20) + 1, 1)):
        assert L.amlike_linear_create(*args, ctypes.byref(h)) == _lib.EINVAL and not h.value
    assert L.amlike_linear_create(p, 8, None, 8, 4, 1, None) == _lib.EINVAL
    for dim, eps in ((0, 1e-5), (-1, 1e-5), (32769, 1e-5), (8, 0.0), (8, -1.0), (8, 2.0), (8, math.nan), (8, math.inf), (8, 1e-31)):
        assert L.amlike_norm_create(None, dim, eps, ctypes.byref(h)) == _lib.EINVAL and not h.value
    assert L.amlike_norm_create(None, 8, 1e-5, None) == _lib.EINVAL
    assert L.amlike_norm_destroy(None) == _lib.OK and L.amlike_linear_destroy(None) == _lib.OK
    assert L.amlike_norm_dim(None) == 0 and L.amlike_linear_output_dim(None) == 0
    assert L.amlike_norm_device(None) == -1 and L.amlike_linear_device(None) == -1 and L.amlike_linear_type(None) == -1


def test_python_mirror_checks_shapes():
    with pytest.raises(ValueError):
        dense.Linear(np.ones(3, np.float32))
    with pytest.raises(ValueError):
        dense.Linear(np.ones((3, 2), np.float32), np.ones(2, np.float32))
    with pytest.raises(ValueError):
        dense.RmsNorm(4, np.ones(3, np.float32))
    with pytest.raises(KeyError):
        dense.Matrix(0, "int4", 1)


def test_the_reference_of_the_8_bit_form():
    """Every e4m3 value survives, and a plan of borders gives the scales of the definition."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 0x7F) != 0x7F]
    v = codes.view(torch.float8_e4m3fn).double()
    x = torch.zeros((len(v), 32), dtype=torch.float64)
    x[:, 0], x[:, 1] = v, 448.0
    q, s = U.to_mx8(x)
    assert torch.equal(U.from_mx8(q, s), x) and (s == 127).all()
    for top, k in ((448.0, 0), (448.0001, 1), (224.0, -1), (1.75, -8), (1.7501, -7), (2.0 ** 127, 119), (0.0, -127), (2.0 ** -149, -127)):
        assert int(U.mx8_exponents(torch.full((1, 32), top, dtype=torch.float64))[0, 0]) == k


@pytest.mark.parametrize("big", [2 ** 31, 2 ** 32 + 3, -2 ** 31 - 1, 2 ** 40])
def test_python_mirror_refuses_counts_that_leave_32_bits(big):
    """Beyond 32 bits ctypes would pass on what is left of them: 2^32 + 3 rows would be 3."""
    x, out = dense.Matrix(4096, "bf16", 64), dense.Matrix(1 << 20, "f32", 64)
    for rows, cols in ((big, 64), (4, big)):
        with pytest.raises(ValueError):
            dense.ConvertDevice(x, rows, cols, out)
    with pytest.raises(ValueError):
        dense.RmsNorm(big)
    for cls in (dense.RmsNorm, dense.Linear):  # (the check comes before the handle is looked at)
        h = cls.__new__(cls)
        with pytest.raises(ValueError):
            h.ApplyDevice(x, big, out)
    wide = np.lib.stride_tricks.as_strided(np.zeros(2, np.float32), shape=(1, 2), strides=(4 * (2 ** 32 + 2), 4))
    a, ld = dense._rows(wide, 2, "x")  # a stride too large for the C side is copied away
    assert ld == 2 and a.flags.c_contiguous


def test_python_mirror_refuses_strides_that_leave_64_bits():
    for kw in (dict(ld=2 ** 63), dict(ld=2 ** 64 + 64), dict(ld=64, ld_scales=2 ** 64 + 2), dict(ptr=2 ** 64 + 4096, ld=64), dict(ptr=-1, ld=64)):
        with pytest.raises(ValueError):
            dense.Matrix(kw.pop("ptr", 4096), "mx8", kw.pop("ld"), 1 << 20, kw.pop("ld_scales", 2))


# (two matrices of 4 x 64 bf16 in a stretch of memory, and how they lie)
APART = [(dict(ld=128), dict(ptr=4096 + 128, ld=128)),                                 # side by side
         (dict(ptr=4096 + 128, ld=128), dict(ld=128)),
         (dict(ld=192), dict(ptr=4096 + 128, type_="f32", ld=96)),                     # 128 and 256 bytes of 384
         (dict(ld=128), dict(ptr=4096 + 128, ld=256)),                                 # every second row's second half
         (dict(ld=128), dict(ptr=4096 + 3 * 256 + 128, ld=64)),                        # behind the last row
         (dict(ld=128), dict(ptr=4096 + 128, type_="mx8", ld=256, scales=4096 + 192, ld_scales=256))]
MEETING = [(dict(ld=128), dict(ptr=4096 + 126, ld=128)), (dict(ptr=4096 + 126, ld=128), dict(ld=128)),
           (dict(ld=128), dict(ptr=4096 + 130, ld=128)), (dict(ld=128), dict(ptr=4096 + 128, ld=64)),
           (dict(ld=128), dict(ptr=4096 + 3 * 256 + 126, ld=64)), (dict(ld=128), dict(ptr=4096 + 128, type_="f32", ld=64)),
           (dict(ld=128), dict(ptr=4096 + 128, type_="mx8", ld=256, scales=4096 + 255, ld_scales=256))]


@pytest.mark.parametrize("x,out", MEETING)
def test_matrices_that_share_bytes_are_refused(x, out):
    assert convert(matrix(**x), 4, 64, matrix(**out)) == _lib.EINVAL
    assert "overlap" in _lib.lib().amlike_last_error().decode()


@pytest.mark.parametrize("x,out", APART)
def test_matrices_side_by_side_are_not_refused(x, out):
    """Without a GPU the call ends where it looks for one, behind the checks."""
    if _lib.lib().amlike_device_count() > 0:
        pytest.skip("the addresses are made up")
    assert convert(matrix(**x), 4, 64, matrix(**out)) == _lib.ENODEV


def test_overlap_is_exact():
    """Small matrices in a small stretch of memory against the sets of their bytes."""
    if _lib.lib().amlike_device_count() > 0:
        pytest.skip("the addresses are made up")
    rng = np.random.default_rng(1)
    sizes = {"f32": 4, "bf16": 2, "f16": 2, "mx8": 1}
    met = 0
    for _ in range(6000):
        rows, cols = int(rng.integers(1, 12)), int(rng.integers(1, 40))
        bytes_, args = [], []
        for t in (["f32", "bf16", "f16"][rng.integers(3)], list(sizes)[rng.integers(4)]):
            at, ld = 4096 + 4 * int(rng.integers(0, 300)), cols + int(rng.integers(0, 4)) * int(rng.integers(0, 60))
            groups = (cols + 31) // 32
            scales, ld_scales = 4096 + int(rng.integers(0, 1200)) if t == "mx8" else 0, groups + int(rng.integers(0, 80))
            mine = {at + (r * ld + c) * sizes[t] + i for r in range(rows) for c in range(cols) for i in range(sizes[t])}
            if t == "mx8":
                own = {scales + r * ld_scales + c for r in range(rows) for c in range(groups)}
                while mine & own:  # (its scales lie elsewhere)
                    scales += 1 << 20
                    own = {v + (1 << 20) for v in own}
                mine |= own
            bytes_.append(mine)
            args.append(matrix(ptr=at, type_=t, ld=ld, scales=scales, ld_scales=ld_scales))
        meet = bool(bytes_[0] & bytes_[1])
        met += meet
        assert convert(args[0], rows, cols, args[1]) == (_lib.EINVAL if meet else _lib.ENODEV)
    assert 1000 < met < 5000  # both happen


def test_overlap_of_matrices_as_large_as_there_are():
    """2^31 - 1 rows whose strides share no divisor: refused or not within no time."""
    if _lib.lib().amlike_device_count() > 0:
        pytest.skip("the addresses are made up")
    rows = 2 ** 31 - 1
    for ld, at, meet in ((100003, 2 * 100003 * rows - 16, False), (100003, 2 * 100003 * (rows - 1) + 14, True), (100001, 0, True),
                         (100003, 16, False), (100003, 14, True), (100003, 2 * 100003 - 16, False), (100003, 2 * 100003 - 14, True)):
        a, b = matrix(ptr=4096, ld=100003), matrix(ptr=4096 + at, ld=ld)
        assert convert(a, rows, 8, b) == (_lib.EINVAL if meet else _lib.ENODEV), (ld, at)


@pytest.mark.parametrize("scales,ld_scales", [(4096, 4), (4096 + 62, 4), (4096 + 3 * 128 + 63, 1 << 20), (4096 + 63, 128), (4096 - 1, 4)])
def test_values_and_scales_of_an_output_that_share_bytes_are_refused(scales, ld_scales):
    """(Which of a value and a scale was written last would be anybody's guess.)"""
    x = matrix(ptr=1 << 20)
    assert convert(x, 4, 64, matrix(ptr=4096, type_="mx8", ld=128, scales=scales, ld_scales=ld_scales)) == _lib.EINVAL
    assert "scales overlap" in _lib.lib().amlike_last_error().decode()
    # bytes [4096, 4160) and two scales
    assert convert(x, 1, 64, matrix(ptr=4096, type_="mx8", ld=64, scales=4095, ld_scales=2)) == _lib.EINVAL
    assert convert(x, 1, 64, matrix(ptr=4096, type_="mx8", ld=64, scales=4159, ld_scales=2)) == _lib.EINVAL


@pytest.mark.parametrize("rows,scales,ld_scales", [(4, 4096 + 64, 4), (4, 4096 + 64, 128), (4, 4096 + 126, 128), (1, 4094, 2), (1, 4160, 2)])
def test_scales_of_an_output_between_its_values_are_not_refused(rows, scales, ld_scales):
    if _lib.lib().amlike_device_count() > 0:
        pytest.skip("the addresses are made up")
    out = matrix(ptr=4096, type_="mx8", ld=128, scales=scales, ld_scales=ld_scales)
    assert convert(matrix(ptr=1 << 20), rows, 64, out) == _lib.ENODEV


def test_no_rows_are_no_overlap():
    assert convert(matrix(ptr=1 << 20), 0, 64, matrix(ptr=4096, type_="mx8", ld=64, scales=4096, ld_scales=2)) == _lib.OK
