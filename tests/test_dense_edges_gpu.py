"""The dense-layer operators at the ends of what they take, on the GPU."""
import ctypes

import numpy as np
import pytest
import torch

import dense_util as U
from kaldi_amd import _lib, dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("tout", ["f32", "bf16", "f16"])
def test_silu_of_large_negative_arguments(amlike_device, rows, tout):
    """x / (1 + exp(-x)) is a normal number down to x = -91, where 1 / (1 + exp(-x)) no longer is from -87.4 on.
    Exponentials' arguments of up to |x| in all carry half a step each and the constant's; two of them, the
    reciprocal (a unit each) and four products and sums stay below (6 + 2 |x|) units."""
    x = torch.cat([torch.linspace(-104, -60, 353), torch.tensor([-87.25, -87.5, -88.0, -88.5, -89.0, -1e3, -3e38, 0.0, 30.0, 3e38])])
    x = x.bfloat16().double().repeat(rows, 1)
    n = x.shape[1]
    lin = dense.Linear(np.eye(n, dtype=np.float32), None, "bf16")
    out = U.DeviceMatrix(rows, n, tout)
    lin.ApplyDevice(U.DeviceMatrix(rows, n, "bf16", fill=x).m, rows, out.m, activation="silu")
    torch.cuda.synchronize()
    want = x / (1 + torch.exp(-x))
    U.check_output(out, want, (6 + 2 * x.abs().clamp(max=200)) * 2.0 ** -23 * want.abs())


class Slices:
    """Column blocks of one bf16 buffer whose first and last columns are guards."""

    def __init__(self, rows, widths, seed):
        self.rows, self.widths = rows, widths
        self.at = [8 + sum(widths[:i]) for i in range(len(widths))]
        ld = 16 + sum(widths)
        self.buf = torch.randn((rows, ld), generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        self.start = self.buf.clone()
        self.m = [dense.Matrix(self.buf.data_ptr() + 2 * a, "bf16", ld) for a in self.at]

    def block(self, i, before=False):
        return (self.start if before else self.buf)[:, self.at[i]:self.at[i] + self.widths[i]].cpu().double()

    def assert_only(self, *written):
        keep = torch.ones(self.buf.shape[1], dtype=torch.bool)
        for i in written:
            keep[self.at[i]:self.at[i] + self.widths[i]] = False
        assert torch.equal(self.buf[:, keep.cuda()], self.start[:, keep.cuda()])


@pytest.mark.parametrize("rows", [3, 70, 500])
def test_operands_and_results_side_by_side_in_one_buffer(amlike_device, rows):
    """x, residual, sum and output as column blocks of one wide buffer: the same bits as apart."""
    s = Slices(rows, [200, 200, 200, 200], 1)
    norm = dense.RmsNorm(200)
    norm.ApplyDevice(s.m[0], rows, s.m[3], residual=s.m[1], sum=s.m[2])
    apart = [U.DeviceMatrix(rows, 200, "bf16", fill=s.block(i, True)) for i in range(4)]
    norm.ApplyDevice(apart[0].m, rows, apart[3].m, residual=apart[1].m, sum=apart[2].m)
    torch.cuda.synchronize()
    s.assert_only(2, 3)
    assert torch.equal(s.block(2), apart[2].values()) and torch.equal(s.block(3), apart[3].values())

    s = Slices(rows, [360, 264, 264], 2)
    lin = dense.Linear(torch.randn((264, 360), generator=torch.Generator().manual_seed(3)).numpy(), None, "bf16")
    lin.ApplyDevice(s.m[0], rows, s.m[1], residual=s.m[2])
    apart = [U.DeviceMatrix(rows, s.widths[i], "bf16", 8, fill=s.block(i, True)) for i in range(3)]
    lin.ApplyDevice(apart[0].m, rows, apart[1].m, residual=apart[2].m)
    torch.cuda.synchronize()
    s.assert_only(1)
    assert torch.equal(s.block(1), apart[1].values())

    s = Slices(rows, [64, 64], 4)
    dense.ConvertDevice(s.m[0], rows, 64, s.m[1])
    torch.cuda.synchronize()
    s.assert_only(1)
    assert torch.equal(s.block(1), s.block(0, True))


def test_an_8_bit_layer_between_rows_of_one_buffer(amlike_device):
    """Rows of [x | scales of x | output | scales of the output]: a layer in place in its record."""
    rows, k, n = 130, 256, 512
    x = U.rounded(torch.randn((rows, k), generator=torch.Generator().manual_seed(5)).double(), "mx8")
    w = torch.randn((n, k), generator=torch.Generator().manual_seed(6)).numpy()
    lin = dense.Linear(w, None, "mx8")
    apart, out = U.DeviceMatrix(rows, k, "mx8", 16, fill=x), U.DeviceMatrix(rows, n, "mx8", 16)
    lin.ApplyDevice(apart.m, rows, out.m, activation="relu")
    ld = k + 16 + n + 16
    buf = torch.zeros((rows, ld), dtype=torch.uint8, device="cuda")
    buf[:, :k] = apart.buf[:rows, :k]
    buf[:, k:k + 8] = apart.scales[:rows, :8]
    p = buf.data_ptr()
    lin.ApplyDevice(dense.Matrix(p, "mx8", ld, p + k, ld), rows, dense.Matrix(p + k + 16, "mx8", ld, p + k + 16 + n, ld), activation="relu")
    torch.cuda.synchronize()
    assert torch.equal(buf[:, k + 16:k + 16 + n], out.buf[:rows, :n])
    assert torch.equal(buf[:, k + 16 + n:], out.scales[:rows, :16])
    assert torch.equal(buf[:, :k], apart.buf[:rows, :k]) and (buf[:, k + 8:k + 16] == 0).all()


@pytest.mark.parametrize("type_", ["bf16", "f16"])
def test_what_a_16_bit_matrix_has_as_scales_is_not_looked_at(amlike_device, type_):
    """scales and ld_scales belong to 8-bit matrices: left as anything, they change neither kernel nor bits."""
    rows, k, n = 1024, 1000, 1000
    lin = dense.Linear(torch.randn((n, k), generator=torch.Generator().manual_seed(7)).numpy(), None, type_)
    x = U.DeviceMatrix(rows, k, type_, 8, fill=torch.randn((rows, k), generator=torch.Generator().manual_seed(8)).double())
    r = U.DeviceMatrix(rows, n, "f32", 0, fill=torch.ones((rows, n), dtype=torch.float64))
    want, out = U.DeviceMatrix(rows, n, "f32"), U.DeviceMatrix(rows, n, "f32")
    lin.ApplyDevice(x.m, rows, want.m, residual=r.m)
    odd = [dense.Matrix(m.buf.data_ptr(), m.type, m.ld, 4097, 2 ** 62 + 5) for m in (x, out, r)]
    lin.ApplyDevice(odd[0], rows, odd[1], residual=odd[2])
    torch.cuda.synchronize()
    assert torch.equal(out.values(), want.values())
    norm, y, z = dense.RmsNorm(k), U.DeviceMatrix(rows, k, "f32"), U.DeviceMatrix(rows, k, "f32")
    norm.ApplyDevice(x.m, rows, y.m)
    norm.ApplyDevice(odd[0], rows, dense.Matrix(z.buf.data_ptr(), "f32", z.ld, 4097, -3))
    torch.cuda.synchronize()
    assert torch.equal(y.values(), z.values())


def test_a_refusal_for_memory_leaves_no_error_behind(amlike_device):
    """4 TB of weights, and host rows of 2^48 bytes: refused before the arrays are looked at; neither this library's
    nor anybody else's next call finds the error."""
    L, w, h = _lib.lib(), np.ones(8, np.float32), ctypes.c_void_p()
    fp = w.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
    x, out = U.DeviceMatrix(4, 64, "f32", fill=torch.ones(4, 64)), U.DeviceMatrix(4, 64, "bf16")
    norm = dense.RmsNorm(32768)
    lin = dense.Linear(np.ones((32768, 32), np.float32), None, "bf16")
    torch.cuda.synchronize()

    def too_much():
        assert L.amlike_linear_create(fp, 1 << 20, None, 1 << 20, 1 << 20, 1, ctypes.byref(h)) == _lib.EOOM and not h.value
        yield
        assert L.amlike_norm_apply(norm._h, fp, 32768, None, 0, 2 ** 31 - 1, None, 0, fp, 32768) == _lib.EOOM
        yield
        assert L.amlike_linear_apply(lin._h, fp, 32, 2 ** 31 - 1, 0, None, 0, fp, 32768) == _lib.EOOM
        yield

    for _ in too_much():
        assert "out of memory" in L.amlike_last_error().decode()
        assert L.amlike_convert_dev(x.m.ref, 4, 64, out.m.ref, None) == _lib.OK
    for _ in too_much():
        assert float(torch.ones(5, device="cuda").sum()) == 5.0
    torch.cuda.synchronize()
    assert (out.values() == 1).all()
