"""References in 64 bits and tolerances for the dense-layer operators (torch on the CPU)."""
import math

import torch

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t):
    """Largest relative error of one rounding to nearest."""
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11, "mx8": 2.0 ** -4}[t]


def groups(a):
    rows, cols = a.shape
    return torch.nn.functional.pad(a, (0, -cols % 32)).reshape(rows, -1, 32)


def mx8_exponents(y):
    """Smallest k >= -127 with max|finite y of the group| <= 448 * 2^k, of a float64 matrix."""
    g = groups(y)
    top = torch.where(torch.isfinite(g), g.abs(), torch.zeros_like(g)).amax(2)
    m, e = torch.frexp(top)  # top = m * 2^e, .5 <= m < 1; 448 = .875 * 2^9
    k = e - 9 + (m > 0.875).int()
    return torch.where(top > 0, k, torch.full_like(k, -127)).clamp(min=-127)


def to_mx8(y):
    """float64 -> (e4m3 values, scale bytes), both uint8."""
    rows, cols = y.shape
    k = mx8_exponents(y)
    v = groups(y) * torch.exp2(-k.double()).unsqueeze(2)
    v = torch.where(torch.isfinite(v), v, torch.full_like(v, math.nan))
    # (fp32 holds y * 2^-k of a bf16, f16 or f32 y exactly or far below e4m3's range)
    q = v.reshape(rows, -1)[:, :cols].float().to(torch.float8_e4m3fn)
    return q.view(torch.uint8).contiguous(), (k + 127).to(torch.uint8)


def from_mx8(q, scales):
    rows, cols = q.shape
    v = q.view(torch.float8_e4m3fn).double()
    s = torch.exp2(scales.double() - 127)
    return (groups(v) * s.unsqueeze(2)).reshape(rows, -1)[:, :cols]


def rounded(y, type_):
    """What a device matrix of the type holds of a float64 y, as float64."""
    if type_ == "mx8":
        return from_mx8(*to_mx8(y))
    return y.to(TORCH[type_]).double()


class DeviceMatrix:
    """A device matrix with `pad` more columns in its buffer and `behind` more rows, all of which
    start as a bit pattern that is a NaN in every type."""

    def __init__(self, rows, cols, type_, pad=0, behind=2, fill=None, offset=0):
        from kaldi_amd import dense
        self.rows, self.cols, self.type = rows, cols, type_
        self.ld = cols + pad
        dt = torch.uint8 if type_ == "mx8" else TORCH[type_]
        n = (rows + behind) * self.ld
        raw = torch.full(((n + offset) * dt.itemsize,), 0xFF, dtype=torch.uint8, device="cuda")
        self.buf = raw.view(dt)[offset:].view(rows + behind, self.ld)
        self.scales = None
        if type_ == "mx8":
            # (rows of scales that start on 16 bytes where those of values may, and any others)
            self.ld_scales = ((cols + 31) // 32 + 15) // 16 * 16 if pad % 8 == 0 else (cols + 31) // 32 + 1
            self.scales = torch.full((rows + behind, self.ld_scales), 0xFF, dtype=torch.uint8, device="cuda")
        if fill is not None:
            if type_ == "mx8":
                q, s = to_mx8(fill)
                self.buf[:rows, :cols] = q.cuda()
                self.scales[:rows, :s.shape[1]] = s.cuda()
            else:
                self.buf[:rows, :cols] = fill.to(TORCH[type_]).cuda()
        self.m = dense.Matrix(self.buf.data_ptr(), type_, self.ld, self.scales.data_ptr() if self.scales is not None else 0,
                              self.ld_scales if self.scales is not None else 0)

    def values(self):
        """What it holds, as float64 on the CPU."""
        v = self.buf[:self.rows, :self.cols].cpu()
        if self.type == "mx8":
            return from_mx8(v.contiguous(), self.scales[:self.rows, :(self.cols + 31) // 32].cpu())
        return v.double()

    def assert_rest_untouched(self):
        b = self.buf.view(torch.uint8).cpu()
        es = b.shape[1] // self.ld
        assert (b[self.rows:] == 0xFF).all() and (b[:, self.cols * es:] == 0xFF).all()
        if self.scales is not None:
            s = self.scales.cpu()
            assert (s[self.rows:] == 0xFF).all() and (s[:, (self.cols + 31) // 32:] == 0xFF).all()


def assert_close(got, want, tol, what=""):
    """|got - want| <= tol elementwise; what is not finite has to agree."""
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine] - (tol.expand_as(want)[fine] if torch.is_tensor(tol) else tol)
    assert off.numel() == 0 or float(off.max()) <= 0, "%s: beyond the tolerance by %g" % (what, float(off.max()))


def same(a, b):
    """Equal values, NaN for NaN."""
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def check_output(dm, want, before):
    """dm holds `want` (float64) rounded once, where the value before the rounding may be off by
    `before` (a tensor like want)."""
    got = dm.values()
    if dm.type != "mx8":
        tiny = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}[dm.type]  # half the smallest step
        top = float(torch.finfo(TORCH[dm.type]).max)
        edge = (want.abs() + before) * (1 + half_step(dm.type)) >= top  # may or may not round to infinity
        w = torch.where(edge, got, want)
        assert_close(got, w, before + (w.abs() + before) * half_step(dm.type) + tiny, dm.type)
        return
    k = dm.scales[:dm.rows, :(dm.cols + 31) // 32].cpu().double() - 127
    g, b = groups(torch.where(torch.isfinite(want), want, torch.zeros_like(want))), groups(before)
    at = g.abs().argmax(2, keepdim=True)
    top, slack = g.abs().gather(2, at)[..., 0], b.amax(2)
    assert (top - slack <= 448 * torch.exp2(k)).all(), "a scale is too small"
    assert ((k == -127) | (top + slack > 448 * torch.exp2(k - 1))).all(), "a scale is too large"
    # e4m3: half a step is 2^-4 of the value, below 2^-6 it is 2^-10
    scale = torch.exp2(k).repeat_interleave(32, dim=1)[:, :dm.cols]
    fine = torch.where(torch.isfinite(want), want, torch.full_like(want, math.nan))
    assert_close(got, fine, before + torch.maximum((want.abs() + before) * 2.0 ** -4, scale * 2.0 ** -10), "mx8")
