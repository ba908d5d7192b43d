"""8-bit layers whose scales lie at the ends of their range, on the GPU, against sums of integers that
fp32 holds exactly."""
import math

import pytest
import torch

import dense_util as U
from kaldi_amd import dense

pytestmark = pytest.mark.gpu

# From one row to all forms of both kernels for an fp32 output on 256 compute units; pad 16: rows on 16
# bytes, pad 3: rows anywhere.
SIZES = [(3, 96, 40, 16), (20, 256, 64, 16), (64, 1000, 512, 16), (100, 360, 300, 16), (256, 1024, 4096, 16), (300, 1000, 700, 3),
         (990, 400, 2000, 16), (990, 1008, 4000, 16), (500, 1017, 2000, 3), (1990, 2000, 1990, 16), (4090, 2000, 4090, 16),
         (1990, 601, 1990, 3)]


def ints(rows, cols, lo, hi, seed):
    return torch.randint(lo, hi + 1, (rows, cols), generator=torch.Generator().manual_seed(seed)).double()


def codes(v):
    """e4m3 bytes of values that e4m3 holds."""
    q = v.float().to(torch.float8_e4m3fn)
    assert torch.equal(q.double(), v)
    return q.view(torch.uint8)


def matrix(q, bytes_, pad):
    """A device matrix of the given e4m3 codes and scale bytes (one per group)."""
    m = U.DeviceMatrix(q.shape[0], q.shape[1], "mx8", pad, fill=torch.ones(q.shape, dtype=torch.float64))
    m.buf[:q.shape[0], :q.shape[1]] = q.cuda()
    m.scales[:q.shape[0], :bytes_.shape[1]] = bytes_.to(torch.uint8).cuda()
    return m


def apply(lin, x, n, tout, pad=0):
    out = U.DeviceMatrix(x.rows, n, tout, pad)
    lin.ApplyDevice(x.m, x.rows, out.m)
    torch.cuda.synchronize()
    out.assert_rest_untouched()
    return out.values()


@pytest.mark.parametrize("rows,k,n,pad", SIZES)
def test_groups_of_far_scales_next_to_ordinary_ones(amlike_device, rows, k, n, pad):
    """Scales of x from 2^-127 to 2^127 over e4m3's smallest values (multiples of 2^-9), weights so scaled
    that all products are multiples of 2^-18: at most k * 64 of these, below 2^24.  The weights' own
    groups reach the smallest scale and its smallest values too."""
    groups = (k + 31) // 32
    of = torch.tensor([127, 0, 254, 1, 130, 247, 2, 120, 250, 3])[torch.arange(groups) % 10]  # bytes by group
    xi, wi = ints(rows, k, -8, 8, 1), ints(n, k, -8, 8, 2)
    wide = of.double().repeat_interleave(32)[:k]
    lin = dense.Linear((wi * torch.exp2(118 - wide)).numpy(), None, "mx8")  # times 2^(byte - 127 - 9): 2^-18
    want = xi @ wi.t() * 2.0 ** -18
    got = apply(lin, matrix(codes(xi * 2.0 ** -9), of.expand(rows, groups), pad), n, "f32", pad)
    assert torch.equal(got, want)
    # a smaller output: products below 2^7 times their unit lose nothing in the 8-bit instruction
    got = apply(lin, matrix(codes(xi * 2.0 ** -9), of.expand(rows, groups), pad), n, "bf16", pad)
    assert torch.equal(got, want.bfloat16().double())


@pytest.mark.parametrize("tout", ["f32", "bf16"])
@pytest.mark.parametrize("byte,e", [(0, 118), (1, 118), (2, 118), (3, 118), (246, -146), (246, -100), (247, -147), (247, -100),
                                    (248, -148), (248, -100), (251, -151), (251, -100), (254, -154), (254, -100), (254, -10)])
def test_every_code_under_the_first_and_last_scales(amlike_device, byte, e, tout):
    """A layer that copies its input, times a power of two that brings it back into fp32's range.  (2^-146
    and below are 0 in 8 bits, where the smallest value is 2^-136.)"""
    q = torch.arange(256, dtype=torch.uint8).view(16, 16).repeat_interleave(2, dim=1)
    k = q.shape[1]
    w = torch.eye(k).double() * 2.0 ** e
    lin = dense.Linear(w.numpy(), None, "mx8")
    want = U.from_mx8(q, torch.full((16, 1), byte, dtype=torch.uint8)) * float(U.rounded(w, "mx8")[0, 0])
    got = apply(lin, matrix(q, torch.full((16, 1), byte), 16), k, tout)
    # a row that holds a NaN is NaN: every other product of it is NaN * 0
    bad = torch.isnan(want).any(1)
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])


def test_the_largest_values_that_conversion_writes(amlike_device):
    """3.39e38 is 256 * 2^120 in 8 bits, 2^128: a weight of 2^-20 makes 2^108 of it, one of 0 makes 0."""
    x = torch.zeros(2, 64, dtype=torch.float64)
    x[0, 3], x[1, 40] = 3.39e38, -3.39e38
    w = torch.zeros(3, 64, dtype=torch.float64)
    w[0, 3], w[1, 40] = 2.0 ** -20, 2.0 ** -20
    src, q = U.DeviceMatrix(2, 64, "f32", fill=x), U.DeviceMatrix(2, 64, "mx8", 16)
    dense.ConvertDevice(src.m, 2, 64, q.m)
    lin = dense.Linear(w.numpy(), None, "mx8")
    want = torch.zeros(2, 3, dtype=torch.float64)
    want[0, 0], want[1, 1] = 2.0 ** 108, -2.0 ** 108
    for tout in ("f32", "bf16"):
        assert torch.equal(apply(lin, q, 3, tout), want)
    # and as a weight
    lin = dense.Linear(x.numpy(), None, "mx8")
    v = U.DeviceMatrix(3, 64, "mx8", 16, fill=w)
    for tout in ("f32", "bf16"):
        assert torch.equal(apply(lin, v, 2, tout), want.t())


@pytest.mark.parametrize("rows,k,n,pad", SIZES)
def test_rows_do_not_notice_far_scales_in_others(amlike_device, rows, k, n, pad):
    """Rows of rounded, ordinary numbers keep their bits beside rows with far scales, of zeros and of
    NaN; rows of zeros under byte 0 give zeros."""
    x, w = torch.randn((rows, k), generator=torch.Generator().manual_seed(3)).double(), ints(n, k, -99, 99, 4) / 64
    q, s = U.to_mx8(x)
    lin = dense.Linear(w.numpy(), None, "mx8")
    base = apply(lin, matrix(q, s, pad), n, "f32", pad)
    q2, s2 = q.clone(), s.clone()
    far = torch.arange(rows) % 7
    q2[far == 1] = 0
    s2[far == 1] = 0
    s2[far == 2, 0] = 254
    q2[far == 2, 0] = 0x7E
    s2[far == 3, -1] = 1
    q2[far == 3, -1] = 1
    s2[far == 4, 1] = 255
    got = apply(lin, matrix(q2, s2, pad), n, "f32", pad)
    keep = (far == 0) | (far > 4)
    assert torch.equal(got[keep], base[keep])
    assert (got[far == 1] == 0).all() and torch.isnan(got[far == 4]).all()
    # rows with one small group against 64 bits: an fp32 sum of k products, each addition rounded or cut off
    if (far == 3).any():
        v, wv = U.from_mx8(q2[far == 3], s2[far == 3]), U.rounded(w, "mx8")
        off = (got[far == 3] - v @ wv.t()).abs() - ((k + 2) * 2.0 ** -23 * (v.abs() @ wv.abs().t()) + 2.0 ** -149)
        assert float(off.max()) <= 0


def test_far_scales_of_one_column_and_of_short_rows(amlike_device):
    """One column, and a last group that is short; what a row's scales hold behind its last one is not used."""
    for k in (1, 33, 129):
        groups = (k + 31) // 32
        xi = ints(5, k, 1, 8, 5)
        lin = dense.Linear(torch.full((9, k), 2.0 ** 100, dtype=torch.float64).numpy(), None, "mx8")
        m = matrix(codes(xi * 2.0 ** -9), torch.zeros(5, groups), 16)
        want = (xi.sum(1, keepdim=True) * 2.0 ** -36).expand(5, 9)
        for behind in (0, 254, 255):
            m.scales[:5, groups:] = behind
            out = U.DeviceMatrix(5, 9, "f32")
            lin.ApplyDevice(m.m, 5, out.m)
            torch.cuda.synchronize()
            assert torch.equal(out.values(), want) and math.isfinite(float(want.max()))


@pytest.mark.parametrize("rows,k,n,pad", [(1000, 208, 130, 16), (700, 333, 70, 3), (600, 1040, 2000, 16)])
def test_far_scales_in_a_call_of_several_launches(amlike_device, monkeypatch, rows, k, n, pad):
    """Each launch finds the scales of its own rows; replayed from a graph it gives the same."""
    monkeypatch.setenv("AMLIKE_LINEAR_MAX_BLOCKS", "1")
    groups = (k + 31) // 32
    of = torch.full((rows, groups), 127)
    of[::101, ::3] = 254
    of[50::77] = 0
    xi, wi = ints(rows, k, -8, 8, 7), ints(n, k, -8, 8, 8)
    lin = dense.Linear(wi.numpy(), None, "mx8")
    x = matrix(codes(xi * 2.0 ** -9), of, pad)
    want = (xi * torch.exp2(of.double() - 136).repeat_interleave(32, dim=1)[:, :k]) @ wi.t()
    same = (of == of[:, :1]).all(1)  # (rows of one scale: their sums are exact)
    got = apply(lin, x, n, "f32", pad)
    assert same.sum() > rows // 2 and torch.equal(got[same], want[same])
    mass = (xi.abs() * torch.exp2(of.double() - 136).repeat_interleave(32, dim=1)[:, :k]) @ wi.abs().t()
    over = torch.isinf(got) & (mass >= 2.0 ** 127)  # (no partial sum passes the mass; one beyond fp32's range is infinite)
    assert (over | ((got - want).abs() <= (k + 1) * 2.0 ** -23 * mass)).all() and not over[::101].all()
    out, graph, stream = U.DeviceMatrix(rows, n, "f32"), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        lin.ApplyDevice(x.m, rows, out.m, stream=stream.cuda_stream)
    for _ in range(3):
        out.buf.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.values(), got)
