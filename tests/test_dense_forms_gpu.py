"""Every form of the linear kernels on sums of integers that fp32 holds exactly: every product is there
once, and nothing else."""
import pytest
import torch

import dense_forms as F
import dense_util as U
from kaldi_amd import dense

pytestmark = pytest.mark.gpu


def ints(rows, cols, seed, top=8):
    return torch.randint(-top, top + 1, (rows, cols), generator=torch.Generator().manual_seed(seed), dtype=torch.float32).double()


def run(type_, tout, rows, k, n, aligned, residual):
    x, w, b = ints(rows, k, 1), ints(n, k, 2), ints(1, n, 3, 99)[0]
    r = ints(rows, n, 4, 99) if residual else None
    lin = dense.Linear(w.numpy(), b.numpy(), type_)
    dx = U.DeviceMatrix(rows, k, type_, (k + 31) // 16 * 16 - k if aligned else 3, fill=x)
    dr = U.DeviceMatrix(rows, n, "f32", 1, fill=r) if residual else None
    out = U.DeviceMatrix(rows, n, tout, 8 if aligned else 5)
    lin.ApplyDevice(dx.m, rows, out.m, residual=dr.m if residual else None)
    torch.cuda.synchronize()
    want = torch.from_numpy(x.numpy() @ w.numpy().T) + b
    if residual:
        want = want + r
    if tout == "mx8":
        U.check_output(out, want, torch.zeros_like(want))
    else:
        assert torch.equal(out.values(), U.rounded(want, tout))
    out.assert_rest_untouched()
    return dx


@pytest.mark.parametrize("type_,tout,rows,k,n,aligned", F.CASES)
def test_form_is_exact_on_small_integers(amlike_device, type_, tout, rows, k, n, aligned):
    dx = run(type_, tout, rows, k, n, aligned, residual=rows * n < 1 << 22)
    if torch.cuda.get_device_properties(0).multi_processor_count == F.UNITS:  # (else the sizes take other forms)
        assert F.is_aligned(type_, k, dx.ld, dx.ld_scales if type_ == "mx8" else 0) == aligned


@pytest.mark.parametrize("type_,tout", [("bf16", "f32"), ("f16", "mx8"), ("bf16", "bf16"), ("mx8", "f32"), ("mx8", "bf16"), ("mx8", "mx8")])
@pytest.mark.parametrize("rows,k,n", [(1000, 208, 130), (257, 1040, 70), (512, 333, 700), (3000, 400, 2000)])
def test_a_call_in_several_launches(amlike_device, monkeypatch, type_, tout, rows, k, n):
    """Stretches of 256 rows, the last one short or not: what an output beyond 2^22 blocks would need."""
    monkeypatch.setenv("AMLIKE_LINEAR_MAX_BLOCKS", "1")
    for residual in (False, True):
        run(type_, tout, rows, k, n, k % 16 == 0, residual)
