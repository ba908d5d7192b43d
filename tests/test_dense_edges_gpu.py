"""The dense-layer operators at the ends of what they take, on the GPU."""
import numpy as np
import pytest
import torch

import dense_util as U
from kaldi_amd import dense

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
