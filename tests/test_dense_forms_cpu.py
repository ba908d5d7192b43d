"""Which form of the linear kernels a call takes, and that the GPU tests' sizes take every one."""
import math
import random

import pytest

import dense_forms as F
from kaldi_amd import _lib, dense


def test_every_reachable_form_is_among_the_tested_sizes():
    rng, reached = random.Random(1), {}
    for _ in range(40000):
        type_, out = rng.choice(["bf16", "f16", "mx8"]), rng.choice(["f32", "bf16", "f16", "mx8"])
        rows, k, n = (int(math.exp(rng.uniform(0, top))) for top in (11.5, 9.5, 10.5))
        aligned = rng.random() < 0.5
        if aligned:
            k = (k + 15) // 16 * 16
        reached.setdefault(F.form(type_, out, rows, k, n, aligned), (type_, out, rows, k, n, aligned))
    tested = {F.form(*c) for c in F.CASES}
    assert len(reached) > 40
    missing = {f: c for f, c in reached.items() if f not in tested}
    assert not missing, missing


@pytest.mark.parametrize("case", F.CASES)
def test_the_sizes_are_aligned_as_they_say(case):
    type_, _, _, k, _, aligned = case
    assert not aligned or F.is_aligned(type_, k, (k + 31) // 16 * 16, 16)


def test_sizes_out_of_range_have_no_kernel():
    assert dense.linear_kernel_info("bf16", "f32", 1, 64, 64).startswith("linear_thin_kernel<1,")
    for args in ((0, 64, 64), (-1, 64, 64), (4, 0, 64), (4, 64, 0), (4, (1 << 20) + 1, 64), (4, 64, (1 << 20) + 1)):
        assert dense.linear_kernel_info("bf16", "f32", *args) == ""
    assert dense.linear_kernel_info("f32", "f32", 4, 64, 64) == "" and dense.linear_kernel_info("bf16", "f32", 4, 64, 64, units=0) == ""
    assert _lib.lib().amlike_linear_kernel_info(1, 4, 4, 64, 64, 1, 256) == b""
    # the largest sizes there are
    for out in ("f32", "mx8"):
        assert dense.linear_kernel_info("mx8", out, 2 ** 31 - 1, 1 << 20, 1 << 20) != ""
